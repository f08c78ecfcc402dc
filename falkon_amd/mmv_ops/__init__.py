from .fmmv import fdmmv, fmmv  # noqa: F401
from .layer_norm import layer_norm  # noqa: F401
