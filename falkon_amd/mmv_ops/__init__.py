from .attention import attention, cached_attention  # noqa: F401
from .fmmv import fdmmv, fmmv  # noqa: F401
from .layer_norm import layer_norm  # noqa: F401
