"""Layer norm of rows, with its backward pass, on the MI355X.

Kernels compare rows by distances and inner products, so what rows are scaled to decides what a kernel sees.  The
distance kernels divide features by given lengthscales; ``layer_norm`` centres and scales every row by its own
statistics and then applies a learned weight and bias, differentiable in all three:

    y = (x - mean(x)) / sqrt(var(x) + eps) * weight + bias          over the last dimension

The reference has no counterpart.  The work is done by ``flk_layer_norm`` and ``flk_layer_norm_backward``; nothing is
computed on the CPU.
"""
from typing import Optional

import torch

from .. import _backend
from .fmmv import _current, _stream_handle

__all__ = ("layer_norm",)

_DTYPE_CODE = {torch.float32: _backend.FLK_F32, torch.float64: _backend.FLK_F64, torch.float16: _backend.FLK_F16,
               torch.bfloat16: _backend.FLK_BF16}


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as a matrix of rows whose values lie next to each other (a view wherever its strides allow one)."""
    x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, eps, stats: bool):
    lib = _backend.load()
    x2 = _rows(x)
    rows, d = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        wide = torch.float64 if x.dtype == torch.float64 else torch.float32
        mean, rstd = torch.empty((2, rows), dtype=wide, device=x.device).unbind(0)
    affine = weight if weight is not None else bias
    code = _DTYPE_CODE[x.dtype]
    with _current(x.device):
        rc = lib.flk_layer_norm(x2.data_ptr(), rows, d, x2.stride(0), _ptr(weight), _ptr(bias),
                                code if affine is None else _DTYPE_CODE[affine.dtype], eps, y.data_ptr(), _ptr(mean), _ptr(rstd),
                                code, _stream_handle(x.device))
    _backend.raise_for_status(rc, "flk_layer_norm")
    return y, mean, rstd


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        lib = _backend.load()
        x2, dy2 = _rows(x), _rows(dy)
        rows, d = x2.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=x.device) if need_w else None
        db = torch.empty(bias.shape, dtype=bias.dtype, device=x.device) if need_b else None
        code = _DTYPE_CODE[x.dtype]
        affine = weight if weight is not None else bias
        nbytes = lib.flk_layer_norm_backward_workspace_bytes(rows, d, code) if need_w or need_b else 0
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        with _current(x.device):
            rc = lib.flk_layer_norm_backward(x2.data_ptr(), rows, d, x2.stride(0), dy2.data_ptr(), dy2.stride(0), _ptr(weight),
                                             code if affine is None else _DTYPE_CODE[affine.dtype], mean.data_ptr(),
                                             rstd.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), code, _ptr(ws), nbytes,
                                             _stream_handle(x.device))
        _backend.raise_for_status(rc, "flk_layer_norm_backward")
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Every row of ``x`` (its last dimension) centred, scaled to unit variance, times ``weight``, plus ``bias``.

    Parameters
    ----------
    x : GPU tensor of any number of rows, of float32, float64, float16 or bfloat16.  Rows whose values are not next to
        each other in memory are copied first.
    weight, bias : one value per feature, either or both absent; contiguous, of one type: that of ``x`` or, for 16-bit
        ``x``, float32.
    eps : added to the variance.

    Returns a new contiguous tensor like ``x``.  Sums are held in 32 bits (64 for float64) and results rounded once; rows far from zero
    are as exact as others (a constant row is zero).
    Differentiable in ``x``, ``weight`` and ``bias`` (once); gradients are the same run to run.  The call is
    asynchronous on the current stream and can be captured into a graph; to capture its backward pass, first let go of every
    eager result that was computed from the same leaves (torch ties a leaf's gradient to the stream of the first graph alive,
    and capturing across streams that way ends the process).
    """
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPE_CODE:
        raise TypeError(f"layer_norm takes float32, float64, float16 or bfloat16 tensors, not {getattr(x, 'dtype', type(x))}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs at least one feature")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
        if t.shape != x.shape[-1:]:
            raise ValueError(f"{name} must have {x.shape[-1]} entries, got shape {tuple(t.shape)}")
        if t.device != x.device:
            raise RuntimeError(f"{name} must be on the device of x")
        if t.dtype != x.dtype and not (t.dtype == torch.float32 and x.dtype != torch.float64):
            raise TypeError(f"{name} must be of the type of x or, for 16-bit x, float32, not {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must be of one type")
    if x.device.type != "cuda":
        raise RuntimeError("layer_norm runs on the GPU only: tensors must be on a ROCm device")
    weight = weight if weight is None else weight.contiguous()
    bias = bias if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]
