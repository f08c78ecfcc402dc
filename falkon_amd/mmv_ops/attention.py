"""Attention on the MI355X: the row-normalised product of the exponential kernel, and its form over a cache.

``fmmv`` computes ``K(X1, X2) @ v``.  ``attention`` computes the same product with the kernel ``exp(scale * <q, k>)`` and every
row divided by its sum, as a kernel smoother (Nadaraya-Watson) or an attention layer has it, never storing the matrix:

    x_ij  = scale * <q_i, k_j>
    x_ij <- softcap * tanh(x_ij / softcap)                     if softcap > 0
    x_ij <- x_ij - slopes[head] * |pos_i - j|                  if slopes are given
    out_i = sum_j softmax_j(x_ij) v_j                          over the keys j that row i sees

The queries stand at the newest positions of the keys: ``pos_i = i + (number of keys) - (number of queries)``.  A row that
sees no key, or none with a score above minus infinity, is zero.  Keys that no row sees leave no trace in a result or a gradient, whatever
they hold (NaN included); neither does a NaN or an infinity of a key reach a row that does not see it, nor one of a row the keys that it
does not see.  What sees them gets what the formula gives in 32 bits (zero times an infinity is NaN).

Scores, maxima, sums and outputs are held in 32 bits; for 16-bit data the weights (and their gradients) are rounded to
that type before the second product, which is what the matrix cores take (float16's shifted, so that small ones keep their digits).  Scores of more than 1e9 in size are beyond statistics
in 32 bits (a rounding of one is more than an exponent holds): such a row may be NaN.  Results and gradients are the same run to run.
The reference has no counterpart.  The work is done by ``flk_attention``, ``flk_attention_backward`` and
``flk_attention_cached``; nothing is computed on the CPU.
"""
import math
from typing import Optional, Tuple, Union

import torch

from .. import _backend
from .fmmv import _current, _stream_handle

__all__ = ("attention", "cached_attention")

_DTYPE_CODE = {torch.float32: _backend.FLK_F32, torch.float16: _backend.FLK_F16, torch.bfloat16: _backend.FLK_BF16}


def _unit(t: torch.Tensor) -> torch.Tensor:
    """``t`` with the values of a row next to each other (copied only if they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _bsh(t: torch.Tensor):
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _check_operands(what, q, k, v):
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
    if q.dtype not in _DTYPE_CODE:
        raise TypeError(f"{what} takes float32, float16 or bfloat16 tensors, not {q.dtype}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must be of one type, not {q.dtype}, {k.dtype} and {v.dtype}")
    if k.dim() != 4 or v.dim() != 4 or q.dim() != 4:
        raise ValueError(f"{what}: q, k and v must have four dimensions (batch, rows, heads, values)")
    if k.shape[:3] != v.shape[:3] or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{what}: shapes {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)} of q, k and v do not fit together")
    if q.shape[2] == 0 or k.shape[2] == 0 or q.shape[3] == 0 or v.shape[3] == 0:
        raise ValueError(f"{what}: heads and head sizes must not be empty")
    if q.shape[2] % k.shape[2] != 0:
        raise ValueError(f"{what}: {q.shape[2]} query heads cannot share {k.shape[2]} key heads evenly")


def _check_score(what, hq, scale, softcap, slopes, d):
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    softcap = float(softcap)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not (softcap >= 0.0 and math.isfinite(softcap)):
        raise ValueError("softcap must be finite and not negative")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor) or slopes.dtype != torch.float32:
            raise TypeError("slopes must be a float32 tensor")
        if tuple(slopes.shape) != (hq,):
            raise ValueError(f"slopes must have one entry per query head ({hq}), got shape {tuple(slopes.shape)}")
        slopes = slopes.contiguous()
    return scale, softcap, slopes


def _check_whole(t, name, shape):
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be an int32 or int64 tensor")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    return _unit(t if t.dtype == torch.int32 else t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32))


def _check_devices(what, q, *others):
    if q.device.type != "cuda":
        raise RuntimeError(f"{what} runs on the GPU only: tensors must be on a ROCm device")
    for t in others:
        if t is not None and t.device != q.device:
            raise RuntimeError(f"{what}: all tensors must be on the same device")


def _workspace(nbytes: int, dev) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _forward(q, k, v, slopes, scale, softcap, causal, prefix, documents, want_lse, train=False):
    lib = _backend.load()
    b, sq, hq, d = q.shape
    sk, hk, dv = k.shape[1], k.shape[2], v.shape[3]
    out = torch.empty((b, sq, hq, dv), dtype=q.dtype, device=q.device)
    # what rounding takes from 16-bit results: dout.out, which the backward pass subtracts from every term, needs it
    rest = torch.empty_like(out) if train and q.dtype != torch.float32 else None
    lse = torch.empty((b, hq, sq), dtype=torch.float32, device=q.device) if want_lse else None
    code = _DTYPE_CODE[q.dtype]
    nbytes = lib.flk_attention_workspace_bytes(b, sq, sk, hq, dv, documents is not None, code)
    ws = _workspace(nbytes, q.device)
    with _current(q.device):
        rc = lib.flk_attention(*_bsh(q), *_bsh(k), *_bsh(v), b, sq, sk, hq, hk, d, dv, scale, softcap, _ptr(slopes), causal,
                               _ptr(prefix), _ptr(documents), documents.stride(0) if documents is not None else 0,
                               out.data_ptr(), _ptr(rest), _ptr(lse), code, _ptr(ws), nbytes, _stream_handle(q.device))
    _backend.raise_for_status(rc, "flk_attention")
    return out, rest, lse


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, scale, softcap, causal, prefix, documents):
        out, rest, lse = _forward(q, k, v, slopes, scale, softcap, causal, prefix, documents, True, True)
        ctx.save_for_backward(q, k, v, slopes, prefix, documents, out, rest, lse)
        ctx.plain = scale, softcap, causal
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)                   # no tensor of zeros for the gradient that lse does not have
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 9
        q, k, v, slopes, prefix, documents, out, rest, lse = ctx.saved_tensors
        scale, softcap, causal = ctx.plain
        need_q, need_k, need_v, need_slopes = ctx.needs_input_grad[:4]
        lib = _backend.load()
        b, sq, hq, d = q.shape
        sk, hk, dv = k.shape[1], k.shape[2], v.shape[3]
        dev = q.device
        dout = _unit(dout)
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if need_q else None
        dk = dv_ = dslopes = None
        if need_k or need_v:
            dk, dv_ = torch.empty(k.shape, dtype=q.dtype, device=dev), torch.empty(v.shape, dtype=q.dtype, device=dev)
        if need_slopes:
            dslopes = torch.empty(slopes.shape, dtype=torch.float32, device=dev)
        code = _DTYPE_CODE[q.dtype]
        nbytes = lib.flk_attention_backward_workspace_bytes(b, sq, sk, hq, hk, d, dv, need_slopes, documents is not None, code)
        ws = _workspace(nbytes, dev)
        with _current(dev):
            rc = lib.flk_attention_backward(
                *_bsh(q), *_bsh(k), *_bsh(v), out.data_ptr(), _ptr(rest), lse.data_ptr(), *_bsh(dout), b, sq, sk, hq, hk, d, dv, scale, softcap,
                _ptr(slopes), causal, _ptr(prefix), _ptr(documents), documents.stride(0) if documents is not None else 0,
                _ptr(dq), _ptr(dk), _ptr(dv_), _ptr(dslopes), code, _ptr(ws), nbytes, _stream_handle(dev))
        _backend.raise_for_status(rc, "flk_attention_backward")
        return dq, dk if need_k else None, dv_ if need_v else None, dslopes, None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False, scale: Optional[float] = None,
              softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, prefix: Optional[torch.Tensor] = None,
              documents: Optional[torch.Tensor] = None, return_lse: bool = False
              ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Softmax-weighted sums of ``v`` (see the module's formulas), matrix-free, with gradients.

    Parameters
    ----------
    q : (batch, queries, heads, d), or a matrix (queries, d).
    k : (batch, keys, key heads, d), or a matrix (keys, d).  Each key head serves ``heads / key heads`` consecutive query heads.
    v : (batch, keys, key heads, dv), or a matrix (keys, dv).
        GPU tensors of one type: float32, float16 or bfloat16; d and dv up to 128; any strides (a tensor whose values
        within a row are not next to each other is copied first).
    causal : a row sees keys up to its own position only.
    scale : factor of the inner products, ``1 / sqrt(d)`` by default, at most 1e18 in size.
    softcap : cap of the scores, 0 for none; from 1e-20 to 1e20, or to 4096 for 16-bit data (whose scores would lose digits to a
        larger one).
    slopes : float32, one per query head: decay of the score with the distance between a row's and a key's position.
    prefix : (batch,) whole numbers, with ``causal`` only: the first ``prefix[b]`` keys are seen by every row.
    documents : (batch, keys) whole numbers of at most 32 bits: a row sees keys with its own number only, and nothing if that is negative
        (padding).  Needs at least as many keys as queries.  Rows of one document that lie together are found without
        reading the others.
    return_lse : also return the logarithm of every row's sum, float32 of shape (batch, heads, queries), or (queries,) for
        matrices; minus infinity for a row that sees nothing.  It is not differentiable.

    Returns a new contiguous tensor (batch, queries, heads, dv), or (queries, dv).  Differentiable (once) in q, k, v and
    slopes; gradients of shared key heads are summed over the heads that share them.  The call is asynchronous on the
    current stream and can be captured into a graph; to capture its backward pass, first let go of every eager result that
    was computed from the same leaves (torch ties a leaf's gradient to the stream of the first graph alive, and
    capturing across streams that way ends the process).
    """
    matrix = isinstance(q, torch.Tensor) and q.dim() == 2
    if matrix:
        for t, name in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or t.dim() != 2:
                raise ValueError(f"{name} must be a matrix like q")
        q, k, v = q[None, :, None], k[None, :, None], v[None, :, None]
    _check_operands("attention", q, k, v)
    b, sq, hq, d = q.shape
    sk = k.shape[1]
    scale, softcap, slopes = _check_score("attention", hq, scale, softcap, slopes, d)
    if prefix is not None:
        if not causal:
            raise ValueError("prefix belongs to a causal mask")
        prefix = _check_whole(prefix, "prefix", (b,)).contiguous()
    if documents is not None:
        if sq > sk:
            raise ValueError(f"documents need every query to stand at a key's position, got {sq} queries and {sk} keys")
        documents = _check_whole(documents, "documents", (b, sk))
    _check_devices("attention", q, k, v, slopes, prefix, documents)
    q, k, v = _unit(q), _unit(k), _unit(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (slopes is not None and slopes.requires_grad)):
        out, lse = _AttentionFn.apply(q, k, v, slopes, scale, softcap, bool(causal), prefix, documents)
    else:
        out, _, lse = _forward(q, k, v, slopes, scale, softcap, bool(causal), prefix, documents, return_lse)
    if matrix:
        out, lse = out[0, :, 0], lse[0, 0] if return_lse else None
    return (out, lse) if return_lse else out


def cached_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *,
                     scale: Optional[float] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``attention`` of the newest tokens of sequences of different lengths over their cached keys and values.

    Parameters
    ----------
    q : (batch, tokens, heads, d), or (batch, heads, d) for one token each.
    k_cache, v_cache : (batch, capacity, key heads, d) and (batch, capacity, key heads, dv), the new tokens' keys and values
        already written.  Types, sizes and strides as for ``attention``; what lies behind a sequence's end is not read.
    lengths : (batch,) whole numbers: keys each sequence has, new tokens included; values outside [0, capacity] count as
        the nearest of the two.  Token t of n stands at position ``lengths[b] - n + t`` and sees the keys up to it.
    scale, softcap, slopes : as for ``attention``.

    Returns a new contiguous tensor (batch, tokens, heads, dv), or (batch, heads, dv); a token whose position is negative is
    zero.  Not differentiable.  Asynchronous, and the lengths are read on the GPU: a captured call follows them.
    """
    single = isinstance(q, torch.Tensor) and q.dim() == 3
    if single:
        q = q[:, None]
    _check_operands("cached_attention", q, k_cache, v_cache)
    b, t, hq, d = q.shape
    capacity, hk, dv = k_cache.shape[1], k_cache.shape[2], v_cache.shape[3]
    scale, softcap, slopes = _check_score("cached_attention", hq, scale, softcap, slopes, d)
    lengths = _check_whole(lengths, "lengths", (b,)).contiguous()
    _check_devices("cached_attention", q, k_cache, v_cache, lengths, slopes)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k_cache, v_cache, slopes)):
        raise RuntimeError("cached_attention has no gradient: call attention, or detach its inputs")
    q, k_cache, v_cache = _unit(q), _unit(k_cache), _unit(v_cache)
    lib = _backend.load()
    out = torch.empty((b, t, hq, dv), dtype=q.dtype, device=q.device)
    nbytes = lib.flk_attention_cached_workspace_bytes(b, t, capacity, hq, hk, dv)
    ws = _workspace(nbytes, q.device)
    with _current(q.device):
        rc = lib.flk_attention_cached(*_bsh(q), *_bsh(k_cache), *_bsh(v_cache), lengths.data_ptr(), b, t, capacity, hq, hk, d, dv,
                                      scale, softcap, _ptr(slopes), out.data_ptr(), _DTYPE_CODE[q.dtype], _ptr(ws), nbytes,
                                      _stream_handle(q.device))
    _backend.raise_for_status(rc, "flk_attention_cached")
    return out[:, 0] if single else out
