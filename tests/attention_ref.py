"""Attention and its gradients from the definition, in 64 bits on the CPU, with a bound of the error that arithmetic in the
tested type allows for every value.

With u = 2^-24 (float32 arithmetic) and e half a step of the data's type relative to a value (0 for float32 data, whose steps
are already counted by u):

    score      dx  = u (d + 16) scale sum|q||k|  (+ 16 u cap) (+ 4 u slope dist)      d products, summed in any order
    weight     a factor exp(+-dx_i) in p and in its row's sum: 2 max_j dx_ij relative, e for the rounding of p before the
               second product, u (n + 32) for the sums over n keys
    out        (2 dx + e + u (n + 32)) sum p|v| + e |out|
    dS         p (error of dP - delta) + |dS| (4 dx + 2 e + u (n + 32)), where
               dP has u (dv + 16) sum|dout||v| and delta sum|dout| (error of out) + u (dv + 16) sum|dout||out|
    dq         scale sum_j |k| (error of dS) + scale u (n + 32) sum |dS||k| + e |dq|;  dk, dv, dslopes likewise
    float16    half a step of its smallest values, 2^-25, for every weight, dS and result

The cap's derivative 1 - tanh^2 adds 64 u |dS|.
"""
import math

import torch

U = 2.0 ** -24


def visible(b, sq, sk, causal=False, prefix=None, documents=None):
    pos = torch.arange(sk - sq, sk)[None, :, None]
    key = torch.arange(sk)[None, None, :]
    see = (key <= pos) if causal else torch.ones(1, sq, sk, dtype=torch.bool)
    see = see.expand(b, sq, sk)
    if prefix is not None:
        see = see | (key < prefix.cpu().long()[:, None, None])
    if documents is not None:
        ids = documents.cpu().long()
        mine = ids[:, sk - sq:] if sq else ids[:, :0]
        see = see & (mine[:, :, None] == ids[:, None, :]) & (mine[:, :, None] >= 0)
    return see


def reference(q, k, v, dout=None, scale=None, softcap=0.0, slopes=None, **mask):
    """{name: (value, bound)} of out, lse and, with dout, dq, dk, dv and dslopes."""
    dtype = q.dtype
    e = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    b, sq, hq, d = q.shape
    sk, hk, dv = k.shape[1], k.shape[2], v.shape[3]
    g = hq // hk
    scale = 1 / math.sqrt(d) if scale is None else scale
    see = visible(b, sq, sk, **mask)[:, None]                                   # b 1 sq sk
    hidden = ~see.any(2, keepdim=True).transpose(2, 3)                          # keys that no row sees: b 1 sk 1
    qh = q.permute(0, 2, 1, 3)
    kh, vh = (t.permute(0, 2, 1, 3).masked_fill(hidden, 0.0).repeat_interleave(g, 1) for t in (k, v))
    x = scale * qh @ kh.transpose(2, 3)
    dx = U * (d + 16) * abs(scale) * (qh.abs() @ kh.abs().transpose(2, 3))
    tanh = None
    if softcap:
        tanh = torch.tanh(x / softcap)
        x, dx = softcap * tanh, dx + 16 * U * softcap
    dist = (torch.arange(sk - sq, sk)[:, None] - torch.arange(sk)[None, :]).abs().double()
    if slopes is not None:
        decay = slopes.detach().double().cpu()[None, :, None, None] * dist
        x, dx = x - decay, dx + 4 * U * decay.abs()
    x = x.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(x, 3, keepdim=True) if sk else torch.full((b, hq, sq, 1), -math.inf, dtype=torch.float64)
    p = torch.exp(x - lse.masked_fill(torch.isinf(lse), 0.0))
    dx = dx.masked_fill(~see, 0.0).amax(3, keepdim=True) if sk else torch.zeros(b, hq, sq, 1, dtype=torch.float64)
    seen = see.double().expand(b, hq, sq, sk)
    o = p @ vh
    rel = 2 * dx + e + U * (sk + 32)
    do_ = rel * (p @ vh.abs()) + tiny * (seen @ vh.abs()) + e * o.abs() + tiny
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    res = {"out": (back(o), back(do_)),
           "lse": (lse[..., 0], (dx + U * (sk + 32 + 4 * lse.abs().masked_fill(torch.isinf(lse), 0.0)))[..., 0])}
    if dout is None:
        return res
    n = max(sq, sk) * g + 32
    dd = dout.detach().double().cpu().permute(0, 2, 1, 3)
    dp = dd @ vh.transpose(2, 3)
    delta = (dd * o).sum(3, keepdim=True)
    ddp = U * (dv + 16) * (dd.abs() @ vh.abs().transpose(2, 3))
    ddelta = (dd.abs() * do_).sum(3, keepdim=True) + U * (dv + 16) * (dd * o).abs().sum(3, keepdim=True)
    ds = p * (dp - delta)
    dds = p * (ddp + ddelta) + ds.abs() * (4 * dx + 2 * e + U * (n + 64)) + tiny * seen

    def shared(t):
        return t.reshape(b, hk, g, sk, -1).sum(2).permute(0, 2, 1, 3)
    dvv = shared(p.transpose(2, 3) @ dd)
    pd = p * (4 * dx + e + U * n) + tiny * seen
    res["dv"] = dvv, shared(pd.transpose(2, 3) @ dd.abs()) + e * dvv.abs() + tiny
    if slopes is not None:
        res["dslopes"] = (-(ds * dist).sum((0, 2, 3)), ((dds + U * n * ds.abs()) * dist).sum((0, 2, 3)))
    if tanh is not None:
        dds = dds * (1 - tanh ** 2) + 64 * U * ds.abs()
        ds = ds * (1 - tanh ** 2)
    dds = dds + U * n * ds.abs()
    dq = scale * back(ds @ kh)
    res["dq"] = dq, abs(scale) * back(dds @ kh.abs()) + e * dq.abs() + tiny
    dk = scale * shared(ds.transpose(2, 3) @ qh)
    res["dk"] = dk, abs(scale) * shared(dds.transpose(2, 3) @ qh.abs()) + e * dk.abs() + tiny
    return res


def check(got, want, names):
    for name in names:
        g = got[name].detach().double().cpu()
        value, bound = want[name]
        assert g.shape == value.shape, (name, g.shape, value.shape)
        same = (torch.isinf(value) & (g == value)) | (torch.isnan(value) & torch.isnan(g))
        off = torch.where(same, torch.zeros_like(value), (g - value).abs())
        worst = (off / (bound + 1e-30)).max().item() if value.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.3g} times its bound (largest difference {off.max().item():.3g})"
