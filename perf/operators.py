"""Timed cases of the normalised products: attention, attention over a cache, and the layer norm.

``own`` chooses between the library's operators and the same mathematics in elementary torch operations (products,
sums, exp, comparisons), which compute in 32 bits and round once at the end.

    attention          x = scale * q.k,  x <- cap * tanh(x / cap),  x <- x - slope * |i - j|,
                       out = sum_j softmax_j(x, visible j) v_j;  a row that sees nothing is zero
    cached_attention   the same for the newest tokens of sequences whose keys and values lie in a cache
    layer_norm         y = (x - mean) / sqrt(var + eps) * w + b, by rows
"""
import math

import torch

own = False

_TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attention_case(name, **more):
    case = {"op": "attention", "dtype": "bf16", "train": False, "b": 1, "sq": 64, "sk": 64, "hq": 8, "hk": 8, "d": 64,
            "dv": 64, "causal": False, "prefix": False, "docs": 0, "slopes": False, "cap": 0.0}
    return {**case, **more, **({"name": name} if name else {})}


def _cached_case(name, **more):
    case = {"op": "cached", "dtype": "bf16", "b": 1, "t": 1, "capacity": 1024, "lo": 1.0, "hi": 1.0, "hq": 8, "hk": 8,
            "d": 64, "slopes": False, "cap": 0.0}
    return {**case, **more, **({"name": name} if name else {})}


def _norm_case(name, **more):
    case = {"op": "norm", "dtype": "f32", "train": False, "rows": 1, "d": 784, "affine": True}
    return {**case, **more, **({"name": name} if name else {})}


def listed():
    return [
        # kernel smoothing on the benchmark's own features: 1e5 rows of 28 features against 2000 centres, 4 outputs
        _attention_case("smooth_f32", dtype="f32", sq=100_000, sk=2000, hq=1, hk=1, d=28, dv=4),
        # a handful of short texts scored in one call: latency counts
        _attention_case("short_f16", dtype="f16", b=4, sq=77, sk=77, causal=True),
        # one long prompt, shared key heads
        _attention_case("prompt_bf16", sq=8192, sk=8192, hq=32, hk=8, d=128, dv=128, causal=True),
        # a training step on packed documents with padding behind the last one, capped scores
        _attention_case("train_docs_bf16", train=True, b=2, sq=4096, sk=4096, hq=32, hk=8, d=128, dv=128, causal=True,
                        docs=6, cap=30.0),
        # a training step with a visible prefix and a learned decay with the distance, odd length
        _attention_case("train_prefix_f16", dtype="f16", train=True, b=4, sq=1023, sk=1023, hq=12, hk=12, causal=True,
                        prefix=True, slopes=True),
        # a training step in single precision between two sets of different, odd sizes
        _attention_case("train_cross_f32", dtype="f32", train=True, b=2, sq=1000, sk=1537, hq=8, hk=2, d=80, dv=80),
        # one user's next token over a short cache: latency counts
        _cached_case("token_f16", dtype="f16", hi=0.5),
        # a full batch of sequences of all lengths, shared key heads
        _cached_case("batch_bf16", b=64, capacity=16384, lo=0.02, hq=32, hk=8, d=128),
        # four tokens at once over one very long cache, decay with the distance and capped scores
        _cached_case("long_bf16", t=4, capacity=131072, hi=0.93, hq=32, hk=4, d=128, slopes=True, cap=50.0),
        # one row of features before it is predicted on
        _norm_case("row_f16", dtype="f16"),
        # the benchmark's own matrix of 1e6 rows with 28 features
        _norm_case("rows_f32", rows=1_000_000, d=28),
        # a training step over the hidden rows of a large batch
        _norm_case("train_bf16", dtype="bf16", train=True, rows=16384, d=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "train", "train", "cached", "cached", "norm", "norm"])
    if op == "norm":
        dtype = rng.choice(["f32", "bf16", "f16", "f64"])
        d = _log(rng, 5, 16384)
        rows = _log(rng, 1, min(1_000_000, 60_000_000 // d))
        return _norm_case(None, dtype=dtype, train=rng.random() < 0.5, rows=rows, d=d, affine=rng.random() < 0.8)
    dtype = rng.choice(["bf16", "f16", "f32"])
    hk = rng.choice([1, 2, 3, 4, 8])
    hq = hk * rng.choice([1, 1, 2, 4, 7, 8])
    d = rng.choice([_log(rng, 8, 128), 64, 128, 32, 96])
    slopes = rng.random() < 0.3
    cap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if op == "cached":
        capacity = _log(rng, 200, 65536)
        b = _log(rng, 1, max(1, min(64, 60_000_000 // (capacity * hk))))
        return _cached_case(None, dtype=dtype, b=b, t=rng.choice([1, 1, 1, 2, 5, 8]), capacity=capacity,
                            lo=rng.uniform(0.05, 0.9), hi=rng.uniform(0.3, 1.0), hq=hq, hk=hk, d=d, slopes=slopes, cap=cap)
    pairs = (4.0e7 if dtype == "f32" else 4.0e8) * (0.3 if op == "train" else 1.0)
    sk = _log(rng, 17, 6000)
    causal = rng.random() < 0.6
    sq = sk if causal else _log(rng, 1, 6000)
    most = max(1, int(pairs / (hq * sq * sk)))
    while hq * sq * sk > pairs:
        sq, sk = sq // 2 + 1, sk // 2 + 1
    return _attention_case(None, dtype=dtype, train=op == "train", b=_log(rng, 1, min(8, most)), sq=sq, sk=sk, hq=hq, hk=hk,
                           d=d, dv=d, causal=causal, prefix=causal and rng.random() < 0.3,
                           docs=rng.choice([0, 0, 3, 7]) if sq == sk and sk >= 64 else 0, slopes=slopes, cap=cap)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _slopes(hq, dev):
    """Decays from 1/2 down to 1/256 over the heads."""
    return torch.exp2(-1.0 - 7.0 * torch.arange(hq, dtype=torch.float32, device=dev) / max(1, hq - 1))


def _documents(b, s, docs, gen, dev):
    """``docs`` documents of random lengths a row, the places behind the last one (a sixteenth of the row) padding (-1)."""
    used = s - s // 16
    cuts = torch.rand(b, docs - 1, generator=gen, device=dev).mul_(used).long()
    ids = torch.zeros(b, s, dtype=torch.int32, device=dev)
    ids.scatter_add_(1, cuts, torch.ones_like(cuts, dtype=torch.int32))
    ids = ids.cumsum(1).to(torch.int32)
    ids[:, used:] = -1
    return ids


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(scale).to(dtype)

    state = {"case": dict(case)}
    if case["op"] == "norm":
        state["x"] = (normal(case["rows"], case["d"], scale=1.5) + 0.25).to(dtype)
        state["w"] = (normal(case["d"], scale=0.2) + 1).to(dtype) if case["affine"] else None
        state["bias"] = normal(case["d"], scale=0.2) if case["affine"] else None
        if case["train"]:
            state["dout"] = normal(case["rows"], case["d"])
            for n in ("x", "w", "bias"):
                if state[n] is not None:
                    state[n].requires_grad_()
        return state
    b, hq, hk, d = case["b"], case["hq"], case["hk"], case["d"]
    state["slopes"] = _slopes(hq, dev) if case["slopes"] else None
    if case["op"] == "cached":
        cap, t = case["capacity"], case["t"]
        state["q"] = normal(b, t, hq, d, scale=1.5)
        state["k"], state["v"] = normal(b, cap, hk, d), normal(b, cap, hk, d)
        lens = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        state["lengths"] = lens[torch.randperm(b, generator=gen, device=dev)].contiguous()
        return state
    sq, sk = case["sq"], case["sk"]
    state["q"], state["k"] = normal(b, sq, hq, d, scale=1.5), normal(b, sk, hk, d)
    state["v"] = normal(b, sk, hk, case["dv"])
    state["prefix"] = (torch.rand(b, generator=gen, device=dev) * (sk // 2)).to(torch.int32) if case["prefix"] else None
    state["documents"] = _documents(b, sk, case["docs"], gen, dev) if case["docs"] else None
    if case["train"]:
        state["dout"] = normal(b, sq, hq, case["dv"])
        for n in ("q", "k", "v", "slopes"):
            if state[n] is not None:
                state[n].requires_grad_()
    return state


def _lengths(case):
    """Lengths spread evenly over [lo, hi] of the capacity (prepare shuffles them by its seed)."""
    b, cap = case["b"], case["capacity"]
    lo, hi = min(case["lo"], case["hi"]), case["hi"]
    return [max(1, int(cap * (hi if b == 1 else lo + (hi - lo) * i / (b - 1)))) for i in range(b)]


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    if op == "cached":
        return _own_cached(state) if own else _plain_cached(state)
    return _own_attention(state) if own else _plain_attention(state)


def _own_attention(state):
    from falkon_amd import attention
    case = state["case"]
    out = attention(state["q"], state["k"], state["v"], causal=case["causal"], prefix=state["prefix"],
                    documents=state["documents"], slopes=state["slopes"], softcap=case["cap"])
    if not case["train"]:
        return {"out": out}
    names = [n for n in ("q", "k", "v", "slopes") if state[n] is not None]
    grads = torch.autograd.grad(out, [state[n] for n in names], state["dout"])
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _own_cached(state):
    from falkon_amd import cached_attention
    return {"out": cached_attention(state["q"], state["k"], state["v"], state["lengths"], slopes=state["slopes"],
                                    softcap=state["case"]["cap"])}


def _own_norm(state):
    from falkon_amd import layer_norm
    y = layer_norm(state["x"], state["w"], state["bias"])
    if not state["case"]["train"]:
        return {"out": y}
    names = [n for n in ("x", "w", "bias") if state[n] is not None]
    grads = torch.autograd.grad(y, [state[n] for n in names], state["dout"])
    return {"out": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _by_key_head(x, hk):
    """(b, s, h, d) -> (b, hk, g * s, d) in 32 bits: the heads that share a key head, one after the other."""
    b, s, h, d = x.shape
    return x.detach().float().reshape(b, s, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, (h // hk) * s, d)


def _by_query(x, s):
    """(b, hk, g * s, d) -> (b, s, h, d)."""
    b, hk, gs, d = x.shape
    return x.reshape(b, hk, gs // s, s, d).permute(0, 3, 1, 2, 4).reshape(b, s, hk * (gs // s), d)


def _plain_softmax(x, visible):
    x = x.masked_fill_(~visible, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp_min(1e-37))


def _plain_attention(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    b, sq, hq, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    g = hq // hk
    scale = 1.0 / math.sqrt(d)
    pos = torch.arange(sk - sq, sk, device=q.device).view(1, sq, 1)
    key = torch.arange(sk, device=q.device).view(1, 1, sk)
    visible = (key <= pos) if case["causal"] else torch.ones(1, sq, sk, dtype=torch.bool, device=q.device)
    if state["prefix"] is not None:
        visible = visible | (key < state["prefix"].view(b, 1, 1))
    if state["documents"] is not None:
        ids = state["documents"]
        visible = visible & (ids[:, sk - sq:].unsqueeze(2) == ids.unsqueeze(1)) & (ids >= 0).unsqueeze(1)
    visible = visible.view(-1, 1, 1, sq, sk)
    qf, kf, vf = _by_key_head(q, hk), _by_key_head(k, hk), _by_key_head(v, hk)
    x = (qf @ kf.transpose(2, 3)).mul_(scale).view(b, hk, g, sq, sk)
    t = None
    if case["cap"]:
        t = x.div_(case["cap"]).tanh_()
        x = t * case["cap"]
    dist = (pos - key).abs().float().view(1, 1, 1, sq, sk)
    if state["slopes"] is not None:
        x = x - state["slopes"].detach().view(1, hk, g, 1, 1) * dist
    p = _plain_softmax(x, visible).view(b, hk, g * sq, sk)
    out = {"out": _by_query(p @ vf, sq).to(q.dtype)}
    if not case["train"]:
        return out
    do = _by_key_head(state["dout"], hk)
    out["dv"] = _by_query(p.transpose(2, 3) @ do, sk).to(q.dtype)
    dp = do @ vf.transpose(2, 3)
    ds = p.mul_(dp.sub_((p * dp).sum(-1, keepdim=True))).view(b, hk, g, sq, sk)
    if state["slopes"] is not None:
        out["dslopes"] = -(ds * dist).sum((0, 3, 4)).reshape(hq)
    if t is not None:
        ds = ds.mul_(1 - t * t)
    ds = ds.view(b, hk, g * sq, sk)
    out["dq"] = _by_query((ds @ kf).mul_(scale), sq).to(q.dtype)
    out["dk"] = _by_query((ds.transpose(2, 3) @ qf).mul_(scale), sk).to(q.dtype)
    return out


def _plain_cached(state):
    case = state["case"]
    q, k, v, lens = state["q"], state["k"], state["v"], state["lengths"]
    b, t, hq, d = q.shape
    cap, hk = k.shape[1], k.shape[2]
    g = hq // hk
    qf, kf, vf = _by_key_head(q, hk), _by_key_head(k, hk), _by_key_head(v, hk)
    pos = lens.long().view(b, 1, 1) - t + torch.arange(t, device=q.device).view(1, t, 1)
    key = torch.arange(cap, device=q.device).view(1, 1, cap)
    x = (qf @ kf.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(b, hk, g, t, cap)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    if state["slopes"] is not None:
        x = x - state["slopes"].view(1, hk, g, 1, 1) * (pos - key).abs().float().view(b, 1, 1, t, cap)
    p = _plain_softmax(x, (key <= pos).view(b, 1, 1, t, cap)).view(b, hk, g * t, cap)
    return {"out": _by_query(p @ vf, t).to(q.dtype)}


def _plain_norm(state):
    wide = torch.float64 if state["x"].dtype == torch.float64 else torch.float32
    x = state["x"].detach().to(wide)
    dtype = state["x"].dtype
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(c.square().mean(-1, keepdim=True) + 1e-5)
    xhat = c * rstd
    w = state["w"].detach().to(wide) if state["w"] is not None else None
    y = xhat if w is None else xhat * w + state["bias"].detach().to(wide)
    out = {"out": y.to(dtype)}
    if not state["case"]["train"]:
        return out
    dy = state["dout"].to(wide)
    gw = dy if w is None else dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    out["dx"] = dx.to(dtype)
    if w is not None:
        out["dw"] = (dy * xhat).sum(0).to(dtype)
        out["dbias"] = dy.sum(0).to(dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(state)
        return _exact_attention(state)


def _exact_norm(state):
    x = state["x"].double()
    n = x.shape[1]
    mean = x.sum(1) / n
    var = (x * x).sum(1) / n - mean * mean
    inv = 1 / torch.sqrt(var + 1e-5)
    z = (x - mean[:, None]) * inv[:, None]
    w = torch.ones(n, dtype=torch.float64, device=x.device) if state["w"] is None else state["w"].double()
    y = z * w + (0.0 if state["bias"] is None else state["bias"].double())
    if not state["case"]["train"]:
        return {"out": y}
    dy = state["dout"].double()
    dz = dy * w
    dx = (n * dz - dz.sum(1, keepdim=True) - z * (dz * z).sum(1, keepdim=True)) * (inv[:, None] / n)
    out = {"out": y, "dx": dx}
    if state["w"] is not None:
        out["dw"], out["dbias"] = (dy * z).sum(0), dy.sum(0)
    return out


def _exact_attention(state):
    """Sequence by sequence and head by head, through the logarithm of the sum."""
    case = state["case"]
    cached, train = case["op"] == "cached", case.get("train", False)
    q, k, v, slopes = state["q"], state["k"], state["v"], state["slopes"]
    b, sq, hq, d = q.shape
    group = hq // k.shape[2]
    lens = state["lengths"].tolist() if cached else [k.shape[1]] * b
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    out = {"out": torch.zeros(b, sq, hq, v.shape[3], dtype=torch.float64, device=q.device)}
    if train:
        out["dq"], out["dk"], out["dv"] = zeros(q), zeros(k), zeros(v)
        if slopes is not None:
            out["dslopes"] = zeros(slopes)
    for i in range(b):
        n = lens[i]
        at = torch.arange(n - sq, n, device=q.device)[:, None]
        key = torch.arange(n, device=q.device)[None, :]
        seen = torch.ones(sq, n, dtype=torch.bool, device=q.device)
        if cached or case["causal"]:
            seen = key <= at
        if not cached and state["prefix"] is not None:
            seen = seen | (key < state["prefix"][i])
        if not cached and state["documents"] is not None:
            ids = state["documents"][i]
            mine = ids[n - sq:]
            seen = seen & (mine[:, None] == ids[None, :]) & (mine[:, None] >= 0)
        for h in range(hq):
            qh, kh, vh = q[i, :, h].double(), k[i, :n, h // group].double(), v[i, :n, h // group].double()
            raw = qh @ kh.T / math.sqrt(d)
            s = torch.tanh(raw / case["cap"]) * case["cap"] if case["cap"] else raw
            if slopes is not None:
                s = s - slopes[h].double() * (at - key).abs()
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse))
            o = p @ vh
            out["out"][i, :, h] = o
            if not train:
                continue
            do = state["dout"][i, :, h].double()
            out["dv"][i, :, h // group] += p.T @ do
            ds = p * (do @ vh.T - (do * o).sum(1, keepdim=True))
            if slopes is not None:
                out["dslopes"][h] -= (ds * (at - key).abs()).sum()
            if case["cap"]:
                ds = ds / torch.cosh(raw / case["cap"]) ** 2
            out["dq"][i, :, h] = ds @ kh / math.sqrt(d)
            out["dk"][i, :, h // group] += ds.T @ qh / math.sqrt(d)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    es = _SIZES[case["dtype"]]
    if case["op"] == "norm":
        n, w = case["rows"] * case["d"], (2 * case["d"] if case["affine"] else 0)
        if not case["train"]:
            return {"bytes": es * (2 * n + w), "flops": 8 * n}
        return {"bytes": es * (4 * n + 2 * w), "flops": 20 * n}     # x and dy read, y and dx written
    d, hq, hk = case["d"], case["hq"], case["hk"]
    if case["op"] == "cached":
        lens = _lengths(case)
        rows = case["b"] * case["t"] * hq
        return {"bytes": es * (2 * sum(lens) * hk * d + 2 * rows * d) + 4 * case["b"],
                "flops": 4 * sum(lens) * case["t"] * hq * d}
    b, sq, sk, dv = case["b"], case["sq"], case["sk"], case["dv"]
    rows, keys = b * sq * hq, b * sk * hk
    size = es * (rows * d + keys * (d + dv) + rows * dv)
    if case["docs"]:      # random cuts: the documents' squares sum to 2 s^2 / (docs + 1) on average
        used = sk - sk // 16
        pairs = 2.0 * used * used / (case["docs"] + 1)
        pairs = pairs / 2 if case["causal"] else pairs
    elif case["causal"]:  # sq == sk; a prefix of s / 4 on average adds the upper half of its square
        pairs = sk * (sk + 1) / 2 + (sk * sk / 24 if case["prefix"] else 0)
    else:
        pairs = sq * sk
    flops = 2.0 * b * hq * pairs * (d + dv)
    if not case["train"]:
        return {"bytes": size, "flops": flops}
    # forward: two products; backward: the scores again, and four more. q, k, v, out and dout read, three gradients written
    return {"bytes": 2 * size + es * rows * dv, "flops": flops * 3.5}
