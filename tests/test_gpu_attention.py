"""``attention`` and ``cached_attention`` against their definition in 64 bits, within bounds derived in ``attention_ref``."""
import math

import pytest
import torch

import falkon_amd
from falkon_amd import attention, cached_attention, layer_norm

from attention_ref import check, reference

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _make(b, sq, sk, hq, hk, d, dv, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, sq, hq, d, generator=g) * 1.3).to(dtype).to(DEV)
    k = torch.randn(b, sk, hk, d, generator=g).to(dtype).to(DEV)
    v = torch.randn(b, sk, hk, dv, generator=g).to(dtype).to(DEV)
    do = torch.randn(b, sq, hq, dv, generator=g).to(dtype).to(DEV)
    return q, k, v, do


def _run(q, k, v, do, slopes=None, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    s = slopes.detach().requires_grad_() if slopes is not None else None
    out, lse = attention(*leaves, slopes=s, return_lse=True, **kw)
    names = ["q", "k", "v"] + (["slopes"] if s is not None else [])
    grads = torch.autograd.grad(out, leaves + ([s] if s is not None else []), do)
    return {"out": out.detach(), "lse": lse, **{"d" + n: x for n, x in zip(names, grads)}}


def _check(q, k, v, do, slopes=None, **kw):
    got = _run(q, k, v, do, slopes, **kw)
    want = reference(q, k, v, do, slopes=slopes, **kw)
    check(got, want, [n for n in ("out", "lse", "dq", "dk", "dv", "dslopes") if n in got])
    plain = attention(q, k, v, slopes=slopes, **kw)
    assert torch.equal(plain.nan_to_num(7.0), got["out"].nan_to_num(7.0))
    return got


# (batch, queries, keys, heads, key heads, d, dv): single rows and keys, both sides of every tile and workgroup, head sizes on
# both sides of every padded size, odd ones (rows that are not aligned), d and dv that differ, shared heads
_SIZES = [(1, 1, 1, 1, 1, 1, 1), (1, 1, 200, 2, 1, 8, 8), (2, 3, 5, 3, 3, 7, 4), (1, 128, 64, 2, 2, 32, 32), (2, 129, 65, 4, 2, 33, 64),
          (1, 127, 255, 6, 2, 64, 64), (1, 130, 130, 2, 1, 96, 65), (1, 257, 192, 2, 2, 128, 128), (3, 31, 33, 7, 1, 80, 128),
          (1, 300, 77, 1, 1, 28, 1), (1, 65, 320, 4, 4, 127, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", _SIZES)
@pytest.mark.parametrize("causal", [False, True])
def test_values_and_gradients(size, dtype, causal):
    _check(*_make(*size, dtype), causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["plain", "causal cap", "prefix", "documents", "decay"])
@pytest.mark.parametrize("sq,sk,d", [(100, 1500, 64), (700, 1100, 128), (1000, 1000, 50)])
def test_divided_keys(dtype, kind, sq, sk, d):
    """Few heads and many keys: a tile's keys, and the queries of a tile of keys, are divided over workgroups."""
    q, k, v, do = _make(1, sq, sk, 2, 1, d, d, dtype, seed=21)
    kw = dict(causal=kind not in ("plain", "decay"))
    if "cap" in kind:
        kw["softcap"] = 4.0
    if kind == "prefix":
        kw["prefix"] = torch.tensor([170], device=DEV)
    if kind == "documents":
        kw["documents"] = _ids("long", 1, sk)
        kw["documents"][:, :200] = -1
    _check(q, k, v, do, torch.tensor([0.01, 0.2], device=DEV) if kind == "decay" else None, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["plain", "causal cap", "prefix decay", "documents", "documents cap decay"])
@pytest.mark.parametrize("d", [28, 64, 81, 128])
def test_many_workgroups(dtype, kind, d):
    """Enough heads to fill the chip: no tile's keys are divided over workgroups, which the sizes above may be."""
    b, s, hq, hk = 16, 135, 16, 8
    q, k, v, do = _make(b, s, s, hq, hk, d, d, dtype, seed=20)
    kw = dict(causal=kind != "plain")
    if "cap" in kind:
        kw["softcap"] = 4.0
    if "prefix" in kind:
        kw["prefix"] = torch.arange(b, device=DEV) * 9
    if "documents" in kind:
        kw["documents"] = _ids("sorted", b, s)
    slopes = torch.arange(hq, device=DEV).float() / 40 if "decay" in kind else None
    _check(q, k, v, do, slopes, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("cap,slope", [(0.0, True), (2.0, False), (30.0, True), (4096.0, False)])
@pytest.mark.parametrize("d", [16, 64, 72, 128])
def test_capped_and_decaying_scores(dtype, causal, cap, slope, d):
    q, k, v, do = _make(2, 150, 170, 4, 2, d, d, dtype, seed=1)
    slopes = torch.tensor([0.5, 0.0, 0.03, 0.004], device=DEV) if slope else None
    _check(q, k, v, do, slopes, causal=causal, softcap=cap, scale=0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,sk", [(200, 200), (70, 200), (200, 70)])
def test_prefix(dtype, sq, sk):
    q, k, v, do = _make(6, sq, sk, 2, 1, 40, 40, dtype, seed=2)
    prefix = torch.tensor([0, 1, 64, 69, 1000, -5], device=DEV)
    _check(q, k, v, do, causal=True, prefix=prefix)
    _check(q, k, v, do, causal=True, prefix=prefix.int(), softcap=10.0)


def _ids(kind, b, s):
    g = torch.Generator().manual_seed(4)
    if kind == "sorted":
        ids = torch.randint(0, 5, (b, s), generator=g).sort(1).values
        ids[:, -s // 10:] = -1
    elif kind == "shuffled":
        ids = torch.randint(-1, 4, (b, s), generator=g)
    elif kind == "long":                                    # documents of about 150 positions, numbers far apart
        ids = (torch.arange(s) // 150 * 1_000_003).expand(b, s).clone()
    elif kind == "padded front":
        ids = torch.zeros(b, s, dtype=torch.int64)
        ids[:, :s // 3] = -7
    else:                                                   # nothing but padding
        ids = torch.full((b, s), -1)
    return ids.to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["sorted", "shuffled", "long", "padded front", "none"])
def test_documents(dtype, causal, kind):
    for sq, sk in ((333, 333), (100, 333)):
        q, k, v, do = _make(2, sq, sk, 2, 1, 48, 48, dtype, seed=3)
        ids = _ids(kind, 2, sk)
        got = _check(q, k, v, do, causal=causal, documents=ids)
        if kind == "none":
            assert not any(bool(got[n].any()) for n in ("out", "dq", "dk", "dv")) and bool(torch.isneginf(got["lse"]).all())
    _check(q, k, v, do, causal=causal, documents=ids.int()[:1].expand(2, sk))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_values_in_hidden_places(dtype):
    """What no row sees leaves no trace; what some rows see reaches those rows alone."""
    b, s = 1, 200
    q, k, v, do = _make(b, s, s, 2, 2, 64, 64, dtype, seed=5)
    ids = torch.zeros(b, s, dtype=torch.int32, device=DEV)
    ids[:, 60:130] = 1
    ids[:, 180:] = -1
    clean = _run(q, k, v, do, causal=True, documents=ids)
    for value in (float("nan"), float("inf"), -float("inf")):
        k2, v2, q2, do2 = k.clone(), v.clone(), q.clone(), do.clone()
        k2[:, 185], v2[:, 190], q2[:, 185], do2[:, 181] = value, value, value, value      # padding
        got = _run(q2, k2, v2, do2, causal=True, documents=ids)
        assert all(torch.equal(got[n], clean[n]) for n in clean)
        k3, v3 = k.clone(), v.clone()
        v3[:, 100], k3[:, 90] = value, float("nan")                                       # rows 90 .. 129 see one of them
        out = attention(q, k3, v3, causal=True, documents=ids)
        assert torch.equal(out[:, :90], clean["out"][:, :90]) and torch.equal(out[:, 130:], clean["out"][:, 130:])
        assert bool(out[:, 90:130].isnan().all())
        got = _run(q, k3, v3, do, causal=True, documents=ids)
        other = torch.ones(s, dtype=torch.bool, device=DEV)
        other[60:130] = False
        assert all(torch.equal(got[n][:, other], clean[n][:, other]) for n in ("dq", "dk", "dv"))
        q5, do5 = q.clone(), do.clone()
        q5[:, 70], do5[:, 100] = float("nan"), value        # keys 60 .. 70, and 60 .. 100, are seen by one of them
        got = _run(q5, k, v, do5, causal=True, documents=ids)
        assert bool(got["dk"][:, 60:101].isnan().all()) and bool(got["dv"][:, 60:101].isnan().all())
        other[60:130] = True
        other[60:101] = False
        assert all(torch.equal(got[n][:, other], clean[n][:, other]) for n in ("dk", "dv"))
        other[60:130] = True
        other[70] = other[100] = False
        assert torch.equal(got["dq"][:, other], clean["dq"][:, other]) and bool(got["dq"][:, [70, 100]].isnan().all())
    v4 = v.clone()
    v4[:, 150, :, 3], v4[:, 150, :, 4] = float("inf"), -float("inf")
    out = attention(q, k, v4, causal=True)
    assert bool(torch.isposinf(out[:, 150:, :, 3]).all()) and bool(torch.isneginf(out[:, 150:, :, 4]).all())
    assert bool(out[:, :150].isfinite().all()) and bool(out[:, 150:, :, 5:].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Heads before rows, one tensor cut into q, k and v, a batch that shares its keys, rows that start anywhere."""
    b, s, h, d = 2, 100, 3, 64
    g = torch.Generator().manual_seed(6)
    big = torch.randn(b, s, h, 3 * d, generator=g).to(dtype).to(DEV)
    do = torch.randn(b, s, h, d, generator=g).to(dtype).to(DEV)
    q, k, v = big.split(d, -1)
    want = {n: t for n, t in _check(q, k, v, do, causal=True).items()}
    for form in (lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), lambda t: t.permute(1, 2, 3, 0).contiguous().permute(3, 0, 1, 2),
                 lambda t: torch.nn.functional.pad(t, (1, 2))[..., 1:1 + d], lambda t: t.flip(0).flip(0)):
        got = _run(form(q), form(k), form(v), form(do), causal=True)
        assert all(torch.equal(got[n], want[n]) for n in want)
    one = k[:1].expand(b, s, h, d)
    _check(q, one, v[:, :, :1].expand(b, s, h, d), do[:, :, :, :1].expand(b, s, h, d), causal=True)
    k1 = k[:1].detach().requires_grad_()                    # the gradient of a broadcast input is summed over the batch
    got = torch.autograd.grad(attention(q, k1.expand(b, s, h, d), v), k1, do)[0]
    each = _run(q, one, v, do)["dk"].float().sum(0, keepdim=True)
    assert torch.allclose(got.float(), each, rtol=0.02, atol=1e-3)


@pytest.mark.gpu
def test_matrices_and_empty_shapes():
    g = torch.Generator().manual_seed(7)
    q, k, v = torch.randn(50, 28, generator=g).to(DEV), torch.randn(30, 28, generator=g).to(DEV), torch.randn(30, 3, generator=g).to(DEV)
    out, lse = attention(q, k, v, return_lse=True)
    want = reference(q[None, :, None], k[None, :, None], v[None, :, None])
    check({"out": out[None, :, None], "lse": lse[None, None]}, want, ("out", "lse"))
    assert torch.equal(attention(q, k, v), out)
    k.requires_grad_()
    assert torch.autograd.grad(attention(q, k, v).sum(), k)[0].shape == k.shape
    for b, sq, sk in ((0, 3, 3), (2, 0, 5), (2, 4, 0), (1, 0, 0)):
        qe, ke, ve, do = _make(b, sq, sk, 2, 1, 16, 24, torch.bfloat16)
        got = _run(qe, ke, ve, do, torch.ones(2, device=DEV), causal=True)
        assert got["out"].shape == (b, sq, 2, 24) and all(not bool(t.any()) for n, t in got.items() if n != "lse")
    got = _run(*_make(2, 40, 20, 2, 2, 16, 16, torch.float32), causal=True)
    assert not bool(got["out"][:, :20].any()) and not bool(got["dq"][:, :20].any()) and bool(torch.isneginf(got["lse"][:, :, :20]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,d,t", [(1000, 500, 28, 1), (300, 2000, 9, 4), (515, 333, 60, 3), (40_000, 70, 28, 2)])
def test_few_outputs(n, m, d, t):
    """Kernel smoothing: float rows of one head, a handful of outputs; hidden bad values among them."""
    q, k, v, do = _make(1, n, m, 1, 1, d, t, torch.float32, seed=22)
    _check(q, k, v, do)
    ids = torch.zeros(1, max(n, m), dtype=torch.int32, device=DEV)
    q, k, v, do = _make(1, min(n, m), m, 1, 1, d, t, torch.float32, seed=23)
    ids = ids[:, :m]
    ids[:, m // 2:] = 1
    clean = _check(q, k, v, do, causal=True, documents=ids)
    v[:, m - 3, :, t - 1] = float("nan")
    got = attention(q, k, v, causal=True, documents=ids)
    assert bool(got[:, -3:, :, t - 1].isnan().all()) and torch.equal(got[:, :-3], clean["out"][:, :-3])
    assert torch.equal(got[..., :t - 1], clean["out"][..., :t - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_scores(dtype):
    """Scores that a plain exponential would overflow on, one key far above the others, large equal scores."""
    q, k, v, do = _make(1, 100, 300, 1, 1, 64, 64, dtype, seed=8)
    k[:, 170] = q[:, 50, :, :] * 8
    _check(q * 4, k, v, do, scale=1.0)
    out = attention(q, torch.ones_like(k) * 50, torch.ones_like(v))
    # 300 equal weights p: out is the sum of p * 1 over the sum of p, two float summations of the same numbers, each within
    # 300 * 2^-24 of the true sum whatever their order, and one division; for 16-bit types that rounds to 1 (half a step
    # is 2^-11 or more) and p, within 2^-15 of a power of two times 1, adds nothing to it
    assert float((out.double() - 1).abs().max()) <= (601 * 2.0 ** -24 if dtype == torch.float32 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_run_to_run_with_shared_heads(dtype):
    q, k, v, do = _make(1, 700, 700, 8, 1, 64, 64, dtype, seed=9)
    slopes = torch.rand(8, device=DEV)
    a, b = (_run(q, k, v, do, slopes, causal=True) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)
    _check(q, k, v, do, slopes, causal=True)


@pytest.mark.gpu
def test_gradients_against_differences():
    q, k, v, do = (t.double().cpu() for t in _make(1, 20, 30, 2, 1, 12, 12, torch.float32, seed=10))
    slopes = torch.tensor([0.2, 0.05], dtype=torch.float64)
    kw = dict(causal=True, softcap=3.0, prefix=torch.tensor([4]))
    got = _run(*(t.float().to(DEV) for t in (q, k, v, do)), slopes.float().to(DEV), causal=True, softcap=3.0, prefix=torch.tensor([4], device=DEV))
    value = lambda *a: float((reference(*a[:3], slopes=a[3], **kw)["out"][0] * do).sum())  # noqa: E731
    g = torch.Generator().manual_seed(11)
    args = (q, k, v, slopes)
    for i, name in enumerate(("dq", "dk", "dv", "dslopes")):
        step = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = ([a + s * h * step if j == i else a for j, a in enumerate(args)] for s in (1, -1))
        want = (value(*up) - value(*down)) / (2 * h)
        have = float((got[name].double().cpu() * step).sum())
        assert abs(have - want) <= 2e-5 * float((got[name].double().cpu() * step).abs().sum()), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_behind_32_bits(dtype):
    """Rows 2^25 + 64 elements apart: the last of 70 keys lies behind 2^31."""
    apart = (1 << 25) + 64
    buf = torch.zeros(70 * apart, dtype=dtype, device=DEV)
    far = buf.as_strided((1, 70, 1, 32), (0, apart, 32, 1))
    q, k, v, do = _make(1, 70, 70, 1, 1, 32, 32, dtype, seed=12)
    near = _run(q, k, v, do, causal=True)
    lens = torch.tensor([70], device=DEV)
    want = cached_attention(q[:, -1], k, v, lens)
    far.copy_(k)
    got = _run(q, far, v, do, causal=True)
    assert all(torch.equal(got[n], near[n]) for n in near) and torch.equal(cached_attention(q[:, -1], far, v, lens), want)
    far.copy_(q)
    got = _run(far, k, v, do, causal=True)
    assert all(torch.equal(got[n], near[n]) for n in near)


@pytest.mark.gpu
def test_streams_and_graphs():
    b, s, h, d = 2, 150, 4, 64
    q, k, v, do = _make(b, s, s, h, 2, d, d, torch.bfloat16, seed=13)
    ids = _ids("sorted", b, s).int()
    slopes = torch.rand(h, device=DEV)
    kw = dict(causal=True, documents=ids, softcap=20.0)
    want = _run(q, k, v, do, slopes, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, slopes, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in want)
    lens = torch.tensor([150, 3], dtype=torch.int32, device=DEV)
    qn = q[:, -1].contiguous()
    graphs = []
    for _ in range(2):                                      # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = _run(q, k, v, do, slopes, **kw)
            tok = cached_attention(qn, k, v, lens)
        graphs.append((graph, res, tok))
    for i in range(4):
        for t in (q, k, v, do, qn):
            t.copy_(torch.randn_like(t))
        lens.copy_(torch.tensor([40 + i, 150 - 50 * i], device=DEV))
        graph, res, tok = graphs[i % 2]
        graph.replay()
        eager = _run(q, k, v, do, slopes, **kw)
        etok = cached_attention(qn, k, v, lens)
        torch.cuda.synchronize()
        assert all(torch.equal(res[n], eager[n]) for n in eager) and torch.equal(tok, etok)


# ---------------------------------------------------------------------------------------------------------------------
# over a cache
# ---------------------------------------------------------------------------------------------------------------------
def _cached_reference(q, k, v, lens, **kw):
    """One sequence at a time: (value, bound) of the whole batch."""
    res = []
    for i, n in enumerate(lens):
        n = max(0, min(n, k.shape[1]))
        r = reference(q[i:i + 1], k[i:i + 1, :n], v[i:i + 1, :n], causal=True, **kw)["out"]
        res.append(r)
    return tuple(torch.cat([r[j] for r in res]) for j in (0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,d,dv,t", [(1, 1, 64, 64, 1), (8, 2, 128, 128, 1), (6, 6, 33, 96, 1), (40, 1, 64, 64, 1), (8, 8, 28, 28, 5),
                                          (14, 2, 96, 80, 7), (2, 1, 127, 1, 33)])
def test_cached(dtype, hq, hk, d, dv, t):
    capacity = 1100
    lens = [1100, 0, 1, t, max(0, t - 1), 513, 31, 1200, -4]
    q, k, v, _ = _make(len(lens), t, capacity, hq, hk, d, dv, dtype, seed=14)
    for i, n in enumerate(lens):                            # what lies behind the end is not read
        n = max(0, min(n, capacity))
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    got = cached_attention(q, k, v, torch.tensor(lens, device=DEV))
    check({"out": got}, {"out": _cached_reference(q, k, v, lens)}, ["out"])
    assert torch.equal(cached_attention(q, k, v, torch.tensor(lens, device=DEV, dtype=torch.int32)), got)
    if t == 1:
        assert torch.equal(cached_attention(q[:, 0], k, v, torch.tensor(lens, device=DEV)), got[:, 0])
    slopes = torch.rand(hq, device=DEV) * 0.1
    got = cached_attention(q, k, v, torch.tensor(lens, device=DEV), slopes=slopes, softcap=5.0, scale=0.15)
    check({"out": got}, {"out": _cached_reference(q, k, v, lens, slopes=slopes, softcap=5.0, scale=0.15)}, ["out"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,capacity,d,t", [(32, 300, 64, 1), (33, 300, 64, 1), (32, 300, 128, 1), (33, 300, 128, 1), (5, 128, 40, 2),
                                            (5, 129, 40, 2), (33, 160, 8, 3), (17, 260, 96, 20)])
def test_cached_on_both_sides_of_the_launch_rules(b, capacity, d, t, dtype):
    """Eight key heads: 256 workgroups and more, caches of four tiles and more, two blocks of rows for a key head."""
    lens = [(37 * i + 5) % (capacity + 1) if i % 7 else (0, 1, capacity)[i // 7 % 3] for i in range(b)]
    q, k, v, _ = _make(b, t, capacity, 16, 8, d, d, dtype, seed=25)
    for i, n in enumerate(lens):
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    got = cached_attention(q, k, v, torch.tensor(lens, device=DEV), softcap=8.0)
    check({"out": got}, {"out": _cached_reference(q, k, v, lens, softcap=8.0)}, ["out"])
    assert torch.equal(cached_attention(q, k, v, torch.tensor(lens, device=DEV), softcap=8.0), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_cached_long_and_hidden(dtype):
    """One long sequence over many workgroups; a new token's bad value does not reach the tokens before it."""
    q, k, v, _ = _make(1, 4, 9000, 4, 2, 64, 64, dtype, seed=15)
    lens = torch.tensor([8700], device=DEV)
    want = cached_attention(q, k, v, lens)
    check({"out": want}, {"out": _cached_reference(q, k, v, [8700])}, ["out"])
    v[0, 8698], k[0, 8699] = float("nan"), float("nan")
    got = cached_attention(q, k, v, lens)
    assert torch.equal(got[:, :2], want[:, :2]) and bool(got[:, 2:].isnan().all())
    heads = k.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)           # heads before rows
    assert torch.equal(cached_attention(q[:, :2], heads, v, lens - 2), want[:, :2])


# ---------------------------------------------------------------------------------------------------------------------
# as they are used together
# ---------------------------------------------------------------------------------------------------------------------
def _plain_norm(x, w, b):
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b


def _layer_params(device, dtype=torch.float32):
    g = torch.Generator().manual_seed(16)
    p = {"w": 1 + 0.1 * torch.randn(64, generator=g), "b": 0.1 * torch.randn(64, generator=g), "qkv": torch.randn(64, 128, generator=g) / 8,
         "o": torch.randn(64, 64, generator=g) / 8}
    return {n: t.to(device=device, dtype=dtype).requires_grad_() for n, t in p.items()}


@pytest.mark.gpu
def test_a_layer_trains_and_then_serves_token_by_token():
    b, s = 2, 90
    p = _layer_params(DEV)
    x = torch.randn(b, s, 64, generator=torch.Generator().manual_seed(17)).to(DEV)

    def layer(x, p, attend, norm):
        z = norm(x, p["w"], p["b"])
        q, k, v = (z @ p["qkv"]).view(*x.shape[:2], 8, 16).split([4, 2, 2], 2)
        return x + attend(q, k, v).reshape(x.shape) @ p["o"], k, v
    y, k, v = layer(x, p, lambda q, k, v: attention(q, k, v, causal=True, softcap=20.0), layer_norm)
    u = torch.randn(y.shape, generator=torch.Generator().manual_seed(18)).to(DEV)
    got = torch.autograd.grad((y * u).sum(), list(p.values()))
    p64 = _layer_params("cpu", torch.float64)

    def plain(q, k, v):
        k, v = (t.repeat_interleave(2, 2) for t in (k, v))
        a = torch.einsum("bihd,bjhd->bhij", q, k) / 4
        a = 20 * torch.tanh(a / 20)
        a = a.masked_fill(torch.ones(s, s, dtype=torch.bool).triu(1), -math.inf).softmax(-1)
        return torch.einsum("bhij,bjhd->bihd", a, v)
    y64 = layer(x.double().cpu(), p64, plain, _plain_norm)[0]
    want = torch.autograd.grad((y64 * u.double().cpu()).sum(), list(p64.values()))
    y, k, v = y.detach(), k.detach(), v.detach()
    assert float((y.double().cpu() - y64.detach()).norm() / y64.detach().norm()) < 1e-5
    for a, e in zip(got, want):
        assert float((a.double().cpu() - e).norm() / e.norm()) < 1e-5
    with torch.no_grad():                                   # the same sequences again, the newest token at a time
        kc, vc = (torch.full((b, 128, 2, 16), float("nan"), device=DEV) for _ in range(2))
        kc[:, :s - 5], vc[:, :s - 5] = k[:, :s - 5], v[:, :s - 5]
        for i in range(s - 5, s):
            lens = torch.full((b,), i + 1, dtype=torch.int32, device=DEV)

            def attend(q, k, v):
                kc[:, i], vc[:, i] = k[:, 0], v[:, 0]
                return cached_attention(q, kc, vc, lens, softcap=20.0)
            yi = layer(x[:, i:i + 1], p, attend, layer_norm)[0]
            assert float((yi[:, 0] - y[:, i]).norm() / y[:, i].norm()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_prefix_of_the_lowest_number(dtype):
    """Counts as none, as every negative one."""
    q, k, v, do = _make(3, 70, 90, 2, 1, 40, 40, dtype, seed=22)
    _check(q, k, v, do, causal=True, prefix=torch.tensor([-2 ** 31, -1, 2 ** 31 - 1], device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_scores_that_are_seen_are_capped(dtype):
    """tanh of an infinite score is one, as it is of a score of thousands, whether or not the key's tile needs a mask."""
    q, k, v, _ = _make(1, 300, 300, 2, 2, 64, 64, dtype, seed=23)
    q[..., 0] = torch.where(q[..., 0] < 0, -1.0, 1.0).to(dtype)
    want, k2 = k.clone(), k.clone()
    for key, sign in ((0, 1), (70, -1), (150, 1), (299, -1)):
        want[:, key, :, 0], k2[:, key, :, 0] = sign * 6e4, sign * float("inf")     # 6e4 * 0.2 / 2: tanh is one in any type
    for kw in (dict(causal=True), dict(), dict(causal=True, slopes=torch.tensor([0.1, 0.0], device=DEV))):
        got = attention(q, k2, v, scale=0.2, softcap=2.0, **kw)
        assert bool(got.isfinite().all()) and torch.equal(got, attention(q, want, v, scale=0.2, softcap=2.0, **kw))


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------
def test_refusals():
    q, k, v = torch.zeros(2, 5, 4, 8), torch.zeros(2, 7, 2, 8), torch.zeros(2, 7, 2, 6)
    ids, pre, lens = torch.zeros(2, 7, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for error, match, call in [
            (RuntimeError, "GPU only", lambda: attention(q, k, v)),
            (RuntimeError, "GPU only", lambda: attention(q[0, :, 0], k[0, :, 0], v[0, :, 0])),
            (TypeError, "takes float32", lambda: attention(q.double(), k.double(), v.double())),
            (TypeError, "of one type", lambda: attention(q, k.half(), v)),
            (TypeError, "must be a tensor", lambda: attention(q, None, v)),
            (ValueError, "four dimensions", lambda: attention(q[0], k[0], v[0])),
            (ValueError, "matrix", lambda: attention(q[0, :, 0], k, v)),
            (ValueError, "do not fit", lambda: attention(q, k, v[:, :6])),
            (ValueError, "do not fit", lambda: attention(q[:1], k, v)),
            (ValueError, "do not fit", lambda: attention(q[..., :7], k, v)),
            (ValueError, "evenly", lambda: attention(q[:, :, :3], k, v)),
            (ValueError, "not be empty", lambda: attention(q[:, :, :0], k, v)),
            (ValueError, "softcap", lambda: attention(q, k, v, softcap=-1.0)),
            (ValueError, "softcap", lambda: attention(q, k, v, softcap=math.nan)),
            (ValueError, "scale", lambda: attention(q, k, v, scale=math.inf)),
            (TypeError, "float32", lambda: attention(q, k, v, slopes=torch.zeros(4, dtype=torch.float64))),
            (ValueError, "per query head", lambda: attention(q, k, v, slopes=torch.zeros(2))),
            (ValueError, "causal", lambda: attention(q, k, v, prefix=pre)),
            (TypeError, "prefix", lambda: attention(q, k, v, causal=True, prefix=pre.float())),
            (ValueError, "prefix", lambda: attention(q, k, v, causal=True, prefix=pre[:1])),
            (TypeError, "documents", lambda: attention(q, k, v, documents=ids.bool())),
            (ValueError, "documents", lambda: attention(q, k, v, documents=ids[:, :5])),
            (ValueError, "documents", lambda: attention(torch.zeros(2, 9, 4, 8), k, v, documents=ids)),
            (RuntimeError, "GPU only", lambda: cached_attention(q, k, v, lens)),
            (ValueError, "lengths", lambda: cached_attention(q, k, v, lens[:1])),
            (TypeError, "lengths", lambda: cached_attention(q, k, v, [1, 2])),
            (ValueError, "four dimensions", lambda: cached_attention(q, k[0], v[0], lens)),
            (ValueError, "evenly", lambda: cached_attention(q[:, 0, :3], k, v, lens))]:
        with pytest.raises(error, match=match):
            call()
    assert falkon_amd.attention is attention


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    q, k, v, _ = _make(1, 4, 4, 1, 1, 130, 8, torch.float16)
    with pytest.raises(NotImplementedError, match="more than 128"):
        attention(q, k, v)
    with pytest.raises(NotImplementedError, match="more than 128"):
        cached_attention(q, k, v, torch.tensor([4], device=DEV))
    q, k, v, _ = _make(1, 4, 4, 1, 1, 8, 8, torch.float16)
    with pytest.raises(RuntimeError, match="same device"):
        attention(q, k, v.cpu())
    with pytest.raises(RuntimeError, match="same device"):
        cached_attention(q, k, v, torch.tensor([4]))
    with pytest.raises(RuntimeError, match="no gradient"):
        cached_attention(q.requires_grad_(), k, v, torch.tensor([4], device=DEV))


def test_c_entry_refusals():
    """Bad arguments come back as codes with a message; none of these calls reaches a kernel."""
    from falkon_amd import _backend
    lib = _backend.load()
    one = 16                                                # any address: never read
    names = "q qb qs qh k kb ks kh v vb vs vh b sq sk hq hk d dv scale cap slopes causal prefix docs docs_b out rest lse dt ws wsb st".split()
    base = dict(zip(names, [one, 8, 8, 8] * 3 + [1, 5, 7, 4, 2, 8, 8, 1.0, 0.0, None, 0, None, None, 0, one, None, None, 0, None, 0, None]))
    call = lambda **kw: lib.flk_attention(*[{**base, **kw}[n] for n in names])  # noqa: E731
    assert call(b=0) == 0 and call(sq=0) == 0
    for bad in (dict(b=-1), dict(hq=0), dict(hq=3), dict(d=0), dict(dt=1), dict(dt=2), dict(cap=-1.0), dict(cap=math.nan), dict(prefix=one),
                dict(docs=one, sq=9), dict(q=None), dict(k=None), dict(out=None)):
        assert call(**bad) == _backend.FLK_EINVAL and _backend.last_error(), bad
    for bad in (dict(d=129), dict(dv=129), dict(sk=(1 << 28) + 1), dict(b=1 << 40), dict(b=1 << 20, sq=1 << 28), dict(cap=1e-30), dict(cap=5000.0, dt=4)):
        assert call(**bad) == _backend.FLK_EUNSUPPORTED, bad
    need = lib.flk_attention_workspace_bytes(1, 5, 7, 4, 8, 1, 0)
    assert need > 0 and lib.flk_attention_workspace_bytes(1, 5, 7, 4, 8, 0, 0) == 0
    assert lib.flk_attention_workspace_bytes(1, 5, 7, 4, 8, 1, 1) == 0
    assert call(docs=one, ws=one, wsb=need - 1) == _backend.FLK_ENOMEM and call(docs=one, wsb=need) == _backend.FLK_ENOMEM
    bnames = ("q qb qs qh k kb ks kh v vb vs vh out rest lse do dob dos doh b sq sk hq hk d dv scale cap slopes causal prefix docs docs_b "
              "dq dk dvo dsl dt ws wsb st").split()
    bbase = {**base, "lse": one, "do": one, "dob": 8, "dos": 8, "doh": 8, "dq": one, "dk": one, "dvo": one, "dsl": None}
    back = lambda **kw: lib.flk_attention_backward(*[{**bbase, **kw}[n] for n in bnames])  # noqa: E731
    for bad in (dict(dk=None), dict(dsl=one), dict(lse=None), dict(do=None), dict(out=None), dict(v=None), dict(hq=5), dict(dt=3000)):
        assert back(**bad) == _backend.FLK_EINVAL and _backend.last_error(), bad
    need = lib.flk_attention_backward_workspace_bytes(1, 5, 7, 4, 2, 8, 8, 0, 0, 0)
    assert need > 0 and back(ws=one, wsb=need - 1) == _backend.FLK_ENOMEM
    assert lib.flk_attention_backward_workspace_bytes(1, 5, 7, 3, 2, 8, 8, 0, 0, 0) == 0
    cnames = "q qb qs qh k kb ks kh v vb vs vh lens b t cap_ hq hk d dv scale cap slopes out dt ws wsb st".split()
    cbase = {**base, "lens": one, "t": 1, "cap_": 100_000}
    cached = lambda **kw: lib.flk_attention_cached(*[{**cbase, **kw}[n] for n in cnames])  # noqa: E731
    assert cached(b=0) == 0 and cached(t=0) == 0
    for bad in (dict(lens=None), dict(q=None), dict(v=None), dict(hq=7), dict(t=-1), dict(dt=1)):
        assert cached(**bad) == _backend.FLK_EINVAL, bad
    need = lib.flk_attention_cached_workspace_bytes(1, 1, 100_000, 4, 2, 8)
    assert need > 0 and cached(ws=one, wsb=need - 1) == _backend.FLK_ENOMEM
    assert lib.flk_attention_max_d(0) == 128 and lib.flk_attention_max_d(1) == 0


def test_c_entries_refuse_scales_and_caps_that_float_cannot_hold():
    """None of these calls reaches a kernel: the pointers are never read."""
    from falkon_amd import _backend
    lib = _backend.load()
    t = [16, 8, 8, 8]
    calls = (lambda scale, cap, dt: lib.flk_attention(*t, *t, *t, 1, 5, 7, 4, 2, 8, 8, scale, cap, None, 0, None, None, 0, 16, None, None, dt,
                                                      None, 0, None),
             lambda scale, cap, dt: lib.flk_attention_backward(*t, *t, *t, 16, None, 16, *t, 1, 5, 7, 4, 2, 8, 8, scale, cap, None, 0, None, None,
                                                               0, 16, 16, 16, None, dt, None, 0, None),
             lambda scale, cap, dt: lib.flk_attention_cached(*t, *t, *t, 16, 1, 1, 9, 4, 2, 8, 8, scale, cap, None, 16, dt, None, 0, None))
    for call in calls:
        for scale in (1e39, -1e39, math.inf, math.nan):
            assert call(scale, 0.0, 0) == _backend.FLK_EUNSUPPORTED and "scale" in _backend.last_error()
        for cap, dt in ((1e39, 0), (3e38, 0), (math.inf, 0), (1e5, 3), (1e-30, 0)):
            assert call(1.0, cap, dt) == _backend.FLK_EUNSUPPORTED and "softcap" in _backend.last_error()


@pytest.mark.gpu
def test_the_largest_scales_and_caps():
    """One key: the score's value is the logarithm of the sum.  A cap of 1e20 leaves a score of about one as it is."""
    q, k, v, _ = _make(1, 1, 1, 1, 1, 8, 8, torch.float32, seed=24)
    s = float((q.double() * k.double()).sum())
    for scale, cap, want in ((1.0, 1e20, s), (1e18, 1e20, 1e20 * math.tanh(s * 1e-2)), (1e18, 1e-20, math.copysign(1e-20, s))):
        out, lse = attention(q, k, v, scale=scale, softcap=cap, return_lse=True)
        assert torch.equal(out, v)
        # eight products with 2^-24 each of sum |q||k|, and 2^-20 for the cap and the units
        bound = scale * 2.0 ** -21 * float((q * k).abs().sum()) + 2.0 ** -20 * abs(want)
        assert abs(float(lse) - want) <= (bound if cap != 1e-20 else 2.0 ** -20 * 1e-20)
