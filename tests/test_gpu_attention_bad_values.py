"""Infinities and NaNs among the operands of ``attention`` and ``cached_attention``: what sees them gets what the formula gives, alike
in tiles with a mask and without one, and what does not see them is the same to the last bit."""
import pytest
import torch

from falkon_amd import attention, cached_attention

from attention_ref import check, reference

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _make(b, sq, sk, hq, hk, d, dv, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((b, sq, hq, d), (b, sk, hk, d), (b, sk, hk, dv), (b, sq, hq, dv))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,dv", [(64, 64), (32, 24), (96, 81), (128, 128)])
def test_bad_values_anywhere_in_a_cached_row(dtype, d, dv):
    """The newest of two tokens has one bad value, in every place of its row in turn: the token before it does not see it, and the
    newest one has it in that place alone."""
    q, k, v, _ = _make(dv, 2, 45, 2, 1, d, dv, dtype, seed=30)
    lens = torch.full((dv,), 45, device=DEV)
    want = cached_attention(q, k, v, lens)
    for value in (float("nan"), float("inf"), -float("inf")):
        bad = v.clone()
        bad[torch.arange(dv), 44, 0, torch.arange(dv)] = value              # sequence i: value i
        got = cached_attention(q, k, bad, lens)
        assert torch.equal(got[:, 0], want[:, 0])
        hit = torch.eye(dv, dtype=torch.bool, device=DEV)[:, None].expand(dv, 2, dv)
        assert bool((got[:, 1][hit].isnan() if value != value else got[:, 1][hit] == value).all())
        assert bool(got[:, 1][~hit].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinite_value_with_a_weight_of_nothing(dtype):
    """exp(-300) is zero in 32 bits, and zero times an infinity is no number of any result: rows that see it say so in tiles with
    a mask and without one, and in that column alone."""
    q, k, v, _ = _make(1, 200, 200, 2, 2, 64, 64, dtype, seed=31)
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[:, [5, 150], :, 0] = -300.0 * 8                                       # the scale is 1 / 8
    v[:, 5, :, 7], v[:, 150, :, 9] = float("inf"), -float("inf")
    for out in (attention(q, k, v, causal=True), cached_attention(q, k, v, torch.tensor([200], device=DEV))):
        assert not bool(out[:, 5:, :, 7].isfinite().any()) and not bool(out[:, 150:, :, 9].isfinite().any())
        out[:, 5:, :, 7], out[:, 150:, :, 9] = 0.0, 0.0
        assert bool(out.isfinite().all())


def _infinite_keys(dtype, capped):
    """Keys with one infinity each, in column 0 or 3, on both sides of the causal masks' tiles.  With a cap their scores are plus or
    minus the cap, without one minus infinity (the queries' column 0 is +-1 there and column 3 is 1), so every row's sum is finite."""
    q, k, v, do = _make(1, 300, 300, 2, 2, 64, 64, dtype, seed=32)
    q[..., 0], q[..., 3] = 1.0, 1.0
    if capped:
        q[:, ::3, :, 0] = -1.0
    bad = [(1, 0, -1), (70, 3, -1), (150, 0, -1), (280, 3, -1)] + ([(40, 0, 1), (200, 3, 1)] if capped else [])
    for key, c, sign in bad:
        k[:, key, :, c] = sign * float("inf")
    return q, k, v, do, bad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("capped", [False, True])
@pytest.mark.parametrize("mask", ["causal", "none", "documents", "prefix"])
def test_gradients_of_rows_that_see_infinite_keys(dtype, capped, mask):
    """A capped score's derivative is zero where the score is infinite, and a weight is zero where it is minus infinity: dq and the slopes'
    gradient are those of a key far out (whose score is as good as infinite), and NaN in the infinity's own column (zero times it)."""
    q, k, v, do, bad = _infinite_keys(dtype, capped)
    far = k.clone()
    for key, c, sign in bad:
        far[:, key, :, c] = sign * 3e4                                       # a score of 6e3: the cap is reached, or exp(-6e3) = 0
    slopes = torch.tensor([0.02, 0.0], device=DEV).requires_grad_()
    kw = dict(causal=mask != "none", scale=0.2, softcap=2.0 if capped else 0.0)
    if mask == "documents":
        kw["documents"] = (torch.arange(300, device=DEV) // 130)[None].contiguous()
    if mask == "prefix":
        kw["prefix"] = torch.tensor([90], device=DEV)
    pos = torch.arange(300, device=DEV)
    see = torch.ones(300, 300, dtype=torch.bool, device=DEV) if mask == "none" else pos[:, None] >= pos[None]
    if mask == "prefix":
        see = see | (pos[None] < 90)
    if mask == "documents":
        see = see & (kw["documents"][0][:, None] == kw["documents"][0][None])

    def run(keys, sl):
        leaves = [t.detach().requires_grad_() for t in (q, keys, v)] + ([sl] if sl is not None else [])
        out = attention(*leaves[:3], slopes=sl, **kw)
        return out.detach(), torch.autograd.grad(out, leaves, do)
    for sl in (slopes, None):
        out, got = run(k, sl)
        out2, want = run(far, sl)
        assert torch.equal(out, out2)
        hit = torch.zeros(1, 300, 2, 64, dtype=torch.bool, device=DEV)
        for key, c, _ in bad:
            hit[:, see[:, key], :, c] = True
        assert bool(got[0][hit].isnan().all())
        assert torch.equal(got[0][~hit], want[0][~hit])
        assert sl is None or torch.equal(got[3], want[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("capped", [False, True])
@pytest.mark.parametrize("sq", [300, 320, 33])
def test_gradients_of_infinite_keys(dtype, capped, sq):
    """dk and dv of every key, the infinite ones among them, are those of keys far out; also where a tile holds rows past the last
    one, whose queries are zero, and zero times an infinity is their score."""
    q, k, v, do, bad = _infinite_keys(dtype, capped)
    q, do = q[:, -sq:], do[:, -sq:]
    far = k.clone()
    for key, c, sign in bad:
        far[:, key, :, c] = sign * 3e4
    for causal in (False, True):
        got, want = ([t for t in _grads(q, keys, v, do, causal=causal and sq <= 300, scale=0.2, softcap=2.0 if capped else 0.0)] for keys in (k, far))
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2]) and bool(want[1].isfinite().all())


def _within(got, want, where):
    """Inside the bounds of ``attention_ref`` at these places.  (A row that is not finite is added to dk and dv by itself, behind the
    others and with unrounded weights, so they are not the same to the last bit.)"""
    value, bound = want
    off = (got.double().cpu() - value).abs()[where.cpu()]
    assert bool((off <= bound[where.cpu()]).all())


def _grads(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(attention(*leaves, **kw), leaves, do)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("mask", ["causal", "none", "documents"])
def test_dv_does_not_depend_on_v(dtype, d, mask):
    """dv is the weights' transpose times dout: NaNs and infinities of v that rows see are in out, dq and dk, and not in dv."""
    q, k, v, do = _make(1, 290, 290, 4, 2, d, d, dtype, seed=33)
    kw = dict(causal=mask != "none")
    if mask == "documents":
        kw["documents"] = (torch.arange(290, device=DEV) // 100)[None].contiguous()
    want = _grads(q, k, v, do, **kw)
    v2 = v.clone()
    v2[:, 130, :, 1], v2[:, 285, :, d - 1] = float("nan"), -float("inf")
    got = _grads(q, k, v2, do, **kw)
    assert torch.equal(got[2], want[2])
    assert not bool(got[0][:, 285:].isfinite().any())
    if mask == "causal":
        assert torch.equal(got[0][:, :130], want[0][:, :130]) and not bool(got[1][:, :286].isfinite().any())
        assert torch.equal(got[1][:, 286:].isfinite(), torch.zeros_like(got[1][:, 286:], dtype=torch.bool))
    if mask == "documents":                                                  # documents 0 .. 99, 100 .. 199, 200 .. 289
        assert torch.equal(got[0][:, :130], want[0][:, :130]) and torch.equal(got[0][:, 200:285], want[0][:, 200:285])
        assert torch.equal(got[1][:, :100], want[1][:, :100]) and not bool(got[1][:, 200:286].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("mask", ["causal", "none", "documents"])
def test_gradients_of_keys_that_see_one_bad_value_of_dout(dtype, d, mask):
    """dv is not finite in that column and dk nowhere; dv's other columns and the other keys are as they were."""
    q, k, v, do = _make(1, 290, 290, 4, 2, d, d, dtype, seed=34)
    kw = dict(causal=mask != "none")
    if mask == "documents":
        kw["documents"] = (torch.arange(290, device=DEV) // 100)[None].contiguous()
    want, exact = _grads(q, k, v, do, **kw), reference(q, k, v, do, **kw)
    for value in (float("nan"), float("inf")):
        do2 = do.clone()
        do2[:, 150, 1, 5] = value                                            # a head that shares key head 0
        got = _grads(q, k, v, do2, **kw)
        lo, hi = {"causal": (0, 151), "none": (0, 290), "documents": (100, 151)}[mask]
        hit = torch.zeros(1, 290, 2, d, dtype=torch.bool, device=DEV)
        hit[:, lo:hi, 0, 5] = True
        assert not bool(got[2][hit].isfinite().any())
        _within(got[2], exact["dv"], ~hit)
        assert torch.equal(got[2][:, :lo], want[2][:, :lo]) and torch.equal(got[2][:, hi:], want[2][:, hi:]) and torch.equal(got[2][:, :, 1], want[2][:, :, 1])
        assert not bool(got[1][:, lo:hi, 0].isfinite().any())
        assert torch.equal(got[1][:, :lo], want[1][:, :lo]) and torch.equal(got[1][:, hi:], want[1][:, hi:]) and torch.equal(got[1][:, :, 1], want[1][:, :, 1])
        row = torch.zeros(1, 290, 4, d, dtype=torch.bool, device=DEV)
        row[:, 150, 1] = True
        assert torch.equal(got[0][~row], want[0][~row]) and not bool(got[0][row].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["causal", "none"])
def test_gradients_of_rows_with_an_infinity_and_a_cap(dtype, mask):
    """Such a row's scores are plus or minus the cap and have no gradient: dv and dq are those of a row far out, dk is NaN in the
    infinity's own column (zero times it) for the keys that the row sees, and elsewhere that of a row far out."""
    q, k, v, do = _make(1, 290, 290, 2, 2, 64, 64, dtype, seed=35)
    k[..., 2] = torch.where(k[..., 2] < 0, -1.0, 1.0).to(dtype)
    far, q2 = q.clone(), q.clone()
    far[:, 140, :, 2], q2[:, 140, :, 2] = 3e4, float("inf")
    kw = dict(causal=mask == "causal", scale=0.2, softcap=2.0)
    got, want = _grads(q2, k, v, do, **kw), _grads(far, k, v, do, **kw)
    hit = torch.zeros(1, 290, 2, 64, dtype=torch.bool, device=DEV)
    hit[:, :141 if mask == "causal" else 290, :, 2] = True
    assert torch.equal(got[0], want[0]) and bool(got[1][hit].isnan().all())
    exact = reference(far, k, v, do, **kw)
    _within(got[1], exact["dk"], ~hit)
    _within(got[2], exact["dv"], torch.ones_like(hit))
    if mask == "causal":
        assert torch.equal(got[1][:, 141:], want[1][:, 141:]) and torch.equal(got[2][:, 141:], want[2][:, 141:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", [False, True])
def test_hidden_bad_keys_with_a_cap(dtype, decay):
    """A hidden score of NaN has a cap's derivative of NaN: it is hidden too."""
    q, k, v, do = _make(1, 200, 200, 2, 2, 64, 64, dtype, seed=36)
    ids = (torch.arange(200, device=DEV) // 70)[None].contiguous()
    ids[:, 180:] = -1
    slopes = torch.tensor([0.1, 0.01], device=DEV).requires_grad_() if decay else None

    def run(k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([slopes] if decay else [])
        return torch.autograd.grad(attention(*leaves[:3], slopes=slopes, causal=True, documents=ids, softcap=3.0), leaves, do)
    want = run(k, v)
    for value in (float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[:, 185, :, 9], v2[:, 190, :, 3] = value, value
        assert all(torch.equal(a, b) for a, b in zip(run(k2, v2), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_where_nothing_is_finite(dtype):
    q, k, v, do = _make(1, 700, 700, 4, 2, 64, 64, dtype, seed=37)
    nan = torch.full_like(q, float("nan"))
    for kw in (dict(), dict(causal=True)):
        for rows, douts in ((nan, do), (q, nan)):
            got = _grads(rows, k, v, douts, **kw)
            assert all(bool(t.isnan().all()) for t in got[:2]) and bool(got[2].isnan().all())
    ids = torch.zeros(1, 700, dtype=torch.int32, device=DEV)
    ids[:, 200:600] = -1                                                     # padding between, which holds nothing else
    want = _grads(q, k, v, do, causal=True, documents=ids)
    q[:, 200:600], do[:, 250:600] = float("nan"), float("inf")
    assert all(torch.equal(a, b) for a, b in zip(_grads(q, k, v, do, causal=True, documents=ids), want))


def _by_the_formula(q, k, v, do, see, scale, cap, slopes):
    """out, dq, dk and dv of one batch entry in 64 bits, place by place over what is seen, with IEEE's rules for what is not finite."""
    g = q.shape[1] // k.shape[1]
    q, k, v, do = (t.double().cpu().transpose(0, 1) for t in (q, k, v, do))
    sq, sk = q.shape[1], k.shape[1]
    dist = (torch.arange(sk - sq, sk)[:, None] - torch.arange(sk)[None]).abs().double()
    out, dq, dk, dv = torch.zeros_like(do), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    seen = lambda t: torch.where(see[:, :, None], t, 0.0)  # noqa: E731
    for h in range(q.shape[0]):
        kh, vh = k[h // g], v[h // g]
        x, grad = scale * (q[h][:, None] * kh[None]).sum(2), 1.0
        if cap:
            t = torch.tanh(x / cap)
            x, grad = cap * t, 1 - t * t
        if slopes is not None:
            x = x - float(slopes[h]) * dist
        x = x.masked_fill(~see, -float("inf"))
        lse = torch.logsumexp(x, 1, keepdim=True)
        lse = torch.where(x.isnan().any(1, keepdim=True) | (x == float("inf")).any(1, keepdim=True), float("nan"), lse)
        p = torch.exp(x - torch.where(lse == -float("inf"), 0.0, lse))
        out[h] = seen(p[:, :, None] * vh[None]).sum(1)
        dp, delta = (do[h][:, None] * vh[None]).sum(2), (do[h] * out[h]).sum(1, keepdim=True)
        ds = p * (dp - delta) * grad
        dq[h] = scale * seen(ds[:, :, None] * kh[None]).sum(1)
        dk[h // g] += scale * seen(torch.where(p == 0, 0.0, ds)[:, :, None] * q[h][:, None]).sum(0)
        dv[h // g] += seen(p[:, :, None] * do[h][:, None]).sum(0)
    return [t.transpose(0, 1) for t in (out, dq, dk, dv)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seed", range(12))
def test_bad_values_scattered_over_all_operands(dtype, seed):
    """A handful of infinities and NaNs anywhere: the same places are finite as by the formula, and those are as exact as ever.  (Where
    a result is not finite, whether it is an infinity or NaN depends on how its sum is made.)"""
    g = torch.Generator().manual_seed(100 + seed)
    pick = lambda *a: a[int(torch.randint(len(a), (1,), generator=g))]  # noqa: E731
    sq, sk, hq, hk, d, dv = pick(40, 130, 300), pick(45, 200, 1100), pick(2, 4), pick(1, 2), pick(16, 45, 80), pick(3, 32, 72)
    q, k, v, do = _make(1, sq, sk, hq, hk, d, dv, dtype, seed=200 + seed)
    q, k = q * 0.5, k * 0.7
    causal, cap = pick(True, False), pick(0.0, 3.0)
    slopes = pick(None, torch.linspace(0.0, 0.05, hq, device=DEV))
    ids = pick(None, torch.arange(sk, device=DEV) * 3 // sk) if sq <= sk else None
    prefix = pick(None, torch.tensor([20], device=DEV)) if causal else None
    for t, many in ((q, pick(0, 2)), (k, pick(0, 2)), (v, pick(0, 2)), (do, pick(0, 2))):
        for _ in range(many):
            at = [int(torch.randint(n, (1,), generator=g)) for n in t.shape]
            t[tuple(at)] = pick(float("inf"), -float("inf"), float("nan"))
    pos, key = torch.arange(sk - sq, sk)[:, None], torch.arange(sk)[None]
    see = key <= pos if causal else torch.ones(sq, sk, dtype=torch.bool)
    if prefix is not None:
        see = see | (key < 20)
    if ids is not None:
        see = see & (ids.cpu()[sk - sq:, None] == ids.cpu()[None])
    want = _by_the_formula(q[0], k[0], v[0], do[0], see, 0.25, cap, slopes)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, scale=0.25, causal=causal, softcap=cap, slopes=slopes, prefix=prefix, documents=None if ids is None else ids[None].contiguous())
    for name, got, value in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do)), want):
        got, fine = got[0].double().cpu(), value.isfinite()
        assert torch.equal(got.isfinite(), fine), name
        if fine.any():                                                       # (weights, their gradients and the result: one rounding each)
            unit = 2.0 ** -16 if dtype == torch.float32 else 2 * torch.finfo(dtype).eps
            assert float((got - value)[fine].norm()) <= unit * float(value[fine].norm()) + 1e-6, name
