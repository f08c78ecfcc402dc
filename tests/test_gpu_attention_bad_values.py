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
