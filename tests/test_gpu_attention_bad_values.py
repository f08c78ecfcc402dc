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
