"""``attention`` of float16 data whose weights or gradients lie below float16's normal numbers (6e-5): products hold them shifted."""
import pytest
import torch

from falkon_amd import attention, cached_attention

from attention_ref import reference

DEV = "cuda:0"
STEP = 2.0 ** -24                                                            # of the smallest float16 numbers


def _grads(q, k, v, do, slopes=None, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([slopes.detach().requires_grad_()] if slopes is not None else [])
    return torch.autograd.grad(attention(*leaves[:3], slopes=leaves[3] if slopes is not None else None, **kw), leaves, do)


def _make(b, sq, sk, hq, hk, d, seed):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(*s, generator=g).half().to(DEV) for s in ((b, sq, hq, d), (b, sk, hk, d), (b, sk, hk, d)))
    return q, k, v, torch.randn(b, sq, hq, d, generator=g).to(DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("power", [-13, -10, 5])
@pytest.mark.parametrize("kind", ["plain", "causal cap", "decay", "few rows"])
def test_gradients_of_small_and_large_dout(d, power, kind):
    """dout times a power of two gives the gradients times that power.  What is rounded before a sum (the scores' gradients, the weights)
    and each result is off by half a step, 2^-11, of itself at most and by a third of that in the mean, so the 2-norm of the difference
    stays below 2^-10 of the values', beside half of the smallest step for every result that is so small."""
    q, k, v, do = _make(1, 40 if kind == "few rows" else 700, 900, 4, 2, d, 50)
    do = (do * 32).round() / 32                                              # exact in float16, also times 2^-13
    slopes = torch.tensor([0.02, 0.0, 0.1, 0.005], device=DEV) if kind == "decay" else None
    kw = dict(causal="causal" in kind, softcap=5.0 if "cap" in kind else 0.0)
    want = reference(q, k, v, do, slopes=slopes, **kw)
    for name, got in zip(("dq", "dk", "dv", "dslopes"), _grads(q, k, v, (do * 2.0 ** power).half(), slopes, **kw)):
        value = want[name][0] * 2.0 ** power
        floor = STEP / 2 * value.numel() ** 0.5 if got.dtype == torch.float16 else 0.0
        assert float((got.double().cpu() - value).norm()) <= 2.0 ** -10 * float(value.norm()) + floor, name


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [1.0, 1e-3])
def test_gradients_of_long_rows(spread):
    """120 000 equal-sized weights of 8e-6.  What is rounded before a sum is off by half a step, 2^-11, of itself at most, the result
    by as much: in the 2-norm of random signs far less than twice that of the values."""
    q, k, v, do = _make(1, 200, 120_000, 1, 1, 32, 51)
    q, do = q * 0.3, (do * spread).half()
    want = reference(q, k, v, do)
    for name, got in zip(("dq", "dk", "dv"), _grads(q, k, v, do)):
        value = want[name][0]
        if name == "dq" or spread == 1.0:
            floor = STEP / 2 * value.numel() ** 0.5                          # what rounding the result to small numbers may cost
            assert float((got.double().cpu() - value).norm()) <= 2.0 ** -11 * float(value.norm()) + floor, name


@pytest.mark.gpu
def test_rows_of_dout_of_very_different_sizes():
    """One row a thousand times the others, one a thousandth; large and small values: nothing overflows, and each row's dq is as exact
    as by itself."""
    q, k, v, do = _make(1, 300, 300, 2, 2, 64, 52)
    do[:, 100], do[:, 200] = do[:, 100] * 1e3, do[:, 200] * 1e-3
    do = do.half()
    dq, dk, dv = _grads(q, k, v, do, causal=True)
    want = reference(q, k, v, do, causal=True)
    for row in (99, 100, 200, 299):
        value = want["dq"][0][:, row]
        assert float((dq[:, row].double().cpu() - value).norm()) <= 2.0 ** -10 * float(value.norm()) + STEP / 2 * 128 ** 0.5
    big = [t.double().cpu() for t in _grads(q, k, v * 2000, do.float().clamp(-4, 4).half(), causal=True, scale=2.0 ** -9)]
    exact = reference(q, k, v * 2000, do.float().clamp(-4, 4).half(), causal=True, scale=2.0 ** -9)
    for name, t in zip(("dq", "dk", "dv"), big):
        assert bool(t.isfinite().all())
        assert float((t - exact[name][0]).norm()) <= 2.0 ** -9 * float(exact[name][0].norm()), name


@pytest.mark.gpu
def test_a_peak_over_a_long_tail():
    """One key's weight is twice those of 130 000 others together: 2^-18 of it each.  The parts of a row's keys join exactly, so there are
    enough rows that their keys are not divided."""
    n, d, heads = 130_001, 32, 512
    q = torch.zeros(1, 1, heads, d, device=DEV, dtype=torch.float16)
    k = torch.zeros(1, n, 1, d, device=DEV, dtype=torch.float16)
    v = (1 + torch.rand(1, n, 1, d, generator=torch.Generator().manual_seed(53))).half().to(DEV)
    q[..., 0], k[:, 77, :, 0] = 3.5, 3.5625                                  # exp(12.47) = 2.6e5
    v[:, 77] = 0
    want = reference(q[:, :, :1], k, v, scale=1.0)["out"][0]
    # half a step, 2^-11, for the result, for the peak's weight and for the tail's, which are rounded alike, all being equal
    got = attention(q, k, v, scale=1.0)
    assert bool(((got.double().cpu() - want).abs() <= 3 * 2.0 ** -11 * want.abs()).all())
    got = cached_attention(q[:, 0, :1], k, v, torch.tensor([n], device=DEV), scale=1.0)
    assert bool(((got.double().cpu() - want[:, 0]).abs() <= 3 * 2.0 ** -11 * want[:, 0].abs()).all())


@pytest.mark.gpu
def test_gradients_of_scores_of_millions():
    """float's step at 1e7 is one, so a weight may come out as e^(1/2): nothing overflows behind it."""
    q, k, v, do = _make(1, 200, 200, 2, 2, 64, 54)
    q, k = q * 900, k * 900
    for t in _grads(q, k, v, do.half(), causal=True):
        assert bool(t.isfinite().all())
