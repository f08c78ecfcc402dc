"""``layer_norm`` and its gradients against the formulas in 64 bits on the CPU.

Tolerances.  16-bit results are the float result rounded once: half a step of the type (``eps / 2``) of the value, plus
what float arithmetic before it adds.  Float arithmetic: mean, variance and the two sums of the backward pass are sums of
d terms in a tree over the row's threads, at most 32 of them in sequence plus ten levels, each rounding off by 2^-24 of
the sum of magnitudes; with the handful of roundings per value around them fewer than 64 roundings act on a value, so
64 * 2^-24 = 4e-6 of the row's largest magnitudes (1e-14 for double).  Sums over N rows: at most N / 8 terms in
sequence before the tree; the tests' N <= 4099 gives fewer than 600 roundings of the sum of magnitudes, and errors
of either sign: 64 roundings' worth is already four standard deviations (sqrt(600) * 0.3 = 7), so the same factor holds.
"""
import pytest
import torch

import falkon_amd
from falkon_amd import GaussianKernel, layer_norm

_WIDE = {torch.float32: 64 * 2.0 ** -24, torch.float64: 64 * 2.0 ** -53, torch.float16: 64 * 2.0 ** -24,
         torch.bfloat16: 64 * 2.0 ** -24}


def _reference(x, w, b, dy, eps=1e-5):
    """(y, dx, dw, db) and the magnitudes that were summed for each, in 64 bits on the CPU."""
    x, dy = x.detach().double().cpu().reshape(-1, x.shape[-1]), dy.double().cpu().reshape(-1, x.shape[-1])
    d = x.shape[1]
    w = torch.ones(d, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(d, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    z = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - z * (g * z).mean(1, keepdim=True))
    # the largest magnitudes that enter a row's sums: a rounding of the mean is 2^-24 of the largest |x|, times rstd in z
    zmag = (x.abs().amax(1, keepdim=True) * rstd).clamp_min(1.0) + z.abs()
    ymag = zmag * w.abs() + b.abs()
    gmax = g.abs().amax(1, keepdim=True)
    dxmag = rstd * gmax * (2 + 2 * zmag * z.abs().amax(1, keepdim=True).clamp_min(1.0))
    return (z * w + b, ymag), (dx, dxmag), ((dy * z).sum(0), (dy.abs() * zmag).sum(0)), (dy.sum(0), dy.abs().sum(0))


def _close(got, want, mag):
    got = got.detach().double().cpu().reshape(want.shape)
    tol = mag * _WIDE[_close.dtype] + (want.abs() * torch.finfo(_close.out).eps / 2 if _close.out.itemsize == 2 else 0)
    tol = tol + (2.0 ** -25 if _close.out == torch.float16 else 0)          # half a step of the smallest float16 values
    worst = ((got - want).abs() / tol.clamp_min(1e-300)).max().item() if want.numel() else 0.0
    assert worst <= 1.0, worst


def _check(x, w, b, dy, y, grads):
    ref = _reference(x, w, b, dy)
    _close.dtype = x.dtype
    for got, (want, mag) in zip((y, *grads), ref):
        if got is not None:
            _close.out = got.dtype
            _close(got, want, mag)


def _make(rows, d, dtype, seed=0, wdtype=None, dev="cuda:0"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, d, generator=g) * 2 + 0.5).to(dtype).to(dev)
    w = (torch.randn(d, generator=g) * 0.3 + 1).to(wdtype or dtype).to(dev)
    b = torch.randn(d, generator=g).to(wdtype or dtype).to(dev)
    dy = torch.randn(rows, d, generator=g).to(dtype).to(dev)
    return x.requires_grad_(), w.requires_grad_(), b.requires_grad_(), dy


# one size on each side of every row layout, odd ones among them, rows that do not fill a workgroup
_SIZES = [(1, 1), (5, 2), (3, 7), (33, 8), (257, 28), (64, 33), (31, 64), (100, 100), (65, 257), (7, 784), (130, 1000),
          (4099, 24), (19, 2048), (17, 4096), (5, 5001), (3, 8192), (3, 16384), (2, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,d", _SIZES)
def test_values_and_gradients(rows, d, dtype):
    x, w, b, dy = _make(rows, d, dtype)
    y = layer_norm(x, w, b)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    grads = torch.autograd.grad(y, (x, w, b), dy)
    _check(x, w, b, dy, y, grads)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), y)
    again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)          # the same run to run
    assert all(torch.equal(g, h) for g, h in zip(grads, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_float_weights_with_16_bit_rows(dtype):
    x, w, b, dy = _make(50, 200, dtype, wdtype=torch.float32)
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    assert grads[1].dtype == torch.float32 and grads[2].dtype == torch.float32
    _check(x, w, b, dy, y, grads)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["none", "weight", "bias", "x only", "weight only", "bias only"])
def test_absent_operands_and_single_gradients(which):
    x, w, b, dy = _make(37, 96, torch.float32)
    if which in ("none", "weight", "bias"):
        w, b = (w if which == "weight" else None), (b if which == "bias" else None)
        leaves = [t for t in (x, w, b) if t is not None]
    else:
        leaves = [{"x only": x, "weight only": w, "bias only": b}[which]]
        for t in (x, w, b):
            t.requires_grad_(t is leaves[0])
    y = layer_norm(x, w, b)
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    _check(x, w, b, dy, y, [None if t is None else got.get(id(t)) for t in (x, w, b)])


@pytest.mark.gpu
def test_strides_alignment_and_broadcast_gradients():
    base = torch.randn(40, 130, device="cuda:0")
    dy = torch.randn(40, 64, device="cuda:0")
    for x in (base[:, 1:65], base[:, 4:68], base[::2, :64].expand(20, 64), base.T[:64].T, base[:1, :64].expand(40, 64)):
        x = x.detach().requires_grad_()
        g = dy[:x.shape[0]]
        y = layer_norm(x)
        _check(x, None, None, g, y, torch.autograd.grad(y, (x,), g))
    x = torch.randn(6, 5, 48, device="cuda:0", requires_grad=True)
    w = torch.randn(49, device="cuda:0")[1:].requires_grad_()               # a weight that starts between two vectors
    y = layer_norm(x, w)
    ones = torch.ones((), device="cuda:0").expand(6, 5, 48)                 # what y.sum().backward() passes
    _check(x, w, None, ones, y, torch.autograd.grad(y.sum(), (x, w)))
    v = torch.randn(17, device="cuda:0")
    assert torch.equal(layer_norm(v), layer_norm(v[None])[0])
    assert layer_norm(torch.empty(0, 5, device="cuda:0")).shape == (0, 5)
    x0 = torch.empty(0, 5, device="cuda:0", requires_grad=True)
    w0 = torch.ones(5, device="cuda:0", requires_grad=True)
    gx, gw = torch.autograd.grad(layer_norm(x0, w0).sum(), (x0, w0))
    assert gx.shape == (0, 5) and torch.equal(gw, torch.zeros(5, device="cuda:0"))


@pytest.mark.gpu
def test_large_offsets_constant_rows_and_bad_values():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(9, 300, generator=g) + 1e4).cuda()                     # sum(x^2) - mean^2 would lose everything here
    dy = torch.randn(9, 300, generator=g).cuda()
    x.requires_grad_()
    y = layer_norm(x)
    _check(x, None, None, dy, y, torch.autograd.grad(y, (x,), dy))
    assert torch.equal(layer_norm(torch.full((3, 100), 7.0, device="cuda:0")), torch.zeros(3, 100, device="cuda:0"))
    bad = torch.randn(20, 28, device="cuda:0")
    good = layer_norm(bad)
    bad[3, 5], bad[7, 0] = float("nan"), float("inf")
    out = layer_norm(bad)
    hit = torch.zeros(20, dtype=torch.bool, device="cuda:0")
    hit[3] = hit[7] = True
    assert bool(out[hit].isnan().all()) and torch.equal(out[~hit], good[~hit])


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, dy = _make(3, 20, torch.float64)
    assert torch.autograd.gradcheck(lambda *a: layer_norm(*a), (x, w, b), eps=1e-6, atol=1e-6)


@pytest.mark.gpu
def test_rows_behind_32_bit_offsets():
    rows, d = 70_000, 32_768                                                # 2.3e9 elements of bfloat16: 4.6 GB
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device="cuda:0")
    x[-3:] = torch.randn(3, d, device="cuda:0").bfloat16()
    y = layer_norm(x)
    assert torch.equal(y[-3:], layer_norm(x[-3:].clone())) and not bool(y[-4].any())


@pytest.mark.gpu
def test_streams_and_graphs():
    x, w, b, dy = _make(100, 784, torch.bfloat16)
    want = layer_norm(x, w, b)
    wgrad = torch.autograd.grad(want, (x, w, b), dy)
    want = want.detach()         # no eager graph of these leaves may live while their backward pass is captured
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer_norm(x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want) and all(torch.equal(g, h) for g, h in zip(grads, wgrad))
    del y, grads
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy = layer_norm(x, w, b)
        gg = torch.autograd.grad(gy, (x, w, b), dy)
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(100, 784, device="cuda:0"))
            dy.copy_(torch.randn(100, 784, device="cuda:0"))
        graph.replay()
        eager = layer_norm(x, w, b)
        egrad = torch.autograd.grad(eager, (x, w, b), dy)
        torch.cuda.synchronize()
        assert torch.equal(gy, eager) and all(torch.equal(g, h) for g, h in zip(gg, egrad))


@pytest.mark.gpu
def test_normalised_rows_into_a_kernel_product():
    """Rows normalised with a learned weight, then compared by a kernel: one gradient through both."""
    g = torch.Generator().manual_seed(5)
    X, C = torch.randn(60, 12, generator=g).cuda(), torch.randn(20, 12, generator=g).cuda()
    v, u = torch.randn(20, 2, generator=g).cuda(), torch.randn(60, 2, generator=g).cuda()
    w = (torch.randn(12, generator=g) * 0.2 + 1).cuda().requires_grad_()
    X.requires_grad_()
    out = GaussianKernel(2.0).mmv(layer_norm(X, w), layer_norm(C, w), v)
    got = torch.autograd.grad((out * u).sum(), (X, w))
    X64, w64 = X.detach().double().cpu().requires_grad_(), w.detach().double().cpu().requires_grad_()

    def norm(x):
        c = x - x.mean(1, keepdim=True)
        return c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * w64
    k = torch.exp(-torch.cdist(norm(X64), norm(C.double().cpu())) ** 2 / 8)
    want = torch.autograd.grad((k @ v.double().cpu() * u.double().cpu()).sum(), (X64, w64))
    for a, e in zip(got, want):
        assert float((a.double().cpu() - e).norm() / e.norm()) < 1e-4


def test_refusals():
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        layer_norm(x)
    with pytest.raises(TypeError, match="layer_norm takes"):
        layer_norm(x.int())
    with pytest.raises(TypeError, match="layer_norm takes"):
        layer_norm([1.0, 2.0])
    with pytest.raises(ValueError, match="at least one feature"):
        layer_norm(torch.zeros(3, 0))
    for w, error in ((torch.ones(7), ValueError), (torch.ones(8, dtype=torch.float64), TypeError)):
        with pytest.raises(error):
            layer_norm(x, w)
    assert falkon_amd.layer_norm is layer_norm


def test_c_entry_refusals():
    """Bad arguments come back as codes with a message; none of these calls reaches a kernel."""
    from falkon_amd import _backend
    lib = _backend.load()
    one = 16                                                                # any address: never read
    call = lambda **k: lib.flk_layer_norm(*[{**dict(x=one, rows=4, d=8, rs=8, w=None, b=None, wd=0, eps=1e-5, y=one, m=None, r=None, dt=0, st=None),  # noqa: E731
                                             **k}[n] for n in ("x", "rows", "d", "rs", "w", "b", "wd", "eps", "y", "m", "r", "dt", "st")])
    assert call(rows=0) == 0
    for bad in (dict(rows=-1), dict(d=0), dict(rs=-8), dict(dt=2), dict(dt=9), dict(x=None), dict(y=None), dict(m=one), dict(eps=-1.0),
                dict(eps=float("nan")), dict(w=one, wd=4), dict(w=one, wd=0, dt=1)):
        assert call(**bad) == _backend.FLK_EINVAL and _backend.last_error(), bad
    assert call(d=(1 << 30) + 1) == _backend.FLK_EUNSUPPORTED
    assert lib.flk_layer_norm_backward_workspace_bytes(100, 8, 7) == 0
    assert lib.flk_layer_norm_backward_workspace_bytes(-1, 8, 0) == 0
    need = lib.flk_layer_norm_backward_workspace_bytes(100, 8, 0)
    assert need > 0
    assert lib.flk_layer_norm_backward(one, 100, 8, 8, one, 8, one, 0, one, one, one, one, one, 0, one, need - 1, None) == _backend.FLK_ENOMEM
    assert lib.flk_layer_norm_backward(one, 100, 8, 8, None, 8, one, 0, one, one, one, one, one, 0, one, need, None) == _backend.FLK_EINVAL


def test_refuses_a_weight_that_is_no_tensor():
    x = torch.zeros(3, 4)
    for kw in (dict(weight=1.0), dict(bias=[0.0] * 4), dict(weight=torch.ones(4), bias=2)):
        with pytest.raises(TypeError, match="must be a tensor"):
            falkon_amd.layer_norm(x, **kw)
