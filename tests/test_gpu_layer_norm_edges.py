"""``layer_norm`` at its edges: no rows, weights that start anywhere, rows far from zero."""
import pytest
import torch

from falkon_amd import _backend, layer_norm

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,code", [(torch.float32, _backend.FLK_F32), (torch.bfloat16, _backend.FLK_BF16)])
@pytest.mark.parametrize("d", [5, 4096, 40_000])
def test_c_entry_with_no_rows(d, dtype, code):
    """The gradients of weight and bias are zero, whatever the row layout and whether or not dx is given."""
    lib = _backend.load()
    x = torch.zeros(1, d, dtype=dtype, device=DEV)
    stat = torch.zeros(1, device=DEV)
    for dx in (x.data_ptr(), None):
        dw, db = torch.ones(d, dtype=dtype, device=DEV), torch.ones(d, dtype=dtype, device=DEV)
        need = lib.flk_layer_norm_backward_workspace_bytes(0, d, code)
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        rc = lib.flk_layer_norm_backward(x.data_ptr(), 0, d, d, x.data_ptr(), d, x.data_ptr(), code, stat.data_ptr(), stat.data_ptr(), dx,
                                         dw.data_ptr(), db.data_ptr(), code, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0, _backend.last_error()
        assert not bool(dw.any()) and not bool(db.any())
    x0, w0 = torch.empty(0, d, dtype=dtype, device=DEV, requires_grad=True), torch.ones(d, dtype=dtype, device=DEV, requires_grad=True)
    gx, gw = torch.autograd.grad(layer_norm(x0, w0).sum(), (x0, w0))
    assert gx.shape == (0, d) and not bool(gw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("first", [1, 4])
def test_float_weights_that_start_anywhere_beside_16_bit_rows(dtype, first):
    """Sixteen bytes into an allocation, or four: eight float weights are more than the 16 bytes that the rows ask for."""
    g = torch.Generator().manual_seed(40)
    x, dy = (torch.randn(30, 64, generator=g).to(dtype).to(DEV) for _ in range(2))
    w, b = (torch.randn(64, generator=g).to(DEV) for _ in range(2))
    far_w, far_b = (torch.nn.functional.pad(t, (first, 0))[first:] for t in (w, b))
    leaves = [[t.detach().requires_grad_() for t in (x, ww, bb)] for ww, bb in ((w, b), (far_w, far_b))]
    assert leaves[1][1].data_ptr() % 32 != 0
    y, far = (layer_norm(*t) for t in leaves)
    assert torch.equal(y, far) or first == 1                                 # (other alignment, another order of the sums)
    assert torch.allclose(y.float(), far.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-5)
    for a, e in zip(torch.autograd.grad(far, leaves[1], dy), torch.autograd.grad(y, leaves[0], dy)):
        assert torch.equal(a, e) or first == 1
        assert torch.allclose(a.float(), e.float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-4)


def _unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [28, 300, 768, 784, 1000, 4096, 5001, 20_000])
def test_constant_rows(dtype, d):
    """Zero, whatever the constant and however many there are.  The first mean is off by at most 64 units u of its value (as in
    test_gpu_layer_norm), the correction by at most 64 u of that, and the largest factor behind it is 1 / sqrt(eps)."""
    values = torch.tensor([100.1, 3333.3, 10000.1, -777.7, 0.1], dtype=torch.float64)
    x = values[:, None].expand(5, d).to(dtype).to(DEV).contiguous().requires_grad_()
    bias = torch.full((d,), 0.25, dtype=dtype, device=DEV).requires_grad_()
    w = torch.ones(d, dtype=dtype, device=DEV).requires_grad_()
    dy = torch.randn(5, d, generator=torch.Generator().manual_seed(41)).to(dtype).to(DEV)
    tol = (64 * _unit(dtype)) ** 2 * values.abs()[:, None] / 1e-5 ** 0.5
    y = layer_norm(x, w)
    assert bool((y.detach().double().cpu().abs() <= tol).all())
    # dx = (dy - mean(dy)) / sqrt(eps) and dw = 0: z is zero to the same bound
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    g = dy.double().cpu()
    want = (g - g.mean(1, keepdim=True)) / 1e-5 ** 0.5
    half = torch.finfo(dtype).eps / 2 if dtype.itemsize == 2 else 0.0
    limit = 64 * _unit(dtype) * g.abs().amax(1, keepdim=True) / 1e-5 ** 0.5 + half * want.abs()
    assert bool(((gx.double().cpu() - want).abs() <= limit).all())
    assert bool((gw.double().cpu().abs() <= (g.abs() * tol).sum(0)).all())
    assert torch.equal(layer_norm(x.detach(), w.detach(), bias.detach()).float().sub(0.25).abs() > 1e-3, torch.zeros(5, d, dtype=torch.bool, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("d", [28, 300, 784, 4096, 5001, 20_000])
def test_rows_far_from_zero(dtype, d):
    """Values about 1e4 with a spread of one.  The differences from the first mean are exact; what follows is off by 64 u of the
    differences, and not of the values."""
    g = torch.Generator().manual_seed(42)
    x = (torch.randn(7, d, generator=g) + 1e4).to(dtype)
    dy, w = torch.randn(7, d, generator=g).to(dtype), (torch.randn(d, generator=g) * 0.3 + 1).to(dtype)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w)]
    y = layer_norm(*leaves)
    gx, gw = torch.autograd.grad(y, leaves, dy.to(DEV))
    # (the mean of values about 1e4 is summed in 64 bits relative to 1e4, where it is exact enough for double results too)
    c = x.double() - 1e4
    c = c - c.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
    z = c * rstd
    gw64 = w.double()
    t = dy.double() * gw64
    want = rstd * (t - t.mean(1, keepdim=True) - z * (t * z).mean(1, keepdim=True))
    top, u = z.abs().amax(1, keepdim=True) + 1, 64 * _unit(dtype)
    assert bool(((y.detach().double().cpu() - z * gw64).abs() <= u * top * gw64.abs()).all())
    assert bool(((gx.double().cpu() - want).abs() <= u * rstd * t.abs().amax(1, keepdim=True) * (2 + 2 * top ** 2)).all())
    assert bool(((gw.double().cpu() - (dy.double() * z).sum(0)).abs() <= u * (dy.double().abs() * top).sum(0)).all())
