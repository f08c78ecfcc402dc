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
