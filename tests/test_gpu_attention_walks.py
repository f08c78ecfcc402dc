"""``attention`` where a workgroup goes over more tiles than it looks over at once (64), for several heads one after the other, and
where only some of the gradients are wanted."""
import pytest
import torch

from falkon_amd import attention

from attention_ref import check, reference

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda:0"


def _make(b, sq, sk, hq, hk, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((b, sq, hq, d), (b, sk, hk, d), (b, sk, hk, d), (b, sq, hq, d))]


def _run(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, **kw)
    return {"out": out.detach(), **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)))}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["plain", "documents", "prefix"])
def test_more_than_64_tiles_and_shared_heads(dtype, kind):
    """4500 keys of 64 a tile (2300 of 32) for few queries, and as many queries for few keys, two heads sharing a key head.  Enough
    batches that tiles are not divided among workgroups."""
    n = 2300 if dtype == torch.float32 else 4500
    for sq, sk in ((40, n), (n, 40), (n, n)):
        if kind == "documents" and sq > sk or sq == sk and kind == "plain":
            continue
        b = 1 if sq == sk else 520 if sq < sk else 260
        if sq == sk:                                                         # the first walk over, the heads behind it start again
            q, k, v, do = _make(1, sq, sk, 16, 2, 16, dtype, 60)
        else:
            q, k, v, do = _make(1, sq, sk, 2, 1, 16, dtype, 60)
            q, k, v, do = (t.expand(b, *t.shape[1:]) for t in (q, k, v, do))
        kw = dict(causal=kind == "prefix" or sq == sk)
        if kind == "documents":
            kw["documents"] = (torch.arange(sk, device=DEV) % 2)[None].expand(b, sk)
        if kind == "prefix":
            kw["prefix"] = torch.full((b,), 30, device=DEV)
        got = _run(q, k, v, do, **kw)
        for n_ in got:
            assert torch.equal(got[n_], got[n_][:1].expand_as(got[n_]))
        one = {k_: v_[:1] if torch.is_tensor(v_) else v_ for k_, v_ in kw.items()}
        heads = slice(None) if sq != sk else slice(8, 16)                    # (one key head's, for the time that the reference takes)
        mine = slice(None) if sq != sk else slice(1, 2)
        want = reference(q[:1, :, heads], k[:1, :, mine], v[:1, :, mine], do[:1, :, heads], **one)
        check({"out": got["out"][:1, :, heads], "dq": got["dq"][:1, :, heads], "dk": got["dk"][:1, :, mine], "dv": got["dv"][:1, :, mine]},
              want, ["out", "dq", "dk", "dv"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,sk,hq", [(300, 300, 4), (1000, 1500, 2)])
def test_some_of_the_gradients(dtype, sq, sk, hq):
    """Each is the same to the last bit whichever others are wanted."""
    q, k, v, do = _make(1, sq, sk, hq, 2, 64, dtype, 61)
    slopes = torch.full((hq,), 0.01, device=DEV)
    full = [t.detach().requires_grad_() for t in (q, k, v, slopes)]
    want = torch.autograd.grad(attention(*full[:3], slopes=full[3], causal=True), full, do)
    plain = torch.autograd.grad(attention(*full[:3], slopes=slopes, causal=True), full[:3], do)
    for wanted in ((0,), (1,), (2,), (3,), (1, 2), (0, 2), (1, 3), (0, 3)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v, slopes))]
        got = torch.autograd.grad(attention(*leaves[:3], slopes=leaves[3], causal=True), [leaves[i] for i in wanted], do)
        of = want if 3 in wanted else plain                                  # (rows are not divided where the slopes' gradient is wanted)
        for i, t in zip(wanted, got):
            assert torch.equal(t, of[i])
