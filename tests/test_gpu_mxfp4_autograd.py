"""The routed experts next to a shared expert that is tuned: its gradient passes through the sum, the experts' own is refused."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _setup(T, dt=torch.bfloat16):
    from mi355moe import mxfp4
    g = torch.Generator(device="cuda").manual_seed(3)
    n, H, I = 8, 256, 64
    ex = mxfp4.Mxfp4Experts.from_dense(torch.randn(n, 2 * I, H, generator=g, device="cuda") * 0.2,
                                       torch.randn(n, H, I, generator=g, device="cuda") * 0.2)
    x = torch.randn(T, H, generator=g, device="cuda").to(dt)
    ids = torch.randint(0, n, (T, 3), generator=g, device="cuda")
    w = torch.rand(T, 3, generator=g, device="cuda")
    w13 = (torch.randn(2 * I, H, generator=g, device="cuda") * 0.1).to(dt)
    w2 = (torch.randn(H, I, generator=g, device="cuda") * 0.1).to(dt)
    return ex, x, ids, w, w13, w2


@pytest.mark.parametrize("T", [3, 70])
def test_tuned_shared_expert(cuda, T):
    """out of autograd with the routed sum added: the gradients are those of the shared expert alone, and a later write is
    noticed by whoever keeps out."""
    from mi355moe import ffn, mxfp4
    ex, x, ids, w, w13, w2 = _setup(T)
    c = torch.randn(T, 256, device="cuda").bfloat16()
    grads = []
    for fold in (False, True):
        xr, w1, wd = x.clone().requires_grad_(), w13.clone().requires_grad_(), w2.clone().requires_grad_()
        out = torch.nn.functional.linear(ffn.gated(xr, w1, 10.0), wd)
        before = out.detach().clone()
        if fold:
            got = mxfp4.moe_forward_ids(ex, xr.detach(), ids, w, out=out, accumulate=True)
            assert got is out and not torch.equal(out.detach(), before)
        (out * c).sum().backward()
        grads.append((xr.grad, w1.grad, wd.grad))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    y = torch.zeros(T, 256, device="cuda").bfloat16()
    p = torch.ones(256, device="cuda").bfloat16().requires_grad_()
    keeps = y * p                                            # keeps y for p's gradient
    mxfp4.moe_forward_ids(ex, x, ids, w, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        keeps.sum().backward()


@pytest.mark.parametrize("T", [3, 70])
def test_gradients_of_the_routed_experts(cuda, T):
    from mi355moe import fused_experts_mxfp4, mxfp4
    ex, x, ids, w, _, _ = _setup(T)
    want = mxfp4.moe_forward_ids(ex, x, ids, w)
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    for a, b in ((xr, w), (x, wr)):
        for r in (mxfp4.moe_forward_ids(ex, a, ids, b), fused_experts_mxfp4(a, ex.w13, ex.w2, b, ids, (ex.w13_scale, ex.w2_scale))):
            assert torch.equal(r, want)
            with pytest.raises(RuntimeError, match="no gradient"):
                r.sum().backward()
        for acc in (False, True):
            with pytest.raises(RuntimeError, match="gradient"):
                mxfp4.moe_forward_ids(ex, a, ids, b, out=torch.zeros_like(x), accumulate=acc)
    with torch.no_grad():
        out = torch.zeros_like(x)
        assert torch.equal(mxfp4.moe_forward_ids(ex, xr, ids, wr, out=out), want)
    leaf = torch.zeros_like(x).requires_grad_()
    for out, acc in ((leaf, False), (leaf, True), (leaf * 1, False)):
        with pytest.raises(RuntimeError, match="gradient"):
            mxfp4.moe_forward_ids(ex, x, ids, w, out=out, accumulate=acc)


def test_matmul_out(cuda):
    from mi355moe import mxfp4
    q, s = mxfp4.quant_rows(torch.randn(5, 64, device="cuda"))
    out = torch.zeros(5, 5, device="cuda")
    v = out._version
    mxfp4.matmul(q, s, q, s, out=out)
    assert out._version > v
    for o in (out.clone().requires_grad_(), out.clone().requires_grad_() * 1):
        with pytest.raises(RuntimeError, match="gradient"):
            mxfp4.matmul(q, s, q, s, out=o)
