"""What the differentiable calls around a layer's experts keep for the backward pass, and what their gradients copy and allocate: only
what some gradient that is asked for reads. What is not kept may be freed or changed in place."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

MB = 1 << 20


def _peak(f):
    """Bytes that f takes at most beside what is there before it."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, out


def _order(T, k, n):
    from mi355moe import dispatch
    return dispatch.sort_tokens(torch.randint(0, n + 2, (T, k), generator=torch.Generator().manual_seed(1)).cuda(), n)


@pytest.mark.parametrize("weights", ["none", "frozen", "learned"])
def test_rows_back_keep_rows_for_the_weights_only(cuda, weights):
    from mi355moe import dispatch
    T, k, H = 256, 4, 512
    plan = _order(T, k, 6)
    g = torch.Generator(device="cuda").manual_seed(2)
    leaf = torch.randn(T * k, H, generator=g, device="cuda").bfloat16().requires_grad_()
    w = None if weights == "none" else torch.rand(T, k, generator=g, device="cuda")
    d = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    want = dispatch.from_experts_backward(d, leaf.detach(), torch.ones(T, k, device="cuda") if w is None else w, plan)
    if weights == "learned":
        w.requires_grad_()
    rows = leaf * 1.0
    out = dispatch.from_experts(rows, w, plan)
    with torch.no_grad():
        rows.mul_(3.0)
    if weights == "learned":
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.backward(d)
        return
    out.backward(d)
    assert torch.equal(leaf.grad, want[0])
    if w is not None:                                            # nothing but shared's gradient is asked for: dout, whatever they become
        shared = d.clone().requires_grad_()
        rows, w2 = leaf.detach().clone(), w.clone()
        out = dispatch.from_experts(rows, w2, plan, shared)
        rows.mul_(3.0), w2.mul_(2.0)
        out.backward(d)
        assert torch.equal(shared.grad, d)
    # and the rows are freed
    leaf.grad = None
    rows = (leaf * 1.0)
    out = dispatch.from_experts(rows, w, plan)
    before = torch.cuda.memory_allocated()
    del rows
    assert before - torch.cuda.memory_allocated() >= T * k * H * 2
    out.backward(d)
    assert torch.equal(leaf.grad, want[0])


def test_rows_backward_reads_rows_for_the_weights_only(cuda):
    """Strided rows are copied where dweights reads them, and there alone."""
    from mi355moe import dispatch
    T, k, H = 1024, 4, 1024
    plan = _order(T, k, 6)
    wide = torch.randn(T * k, H + 8, device="cuda").bfloat16()
    rows, w, d = wide[:, :H], torch.rand(T, k, device="cuda"), torch.randn(T, H, device="cuda").bfloat16()
    both = dispatch.from_experts_backward(d, rows, w, plan)
    bytes_, (drows, dw) = _peak(lambda: dispatch.from_experts_backward(d, rows, w, plan, need_weights=False))
    assert dw is None and torch.equal(drows, both[0]) and drows.is_contiguous()
    assert bytes_ < T * k * H * 2 + MB
    drows, dw = dispatch.from_experts_backward(d, rows, w, plan, need_rows=False)
    assert drows is None and torch.equal(dw, both[1])


def test_linear_gradients_copy_only_what_they_read(cuda):
    """An operand that the kernels cannot read where it lies is copied for the product that reads it, and for no other."""
    from mi355moe import ffn
    M, K, N = 2048, 1024, 1024
    x, w, d = (torch.randn(*s, device="cuda").bfloat16() for s in ((M, K), (N, K), (M, N)))
    odd = lambda t: torch.cat([t[:, :1], t], 1)[:, 1:]  # noqa: E731
    want = ffn.linear_backward(d, None, x, w)
    for need, bad in (((True, False), (odd(x), w)), ((False, True), (x, odd(w)))):
        plain, _ = _peak(lambda: ffn.linear_backward(d, None, x, w, None, None, *need))
        moved, got = _peak(lambda: ffn.linear_backward(d, None, *bad, None, None, *need))
        assert moved == plain, (need, moved, plain)
        assert all(p is None or torch.equal(p, q) for p, q in zip(got, want))
