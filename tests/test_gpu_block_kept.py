"""What the differentiable calls around a layer's experts keep for the backward pass, and what their gradients copy and allocate: only
what some gradient that is asked for reads. What is not kept may be freed or changed in place."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

MB = 1 << 20          # (torch's allocator may count up to 1 MB more for a tensor: a block whose rest is smaller is not split)


def _peak(f):
    """Bytes that f takes at most beside what is there before it."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before, out


def _held(f):
    """(f's results, the bytes that stay allocated with them)."""
    before = torch.cuda.memory_allocated()
    out = f()
    return out, torch.cuda.memory_allocated() - before


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
    T, k, H = 1024, 4, 2048
    plan = _order(T, k, 6)
    wide = torch.randn(T * k, H + 8, device="cuda").bfloat16()
    rows, w, d = wide[:, :H], torch.rand(T, k, device="cuda"), torch.randn(T, H, device="cuda").bfloat16()
    both = dispatch.from_experts_backward(d, rows, w, plan)
    bytes_, (drows, dw) = _peak(lambda: dispatch.from_experts_backward(d, rows, w, plan, need_weights=False))
    assert dw is None and torch.equal(drows, both[0]) and drows.is_contiguous()
    assert bytes_ < T * k * H * 2 + 2 * MB
    drows, dw = dispatch.from_experts_backward(d, rows, w, plan, need_rows=False)
    assert drows is None and torch.equal(dw, both[1])


def test_linear_gradients_copy_only_what_they_read(cuda):
    """An operand that the kernels cannot read where it lies is copied for the product that reads it, and for no other."""
    from mi355moe import ffn
    M, K, N = 4096, 2048, 4096
    x, w, d = (torch.randn(*s, device="cuda").bfloat16() for s in ((M, K), (N, K), (M, N)))
    odd = lambda t: torch.cat([t[:, :1], t], 1)[:, 1:]  # noqa: E731
    want = ffn.linear_backward(d, None, x, w)
    for need, bad in (((True, False), (odd(x), w)), ((False, True), (x, odd(w)))):
        plain, _ = _peak(lambda: ffn.linear_backward(d, None, x, w, None, None, *need))
        moved, got = _peak(lambda: ffn.linear_backward(d, None, *bad, None, None, *need))
        assert abs(moved - plain) < 4 * MB, (need, moved, plain)     # (a copy has 16 MB)
        assert all(p is None or torch.equal(p, q) for p, q in zip(got, want))


def test_linear_keeps_what_its_gradients_read(cuda):
    """x for w's gradient, w for x's, z for x's, w's and the bias' where there is an activation."""
    from mi355moe import ffn
    M, K, N = 1024, 512, 1024
    g = torch.Generator(device="cuda").manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    base = {"x": new(M, K).bfloat16(), "w": (new(N, K) / 16).bfloat16(), "bias": new(N), "residual": new(M, N).bfloat16()}
    d = new(M, N).bfloat16()
    for act in (None, "silu"):
        out, z = ffn.linear_forward(*(base[k] for k in ("x", "w", "bias")), act, base["residual"], save=True)
        grads = ffn.linear_backward(d, z, base["x"], base["w"], act, torch.float32)
        want = dict(zip(("x", "w", "bias"), grads), residual=d)
        for asked in (("x",), ("w",), ("bias",), ("residual",), ("x", "residual"), ("bias", "residual"), ("x", "w"), ("w", "bias"), tuple(base)):
            # what is asked for is not a leaf, so that it may be changed in place
            leaf = {k: base[k].clone().requires_grad_(k in asked) for k in base}
            used = {k: leaf[k] * 1.0 for k in base}

            def call():
                return ffn.linear(used["x"], used["w"], used["bias"], act, used["residual"])

            y, held = _held(call)
            assert torch.equal(y, out)
            kept_z = act is not None and any(k in asked for k in ("x", "w", "bias"))
            assert (held >= M * N * 6) == kept_z, (act, asked, held)
            read = [k for k, by in (("x", "w"), ("w", "x")) if by in asked]
            with torch.no_grad():
                for k in base:
                    if k not in read:
                        used[k].mul_(2.0)
            y.backward(d, retain_graph=True)
            for k in base:
                assert (leaf[k].grad is None) == (k not in asked)
                assert k not in asked or torch.equal(leaf[k].grad, want[k]), (act, asked, k)
            if read:
                with torch.no_grad():
                    used[read[0]].mul_(2.0)
                with pytest.raises(RuntimeError, match="modified by an inplace"):
                    y.backward(d)
    # no gradient of three dimensions, or of no rows, needs the other operand either
    x3 = base["x"].reshape(4, M // 4, K).clone().requires_grad_()
    y = ffn.linear(x3, base["w"])
    y.backward(d.reshape(4, M // 4, N))
    assert torch.equal(x3.grad.reshape(M, K), ffn.linear_backward(d, None, base["x"], base["w"])[0])
    w = base["w"].clone().requires_grad_()
    ffn.linear(base["x"][:0], w).sum().backward()
    assert w.grad.shape == (N, K) and not w.grad.any()
    x0 = base["x"][:0].clone().requires_grad_()
    ffn.linear(x0, base["w"]).sum().backward()
    assert x0.grad.shape == (0, K)


def test_linear_gradients_take_the_scratch_they_use(cuda):
    """Without an activation dout is an operand as it is, without a copy; copies of x and w (K no multiple of 8) are made for the
    product that reads them. (Outputs of more than 512 tiles of 128 x 128: no product is cut into parts.)"""
    from mi355moe import ffn
    M, N, slack = 4096, 4096, 4 * MB
    for K in (2560, 2563):
        K8 = (K + 7) // 8 * 8
        assert M * K > 512 * 128 * 128 and N * K > 512 * 128 * 128
        cx, cw = (0, 0) if K == K8 else (2 * M * K8, 2 * N * K8)
        x, w, d = (torch.randn(*s, device="cuda").bfloat16() for s in ((M, K), (N, K), (M, N)))
        rows = 4 * (M // 64) * N                                 # the bias' sums
        want = ffn.linear_backward(d, None, x, w, None, torch.float32)
        for dx, dw, db in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
            peak, got = _peak(lambda: ffn.linear_backward(d, None, x, w, None, torch.float32 if db else None, bool(dx), bool(dw)))
            assert peak < dx * (2 * M * K + cw) + dw * (2 * N * K + cx) + db * (rows + 4 * N) + slack, (K, dx, dw, db, peak)
            assert all(p is None or torch.equal(p, q) for p, q in zip(got, want))
        # an operand that is no 16-byte rows, and an activation's slope, take dz
        z = torch.randn(M, N, device="cuda")
        for dout, act in ((torch.cat([d[:, :1], d], 1)[:, 1:], None), (d, "silu")):
            peak, got = _peak(lambda: ffn.linear_backward(dout, z, x, w, act, need_dw=False))
            assert 2 * M * N <= peak - 2 * M * K - cw < 2 * M * N + slack
            assert act is not None or torch.equal(got[0], want[0])


def test_a_sum_without_a_norm_behind_it_keeps_no_residual(cuda):
    from mi355moe import norm
    g = torch.Generator(device="cuda").manual_seed(4)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    b, r, post, gate, ds = new(300, 520), new(300, 520), new(520), new(520), new(300, 520)
    _, _, stats = norm.join_forward(b, r, post, gate, scale=0.5, residual_scale=1.5)
    want = norm.join_backward(ds, None, stats, b, r, post, gate, None, 0.5, 1.5)
    leaf = [t.clone().requires_grad_() for t in (b, r, post, gate)]
    stream = leaf[1] * 1.0
    s = norm.join(leaf[0], stream, post=leaf[2], gate=leaf[3], scale=0.5, residual_scale=1.5)
    with torch.no_grad():
        stream.add_(1.0)                                         # the residual stream goes on in place
    s.backward(ds)
    assert all(torch.equal(t.grad, v) for t, v in zip(leaf, want))
    # the explicit form without dy reads no residual either, and gives its gradient where there is one
    some = new(4096, 2048).t()
    _, _, stats = norm.join_forward(some, some)
    d = new(2048, 4096)
    full, want = _peak(lambda: norm.join_backward(d, None, stats, some, some.contiguous(), residual_scale=1.5))
    peak, got = _peak(lambda: norm.join_backward(d, None, stats, some, some, residual_scale=1.5))
    assert all(p is q or torch.equal(p, q) for p, q in zip(got, want)) and torch.equal(got[1], 1.5 * d)
    assert peak < full - 24 * MB, (peak, full)                   # (a copy has 32 MB)
    assert norm.join_backward(d, None, stats, some, None)[1] is None
