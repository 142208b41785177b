"""What the Python layer of the operators around a layer's experts refuses, and the derivatives that they do not have."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


def _bad(f, *args, match=None, **kw):
    with pytest.raises(ValueError, match=match):
        f(*args, **kw)


def test_dispatch_refusals(cuda):
    from mi355moe import _lib, dispatch
    ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    for bad in (ids.float(), ids.short(), ids[0], ids[:, :0], ids[None]):
        _bad(dispatch.sort_tokens, bad, 4)
    for m in (torch.zeros(4, device="cuda"), torch.zeros(2, 2, dtype=torch.int64, device="cuda"), torch.ones(4, dtype=torch.bool, device="cuda")):
        _bad(dispatch.sort_tokens, ids, 4, expert_map=m, match="expert_map")
    for n in (0, -3, 4097):
        with pytest.raises(_lib.MoeError):
            dispatch.sort_tokens(ids, n)
    with pytest.raises(_lib.MoeError):
        dispatch.sort_tokens(torch.zeros(3, 33, dtype=torch.int32, device="cuda"), 4)
    plan = dispatch.sort_tokens(ids, 4)
    x, rows, w = torch.zeros(3, 8, device="cuda"), torch.zeros(6, 8, device="cuda"), torch.zeros(3, 2, device="cuda")
    for bad in (x[:2], x[0], x[:, :0], x.double(), x.int()):
        _bad(dispatch.to_experts, bad, plan)
    for bad in (rows[:5], rows[0], rows.double()):
        _bad(dispatch.from_experts, bad, w, plan)
    for bad in (w[:2], w.t(), w.reshape(-1), w.int(), w.double()):
        _bad(dispatch.from_experts, rows, bad, plan)
        _bad(dispatch.from_experts_backward, x, rows, bad, plan)
    for bad in (x[:2], x.half(), x[:, :7]):
        _bad(dispatch.from_experts, rows, w, plan, shared=bad)
        _bad(dispatch.from_experts_backward, bad, rows, w, plan)
    _bad(dispatch.from_experts, rows.cpu(), w, plan, match="GPU")


def test_linear_refusals(cuda):
    from mi355moe import _lib, ffn
    x, w = torch.zeros(3, 8, device="cuda").half(), torch.zeros(5, 8, device="cuda").half()
    b, r = torch.zeros(5, device="cuda"), torch.zeros(3, 5, device="cuda").half()
    for a in ((x.float(), w.float()), (x.bfloat16(), w), (x[:, :7], w), (x, w[0]), (x, w[:0]), (x, w[:, :0]), (x.sum(), w)):
        _bad(ffn.linear, *a)
    for bad in (b[:4], b[None], b.double(), b.int()):
        _bad(ffn.linear, x, w, bias=bad)
    for bad in (r[:2], r[:, :4], r.float(), r[None]):
        _bad(ffn.linear, x, w, residual=bad)
    for bad in ("SiLU", "tanh", "", 1):
        _bad(ffn.linear, x, w, activation=bad, match="activation")
    z = torch.zeros(3, 5, device="cuda")
    for bad in (None, z.half(), z[:2], z.t().contiguous().t(), z.reshape(-1)):
        _bad(ffn.linear_backward, r, bad, x, w, "silu", match="z must be")
    _bad(ffn.linear_backward, r.float(), z, x, w)
    _bad(ffn.linear_backward, r[:, :4], z, x, w)
    _bad(ffn.linear_backward, r, z, x, w, "silu", torch.int32)
    with pytest.raises(_lib.MoeError):
        ffn.linear(torch.zeros(1, 65537, device="cuda").half(), torch.zeros(1, 65537, device="cuda").half())


def test_norm_refusals(cuda):
    from mi355moe import _lib, norm
    b, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda")
    _bad(norm.join, b.double())
    _bad(norm.join, b.sum())
    _bad(norm.join, b[:, :0])
    for bad in (b[:2], b.half(), b[0]):
        _bad(norm.join, b, bad)
    for bad in (w[:7], w[None], w.double(), w.int()):
        _bad(norm.join, b, post=bad)
        _bad(norm.join, b, pre=bad)
        _bad(norm.rms, b, bad)
    _bad(norm.join, b, post=w, pre=w.half(), match="post is")
    for bad in (w[:7], b[:2], b[:, :2], torch.zeros(1, 8, device="cuda"), w.int(), torch.zeros(3, device="cuda")):
        _bad(norm.join, b, gate=bad)
    _bad(norm.rms, b, None)
    _bad(norm.join_forward, b, need_s=False)
    for eps in (-1e-6, float("nan")):
        with pytest.raises(_lib.MoeError):
            norm.rms(b, w, eps=eps)
    _, _, stats = norm.join_forward(b, pre=w)
    _bad(norm.join_backward, b.half(), None, stats, b, pre=w)
    _bad(norm.join_backward, b[:2], None, stats, b, pre=w)
    _bad(norm.join_backward, None, b, stats, b, match="without pre")
    for bad in (stats[:2], stats.half(), stats.t().contiguous().t(), stats.reshape(-1)):
        _bad(norm.join_backward, b, None, bad, b, pre=w, match="stats")
    with pytest.raises(_lib.MoeError):
        norm.rms(torch.zeros(1, 16385, device="cuda"), torch.zeros(16385, device="cuda"))


def _calls():
    """For each differentiable call its inputs, and what it does with them."""
    from mi355moe import dispatch, ffn, norm
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    plan = dispatch.sort_tokens(torch.tensor([[0, 1], [2, 0], [1, 2]], device="cuda"), 3)
    return [((new(3, 8),), lambda x: dispatch.to_experts(x, plan)),
            ((new(6, 8), new(3, 2), new(3, 8)), lambda r, w, s: dispatch.from_experts(r, w, plan, shared=s)),
            ((new(3, 8).half(), new(16, 8).half(), new(16), new(3, 16).half()), lambda x, w, b, r: ffn.linear(x, w, b, "silu", r)),
            ((new(3, 8), new(3, 8), new(8), new(8), new(8)), lambda b, r, p, t, w: norm.join(b, r, post=p, gate=t, pre=w)[1]),
            ((new(3, 8), new(8)), lambda x, w: norm.rms(x, w))]


def test_forward_mode_is_refused(cuda):
    for inputs, f in _calls():
        want = f(*inputs)
        with fwd.dual_level():
            for i, t in enumerate(inputs):
                for rest in (False, True):
                    args = [fwd.make_dual(t, torch.ones_like(t)) if j == i else u.clone().requires_grad_(rest) for j, u in enumerate(inputs)]
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(*args)
                    with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                        f(*args)
            assert torch.equal(f(*inputs), want)


def test_second_derivatives_are_refused(cuda):
    """A recorded backward pass gives the first derivatives, and refuses to be differentiated."""
    for inputs, f in _calls():
        leaf = [t.clone().requires_grad_() for t in inputs]
        out = f(*leaf)
        d = torch.ones_like(out).requires_grad_()
        plain = torch.autograd.grad(out, leaf, d.detach(), retain_graph=True)
        first = torch.autograd.grad(out, leaf, d, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, plain))
        with pytest.raises(RuntimeError, match="once_differentiable"):
            sum(v.float().sum() for v in first if v.grad_fn is not None and v.grad_fn is not d.grad_fn).backward()


def test_inputs_changed_in_place_are_noticed(cuda):
    for inputs, f in _calls()[1:]:
        leaf = [t.clone().requires_grad_() for t in inputs]
        kept = leaf[0].clone()
        out = f(kept, *leaf[1:])
        with torch.no_grad():
            kept.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            out.sum().backward()


def test_saved_tensors_may_move(cuda):
    """Saved tensors packed and unpacked by hooks (as activation offloading and checkpointing do) come back elsewhere in memory."""
    for inputs, f in _calls():
        leaf = [t.clone().requires_grad_() for t in inputs]
        want = torch.autograd.grad(f(*leaf), leaf, torch.ones_like(f(*inputs)))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
            out = f(*leaf)
        got = torch.autograd.grad(out, leaf, torch.ones_like(out))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_refused_order_takes_no_memory(cuda):
    from mi355moe import _lib, dispatch
    ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    far = torch.zeros(1, dtype=torch.int32, device="cuda").expand(1 << 20, 32)
    torch.cuda.synchronize()
    for bad, n in ((ids, 10 ** 12), (ids, 1 << 30), (ids, -10 ** 12), (far[:, :17], 4)):
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with pytest.raises(_lib.MoeError):
            dispatch.sort_tokens(bad, n)
        assert torch.cuda.max_memory_allocated() - before <= 4 * bad.numel() + (1 << 20)     # (the ids' copy, where they are a view)
