"""GPU parity of the tokens sorted by expert, and back (mi355moe.dispatch), with their definitions in float64 (oracle/block.py):
the order and the rows bit for bit, sums within bounds computed from their roundings."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _name(dt):
    return str(dt).replace("torch.", "")


def _f64(t):
    return t.detach().double().cpu().numpy()


def _within(got, want, tol, what):
    bad = ~(np.abs(_f64(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], int(bad.sum()))


def _ids(T, k, n, seed, dtype=torch.int32, lo=0, hi=None):
    return torch.randint(lo, n if hi is None else hi, (T, k), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _hold(plan, ids, n, emap=None):
    row, pair, offsets = ref.order(ids.cpu().numpy(), n, None if emap is None else emap.cpu().numpy())
    assert plan.row.dtype == plan.pair.dtype == plan.offsets.dtype == torch.int32
    assert np.array_equal(plan.row.cpu().numpy(), row)
    assert np.array_equal(plan.pair.cpu().numpy(), pair)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    return row, offsets


# T, topk, n: one workgroup (to 4096 pairs) and several, waves of one pair and of whole runs, one expert, many
ORDERS = [(1, 1, 1), (1, 8, 288), (3, 5, 7), (64, 1, 2), (65, 3, 8), (200, 8, 288), (512, 8, 60), (4096, 1, 288), (4097, 1, 288),
          (700, 6, 33), (2048, 8, 288), (1025, 32, 512), (33, 31, 1023), (300, 16, 1024), (90, 8, 2047), (700, 8, 2048), (16500, 8, 96),
          (64, 8, 4096), (1500, 8, 4096), (70000, 2, 5)]


@pytest.mark.parametrize("T,k,n", ORDERS)
def test_order(cuda, T, k, n):
    from mi355moe import dispatch
    ids = _ids(T, k, n, T + k)
    _hold(dispatch.sort_tokens(ids, n), ids, n)
    same = torch.full_like(ids, n - 1)                           # every pair of one expert: the order is the pairs' own
    _hold(dispatch.sort_tokens(same, n), same, n)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k", [(5, 3), (300, 8), (900, 8)])
def test_order_with_dropped_pairs(cuda, T, k, dtype):
    """Ids below zero, at and beyond the last expert; a map that leaves out experts and points outside."""
    from mi355moe import dispatch
    n = 12
    ids = _ids(T, k, n, 1, dtype, -4, 20)
    _hold(dispatch.sort_tokens(ids, n), ids, n)
    emap = torch.tensor([3, -1, 0, 11, 12, 5, -7, 1 << 40, 2, 2, 7, -1, 9], device="cuda")
    _hold(dispatch.sort_tokens(ids, n, expert_map=emap), ids, n, emap)
    _hold(dispatch.sort_tokens(ids, n, expert_map=emap.clamp(-9, 99).int()), ids, n, emap)
    none = torch.full_like(emap, -1)
    plan = dispatch.sort_tokens(ids, n, expert_map=none)
    _hold(plan, ids, n, none)
    assert (plan.offsets == 0).all() and (plan.row < 0).all()
    empty = dispatch.sort_tokens(ids, n, expert_map=emap[:0])
    assert (empty.offsets == 0).all() and (empty.row < 0).all()


def test_order_of_wide_ids(cuda):
    from mi355moe import dispatch
    ids = torch.tensor([[1 << 33, 2], [(1 << 32) + 1, -(1 << 40)]], device="cuda")
    _hold(dispatch.sort_tokens(ids, 4), ids, 4)
    strided = _ids(40, 8, 16, 3)[:, ::2]
    _hold(dispatch.sort_tokens(strided, 16), strided, 16)


# T, topk, n, H: rows of one value, of less than 16 bytes, of no whole 16 bytes, of one and of several workgroups
ROWS = [(1, 1, 1, 1), (1, 8, 288, 4096), (3, 2, 4, 3), (17, 4, 8, 7), (33, 3, 8, 8), (40, 6, 16, 65), (70, 8, 32, 136), (129, 5, 9, 513),
        (31, 8, 12, 1027), (20, 32, 64, 264), (9, 4, 8, 2051), (5, 3, 6, 8200), (600, 8, 60, 72)]


@pytest.mark.parametrize("T,k,n,H", ROWS)
@pytest.mark.parametrize("dt", TYPES)
def test_there_and_back(cuda, T, k, n, H, dt):
    from mi355moe import dispatch
    g = torch.Generator(device="cuda").manual_seed(T + H)
    ids = _ids(T, k, n, H, torch.int32, -1, n + 1)
    plan = dispatch.sort_tokens(ids, n)
    row, _ = _hold(plan, ids, n)
    x = torch.randn(T, H, generator=g, device="cuda").to(dt)
    rows = dispatch.to_experts(x, plan)
    assert np.array_equal(_f64(rows), ref.to_rows(_f64(x), row))
    y = torch.randn(T * k, H, generator=g, device="cuda").to(dt)
    w = torch.randn(T, k, generator=g, device="cuda")
    sh = torch.randn(T, H, generator=g, device="cuda").to(dt)
    dout = torch.randn(T, H, generator=g, device="cuda").to(dt)
    half, tiny = ref.HALF[_name(dt)], ref.TINY[_name(dt)]
    for wt in (torch.float32, dt, torch.float16):
        v = w.to(wt)
        out = dispatch.from_experts(y, v, plan, shared=sh)
        _within(out, *ref.from_rows(_f64(y), _f64(v), row, _f64(sh), half, tiny), "out")
        dy, dw = dispatch.from_experts_backward(dout, y, v, plan)
        (ry, ty), (rw, tw) = ref.from_rows_grads(_f64(dout), _f64(y), _f64(v), row, half, tiny)
        _within(dy, ry, ty, "dy")
        hw = ref.HALF[_name(wt)]
        _within(dw, rw, tw * (1 + hw) + np.abs(rw) * hw + ref.TINY[_name(wt)], "dw")
        assert dy.dtype == dt and dw.dtype == wt
    _within(dispatch.from_experts(y, None, plan), *ref.from_rows(_f64(y), None, row, None, half, tiny), "sum")


@pytest.mark.parametrize("dt", TYPES)
def test_gradients_by_autograd(cuda, dt):
    """The differentiable calls give what the explicit ones do, also where only some inputs need a gradient, and add up over uses."""
    from mi355moe import dispatch
    T, k, n, H = 23, 4, 6, 75
    g = torch.Generator(device="cuda").manual_seed(2)
    plan = dispatch.sort_tokens(_ids(T, k, n, 5, torch.int32, -1, n), n)
    x, y = (torch.randn(r, H, generator=g, device="cuda").to(dt) for r in (T, T * k))
    w, sh = torch.rand(T, k, generator=g, device="cuda"), torch.randn(T, H, generator=g, device="cuda").to(dt)
    drows, dout = torch.randn(T * k, H, generator=g, device="cuda").to(dt), torch.randn(T, H, generator=g, device="cuda").to(dt)
    xr = x.clone().requires_grad_()
    dispatch.to_experts(xr, plan).backward(drows)
    assert torch.equal(xr.grad, dispatch.from_experts(drows, None, plan))
    want = dispatch.from_experts_backward(dout, y, w, plan)
    for need in range(1, 8):
        leaf = [t.clone().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((y, w, sh))]
        out = dispatch.from_experts(leaf[0], leaf[1], plan, shared=leaf[2])
        assert torch.equal(out, dispatch.from_experts(y, w, plan, shared=sh))
        out.backward(dout)
        for i, v in enumerate((*want, dout)):
            assert (leaf[i].grad is None) == (not need >> i & 1) and (leaf[i].grad is None or torch.equal(leaf[i].grad, v))
    yr = y.clone().requires_grad_()
    dispatch.from_experts(yr, None, plan).backward(dout)
    assert torch.equal(yr.grad, dispatch.to_experts(dout, plan))
    dispatch.from_experts(yr, None, plan).sum().backward()       # an expanded gradient, strides 0
    assert torch.equal(yr.grad, (dispatch.to_experts(dout, plan).float() + dispatch.to_experts(torch.ones_like(dout), plan).float()).to(dt))


def test_gradients_against_differences(cuda):
    """Both ways are linear: a difference over any step is the derivative, but for the fp32 roundings of the two ends."""
    from mi355moe import dispatch
    T, k, n, H = 12, 3, 5, 40
    g = torch.Generator(device="cuda").manual_seed(4)
    plan = dispatch.sort_tokens(_ids(T, k, n, 6), n)
    y, v = (torch.randn(T * k, H, generator=g, device="cuda") for _ in range(2))
    w, u = (torch.randn(T, k, generator=g, device="cuda") for _ in range(2))
    dout = torch.randn(T, H, generator=g, device="cuda")
    dy, dw = dispatch.from_experts_backward(dout, y, w, plan)
    f = lambda a, b: float((_f64(dispatch.from_experts(a, b, plan)) * _f64(dout)).sum())  # noqa: E731
    # each end is off by (k + 2) U of at most 40 * T * H, and the inputs' own sums by a rounding
    tol = 2 * 8 * ref.U * 40 * T * H
    assert abs(f(y + v, w) - f(y, w) - float((_f64(dy) * _f64(v)).sum())) <= tol
    assert abs(f(y, w + u) - f(y, w) - float((_f64(dw) * _f64(u)).sum())) <= tol


def test_views_and_strides(cuda):
    from mi355moe import dispatch
    T, k, n = 37, 4, 8
    for H, dt in ((72, torch.bfloat16), (75, torch.float16), (40, torch.float32)):
        plan = dispatch.sort_tokens(_ids(T, k, n, 2), n)
        x, y = torch.randn(T, H, device="cuda").to(dt), torch.randn(T * k, H, device="cuda").to(dt)
        w = torch.rand(T, k, device="cuda")
        rows, out = dispatch.to_experts(x, plan), dispatch.from_experts(y, w, plan, shared=x)
        dy, dw = dispatch.from_experts_backward(x, y, w, plan)
        for off in (0, 1, 3, 8):
            wide = torch.zeros(T, H + 17, dtype=dt, device="cuda")
            wide[:, off:off + H] = x
            v = wide[:, off:off + H]
            assert torch.equal(dispatch.to_experts(v, plan), rows)
            assert torch.equal(dispatch.from_experts(y, w, plan, shared=v), out)
            got = dispatch.from_experts_backward(v, y, w, plan)
            assert torch.equal(got[0], dy) and torch.equal(got[1], dw)
        t = x.t().contiguous().t()
        assert torch.equal(dispatch.to_experts(t, plan), rows)
        assert torch.equal(dispatch.from_experts(y.t().contiguous().t(), w.t().contiguous().t(), plan, shared=t), out)
        base = torch.zeros(T * k * H + 1, dtype=dt, device="cuda")
        base[1:] = y.reshape(-1)
        assert torch.equal(dispatch.from_experts(base[1:].view(T * k, H), w, plan, shared=x), out)
        row = x[:1].expand(T, H)
        assert torch.equal(dispatch.to_experts(row, plan), dispatch.to_experts(row.contiguous(), plan))


def test_dropped_pairs_are_not_read(cuda):
    """NaN and infinities where no expert takes the pair: its row, its weight; and a token all of whose pairs are dropped."""
    from mi355moe import dispatch
    T, k, n, H = 9, 3, 4, 40
    ids = _ids(T, k, n, 8, torch.int32, -1, n)
    ids[4] = -1
    plan = dispatch.sort_tokens(ids, n)
    total = int(plan.offsets[-1])
    y, w = torch.randn(T * k, H, device="cuda").bfloat16(), torch.randn(T, k, device="cuda")
    x, sh = torch.randn(T, H, device="cuda").bfloat16(), torch.randn(T, H, device="cuda").bfloat16()
    out, back = dispatch.from_experts(y, w, plan, shared=sh), dispatch.from_experts_backward(x, y, w, plan)
    y[total:] = float("nan")
    w[plan.row < 0] = float("inf")
    assert torch.equal(dispatch.from_experts(y, w, plan, shared=sh), out) and torch.equal(out[4], sh[4])
    dy, dw = dispatch.from_experts_backward(x, y, w, plan)
    assert torch.equal(dy, back[0]) and torch.equal(dw, back[1]) and (dy[total:] == 0).all() and (dw[4] == 0).all()
    x[4] = float("nan")                                          # a token that nobody takes reaches no row
    assert torch.isfinite(dispatch.to_experts(x, plan)).all()


def test_no_tokens(cuda):
    from mi355moe import dispatch
    plan = dispatch.sort_tokens(torch.empty(0, 4, dtype=torch.int32, device="cuda"), 5)
    assert plan.row.shape == (0, 4) and (plan.offsets == 0).all() and plan.offsets.numel() == 6
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    rows = dispatch.to_experts(x, plan)
    w = torch.empty(0, 4, device="cuda", requires_grad=True)
    out = dispatch.from_experts(rows, w, plan)
    out.sum().backward()
    assert out.shape == (0, 16) and x.grad.shape == (0, 16) and w.grad.shape == (0, 4)


def test_captured_step(cuda):
    """Sort, both ways and both gradients in one graph, replayed with new ids and inputs, eager work between the replays; recording a
    gradient is refused during capture, and the capture survives the refusal."""
    from mi355moe import dispatch
    for T, k, n, H in ((2, 8, 32, 64), (900, 8, 60, 75)):
        ids, g = _ids(T, k, n, 1), torch.Generator(device="cuda").manual_seed(1)
        emap = torch.arange(n, device="cuda")
        new = lambda r, c: torch.randn(r, c, generator=g, device="cuda")  # noqa: E731
        x, y, w, d = new(T, H).bfloat16(), new(T * k, H).bfloat16(), new(T, k), new(T, H).bfloat16()
        leaf = x.clone().requires_grad_()
        alive = dispatch.to_experts(leaf, dispatch.sort_tokens(ids, n))

        def step():
            plan = dispatch.sort_tokens(ids, n, expert_map=emap)
            return (dispatch.to_experts(x, plan), dispatch.from_experts(y, w, plan, shared=x), *dispatch.from_experts_backward(d, y, w, plan),
                    plan.row, plan.offsets)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="capture"):
                dispatch.to_experts(leaf, dispatch.sort_tokens(ids, n))
            outs = step()
        for seed in range(4):
            ids.copy_(_ids(T, k, n, 20 + seed)), emap.copy_(torch.randperm(n, generator=torch.Generator().manual_seed(seed)) - 3)
            x.copy_(new(T, H)), y.copy_(new(T * k, H)), w.copy_(new(T, k)), d.copy_(new(T, H))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))
        alive.sum().backward()
        assert torch.isfinite(leaf.grad).all()


def test_two_streams(cuda):
    from mi355moe import dispatch
    sets = []
    for T, n in ((700, 60), (90, 288)):
        g = torch.Generator(device="cuda").manual_seed(T)
        sets.append((_ids(T, 8, n, T), n, torch.randn(T, 520, generator=g, device="cuda").bfloat16(), torch.rand(T, 8, generator=g, device="cuda")))

    def work(i):
        ids, n, x, w = sets[i]
        plan = dispatch.sort_tokens(ids, n)
        rows = dispatch.to_experts(x, plan)
        return plan.row, rows, dispatch.from_experts(rows, w, plan), *dispatch.from_experts_backward(x, rows, w, plan)

    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(work(i))
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(p, q) for p, q in zip(got[i], want[i]))


def test_rows_beyond_32_bit_offsets(cuda):
    """More than 2^31 values of rows: the last rows are their tokens', and come back."""
    from mi355moe import dispatch
    T, k, n, H = 1 << 16, 8, 4, 4104
    ids = torch.arange(T * k, device="cuda").reshape(T, k) % n
    plan = dispatch.sort_tokens(ids, n)
    x = torch.randn(T, H, device="cuda").bfloat16()
    rows = dispatch.to_experts(x, plan)
    for r in (0, T * k // 2, T * k - 1):
        assert torch.equal(rows[r], x[int(plan.pair[r]) // k])
    w = torch.zeros(T, k, device="cuda")
    w[:, 3] = 1.0
    assert torch.equal(dispatch.from_experts(rows, w, plan), x)
    drows, dw = dispatch.from_experts_backward(x, rows, w, plan)
    last = int(plan.row[T - 1, 3])
    assert torch.equal(drows[last], x[T - 1]) and (drows[int(plan.row[T - 1, 2])] == 0).all()
    want = (x[T - 1].double() ** 2).sum()
    assert abs(float(dw[T - 1, 7]) - float(want)) <= (H / 64 + 17) * ref.U * float(want)
