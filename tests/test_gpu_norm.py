"""GPU parity of the norms around a block (mi355moe.norm) and their gradients with their definitions in float64 (oracle/block.py),
within bounds computed from the roundings of the fp32 evaluation and of the results."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
NAMES = ("branch", "residual", "post", "gate", "pre")


def _name(dt):
    return str(dt).replace("torch.", "")


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _within(got, want, tol, what):
    bad = ~(np.abs(_f64(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], int(bad.sum()))


def _inputs(R, H, gate, dt, wt, gt, seed, parts="brpw"):
    """The five tensors (None where `parts` leaves one out: b, r residual, p post, w pre) and two gradients."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = {"branch": (new(R, H) * 0.7 + 0.1).to(dt), "residual": (new(R, H) * 3).to(dt) if "r" in parts else None,
         "post": (1 + 0.3 * new(H)).to(wt) if "p" in parts else None,
         "gate": None if gate is None else new(*{"channel": (H,), "token": (R, 1), "full": (R, H)}[gate]).to(gt),
         "pre": (1 + 0.3 * new(H)).to(wt) if "w" in parts else None}
    return t, new(R, H).to(dt), new(R, H).to(dt)


def _hold_grads(got, t, ds, dy, kw, R):
    want = ref.norm_grads(_f64(ds), _f64(dy), *(_f64(t[k]) for k in NAMES), kw["eps"], kw["scale"], kw["residual_scale"])
    for k, v in zip(NAMES, got):
        if t[k] is None:
            assert v is None
        elif k in want:
            d = _name(t[k].dtype)
            value, mag = want[k]
            assert v.dtype == t[k].dtype and v.shape == t[k].shape
            e = (256 + R) * ref.U * mag
            _within(v, value, e * (1 + ref.HALF[d]) + ref.HALF[d] * np.abs(value) + ref.TINY[d], "d" + k)
        else:
            assert (v == 0).all()


# rows, H: a wave a row, a workgroup a row, every kernel size and its edges, rows of one value
SIZES = [(1, 1), (3, 7), (5, 64), (9, 511), (4, 512), (7, 513), (1, 1024), (17, 1031), (6, 2048), (5, 2056), (3, 4096), (1, 4099), (2, 8192),
         (3, 8200), (2, 16384), (1500, 72), (1100, 520)]


@pytest.mark.parametrize("R,H", SIZES)
@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
@pytest.mark.parametrize("dt", TYPES)
def test_forward_and_gradients(cuda, R, H, gate, dt):
    from mi355moe import norm
    i = SIZES.index((R, H)) + len(gate or "")
    wt, gt = TYPES[i % 3], TYPES[(i // 3) % 3]
    t, ds, dy = _inputs(R, H, gate, dt, wt, gt, R + H)
    kw = dict(eps=1e-5, scale=0.5, residual_scale=1.25)
    s, y, stats = norm.join_forward(t["branch"], t["residual"], t["post"], t["gate"], t["pre"], **kw)
    d = _name(dt)
    f = [_f64(t[k]) for k in NAMES]
    (ws, es), (wy, ey) = ref.norm(*f, 1e-5, 0.5, 1.25, ref.HALF[d], ref.TINY[d])
    _within(s, ws, es, "s")
    _within(y, wy, ey, "y")
    got = norm.join_backward(ds, dy, stats, t["branch"], t["residual"], t["post"], t["gate"], t["pre"], 0.5, 1.25)
    _hold_grads(got, t, ds, dy, kw, R)
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    out = norm.join(leaf["branch"], leaf["residual"], post=leaf["post"], gate=leaf["gate"], pre=leaf["pre"], **kw)
    assert torch.equal(out[0], s) and torch.equal(out[1], y)
    torch.autograd.backward(out, (ds, dy))
    for k, v in zip(NAMES, got):
        assert v is None or torch.equal(leaf[k].grad, v), k


# several rows a wave (8, 16, 32 or 64 lanes each) with a last workgroup that is part full, and more rows than the gradient has at once
SHORT = [(1, 8), (70, 64), (69, 65), (37, 128), (35, 129), (18, 256), (33, 257), (7, 505), (40000, 33), (20000, 100), (5000, 300)]


@pytest.mark.parametrize("R,H", SHORT)
@pytest.mark.parametrize("dt", TYPES)
def test_short_rows(cuda, R, H, dt):
    from mi355moe import norm
    i = SHORT.index((R, H))
    for gate in ("channel", "token") if R > 100 else (None, "channel", "token", "full"):
        t, ds, dy = _inputs(R, H, gate, dt, TYPES[i % 3], TYPES[(i + 1) % 3], R)
        kw = dict(eps=1e-5, scale=0.5, residual_scale=1.25)
        args = [t[k] for k in NAMES]
        s, y, stats = norm.join_forward(*args, **kw)
        (ws, es), (wy, ey) = ref.norm(*(_f64(v) for v in args), 1e-5, 0.5, 1.25, ref.HALF[_name(dt)], ref.TINY[_name(dt)])
        _within(s, ws, es, "s")
        _within(y, wy, ey, "y")
        got = norm.join_backward(ds, dy, stats, *args, 0.5, 1.25)
        _hold_grads(got, t, ds, dy, kw, R)
        again = norm.join_backward(ds, dy, stats, *args, 0.5, 1.25)
        assert all(a is b or torch.equal(a, b) for a, b in zip(got, again))
        # a row's gradients are its own, whatever rows stand beside it
        alone = norm.join_backward(ds[R // 2:R // 2 + 1], dy[R // 2:R // 2 + 1], stats[R // 2:R // 2 + 1], args[0][R // 2:R // 2 + 1],
                                   args[1][R // 2:R // 2 + 1], args[2], args[3] if gate in (None, "channel") else args[3][R // 2:R // 2 + 1],
                                   args[4], 0.5, 1.25)
        assert torch.equal(alone[0][0], got[0][R // 2]) and torch.equal(alone[1][0], got[1][R // 2])


@pytest.mark.parametrize("parts", ["b", "br", "bp", "bw", "brp", "brw", "bpw", "brpw"])
@pytest.mark.parametrize("R,H", [(5, 72), (3, 1029), (700, 264)])
def test_every_set_of_parts(cuda, parts, R, H):
    """Each part left out, each gradient asked for alone, ds or dy missing."""
    from mi355moe import norm
    dt = torch.bfloat16
    for gate in (None, "channel", "token", "full"):
        t, ds, dy = _inputs(R, H, gate, dt, torch.float32, dt, 3, parts)
        kw = dict(eps=1e-6, scale=1.5, residual_scale=0.75)
        args = [t[k] for k in NAMES]
        s, y, stats = norm.join_forward(*args, **kw)
        f = [_f64(v) for v in args]
        (ws, es), want = ref.norm(*f, 1e-6, 1.5, 0.75, ref.HALF["bfloat16"], ref.TINY["bfloat16"])
        _within(s, ws, es, "s")
        assert (y is None) == (want is None)
        if want:
            _within(y, *want, "y")
            alone = norm.join_forward(*args, **kw, need_s=False)
            assert alone[0] is None and torch.equal(alone[1], y) and torch.equal(alone[2], stats)
        for a, b in ((ds, dy), (ds, None), (None, dy)):
            if t["pre"] is None and b is not None or a is None and b is None:
                continue
            got = norm.join_backward(a, b, stats, *args, 1.5, 0.75)
            _hold_grads(got, t, a, b, kw, R)
            for i in range(5):
                need = tuple(i == j for j in range(5))
                one = norm.join_backward(a, b, stats, *args, 1.5, 0.75, need=need)
                assert all(v is None or j == i for j, v in enumerate(one))
                assert one[i] is None or torch.equal(one[i], got[i])


def test_rms(cuda):
    from mi355moe import norm
    for dt in TYPES:
        t, _, dy = _inputs(33, 200, None, dt, torch.float32, dt, 1, "bw")
        x, w = t["branch"].clone().requires_grad_(), t["pre"].clone().requires_grad_()
        y = norm.rms(x, w, eps=1e-5)
        _, want = ref.norm(_f64(x), None, None, None, _f64(w), 1e-5, 1.0, 1.0, ref.HALF[_name(dt)], ref.TINY[_name(dt)])
        _within(y, *want, "y")
        y.backward(dy)
        _, _, stats = norm.join_forward(x, None, None, None, w, 1e-5)
        got = norm.join_backward(None, dy, stats, x, None, None, None, w)
        _hold_grads(got, t, None, dy, dict(eps=1e-5, scale=1.0, residual_scale=1.0), 33)
        assert torch.equal(x.grad, got[0]) and torch.equal(w.grad, got[4])
        # the norm after a block is the same definition; not bit for bit, since a product that goes straight into a 16-bit result
        # may be rounded once (a mixed multiply-add) where one that passes the scale first is rounded to fp32 before
        _within(norm.join(x, post=w, eps=1e-5), *want, "post")


def test_gradients_against_differences(cuda):
    """Directional differences of the float64 forward against the kernels' gradients; the quotient's own error is of the order of
    step^2 = 1e-10 times third derivatives of some tens."""
    from mi355moe import norm
    R, H = 7, 40
    kw = dict(eps=1e-5, scale=0.8, residual_scale=1.1)
    for gate in ("channel", "token", "full"):
        t, ds, dy = _inputs(R, H, gate, torch.float32, torch.float32, torch.float32, 5)
        args = [t[k] for k in NAMES]
        _, _, stats = norm.join_forward(*args, **kw)
        got = norm.join_backward(ds, dy, stats, *args, 0.8, 1.1)

        def loss(f):
            (s, _), (y, _) = ref.norm(*f, 1e-5, 0.8, 1.1, 0.0, 0.0)
            return float((s * _f64(ds)).sum() + (y * _f64(dy)).sum())

        rng = np.random.default_rng(1)
        base = [_f64(v) for v in args]
        for i in range(5):
            v = rng.standard_normal(base[i].shape)
            ends = [loss([b + (k * 1e-5 * v if j == i else 0.0) for j, b in enumerate(base)]) for k in (1, -1)]
            slope = (ends[0] - ends[1]) / 2e-5
            mine = _f64(got[i]).reshape(base[i].shape)
            assert abs(slope - float((mine * v).sum())) <= 2.0 ** -14 * float(np.abs(mine * v).sum()) + 1e-4, (gate, i)


def test_views_and_strides(cuda):
    from mi355moe import norm
    for R, H, dt in ((6, 72, torch.bfloat16), (5, 1029, torch.float16), (9, 2056, torch.float32)):
        t, ds, dy = _inputs(R, H, "full", dt, dt, dt, 2)
        args = [t[k] for k in NAMES]
        s, y, stats = norm.join_forward(*args)
        grads = norm.join_backward(ds, dy, stats, *args)
        for off in (0, 1, 3, 8):
            def wide(v):
                w = torch.zeros(R, H + 17, dtype=v.dtype, device="cuda")
                w[:, off:off + H] = v
                return w[:, off:off + H]

            views = [wide(args[0]), wide(args[1]), args[2], wide(args[3]), args[4]]
            vs, vy, vst = norm.join_forward(*views)
            assert torch.equal(vs, s) and torch.equal(vy, y) and torch.equal(vst, stats)
            assert all(torch.equal(p, q) for p, q in zip(norm.join_backward(wide(ds), wide(dy), stats, *views), grads))
        cols = [v.t().contiguous().t() if v.dim() == 2 else torch.stack([v, v], 1)[:, 0] for v in args]
        assert torch.equal(norm.join_forward(*cols)[1], y)
        deep = [v.reshape(1, R, 1, H) if v.dim() == 2 else v for v in args]
        assert torch.equal(norm.join_forward(*deep)[1], y.reshape(1, R, 1, H))
        one = [v[0] if v.dim() == 2 else v for v in args]
        assert torch.equal(norm.join_forward(*one)[1], y[0])
        leaf = args[0].clone().requires_grad_()
        norm.join(leaf, *args[1:2], post=args[2], gate=args[3], pre=args[4])[1].sum().backward()      # an expanded gradient, strides 0
        want = norm.join_backward(None, torch.ones_like(dy), stats, *args)[0]
        assert torch.equal(leaf.grad, want)


def test_rows_stay_apart(cuda):
    """NaN, infinities and zeros in some rows leave the others as they were; a row of zeros is zero, with eps 0 NaN as the formula
    has it."""
    from mi355moe import norm
    for R, H in ((9, 72), (6, 2056)):
        t, ds, dy = _inputs(R, H, "token", torch.bfloat16, torch.float32, torch.bfloat16, 4)
        args = [t[k] for k in NAMES]
        s, y, stats = norm.join_forward(*args)
        clean = norm.join_backward(ds, dy, stats, *args)
        args[0][1, 5], args[1][3, 0], args[0][4] = float("nan"), float("inf"), 0.0
        s2, y2, st2 = norm.join_forward(*args)
        keep = [r for r in range(R) if r not in (1, 3, 4)]
        assert torch.equal(s2[keep], s[keep]) and torch.equal(y2[keep], y[keep])
        assert torch.isnan(y2[1]).all() and torch.isfinite(y2[4]).all()
        got = norm.join_backward(ds, dy, st2, *args)
        for i in (0, 1, 3):
            assert torch.equal(got[i][keep], clean[i][keep])
        zero = torch.zeros(R, H, device="cuda")
        assert (norm.rms(zero, args[4]) == 0).all() and torch.isnan(norm.rms(zero, args[4], eps=0.0)).all()


def test_no_rows(cuda):
    from mi355moe import norm
    b = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    for gate in (None, torch.ones(16, device="cuda"), torch.ones(0, 1, device="cuda"), torch.ones(0, 16, device="cuda")):
        s, y = norm.join(b, b.detach(), post=w, gate=gate, pre=w)
        assert s.shape == y.shape == (0, 16)
    (s.sum() + y.sum()).backward()
    assert b.grad.shape == (0, 16) and (w.grad == 0).all()


def test_captured_step(cuda):
    """The explicit pair captured and replayed with new inputs, eager work between the replays; the differentiable form is refused
    during capture when it would record a gradient, and the capture survives the refusal."""
    from mi355moe import norm
    for R, H in ((1, 264), (300, 2056)):
        t, ds, dy = _inputs(R, H, "channel", torch.bfloat16, torch.float32, torch.bfloat16, 1)
        args = [t[k] for k in NAMES]
        leaf = args[0].clone().requires_grad_()
        alive = norm.rms(leaf, args[4].clone())

        def step():
            s, y, stats = norm.join_forward(*args)
            return (s, y, *norm.join_backward(ds, dy, stats, *args))

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="capture"):
                norm.rms(leaf, args[4])
            outs = step()
        for seed in range(4):
            t2, ds2, dy2 = _inputs(R, H, "channel", torch.bfloat16, torch.float32, torch.bfloat16, 20 + seed)
            for a, k in zip(args, NAMES):
                a.copy_(t2[k])
            ds.copy_(ds2), dy.copy_(dy2)
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))
        alive.sum().backward()
        assert torch.isfinite(leaf.grad).all()


def test_two_streams(cuda):
    from mi355moe import norm
    sets = [_inputs(R, H, "channel", torch.bfloat16, torch.float32, torch.bfloat16, R) for R, H in ((400, 1032), (30, 4096))]

    def work(i):
        t, ds, dy = sets[i]
        args = [t[k] for k in NAMES]
        s, y, stats = norm.join_forward(*args)
        return (s, y, *norm.join_backward(ds, dy, stats, *args))

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
    """More than 2^31 values: the last rows against float64."""
    from mi355moe import norm
    R, H, dt = (1 << 17) + 3, 16384, torch.bfloat16
    b = torch.randn(64, H, device="cuda").to(dt).repeat(R // 64 + 1, 1)[:R]
    b[-5:] = torch.randn(5, H, device="cuda").to(dt)
    w = torch.randn(H, device="cuda")
    s, y, stats = norm.join_forward(b, b, w, None, w, 1e-5, 0.5, 2.0)
    tail = _f64(b[-5:])
    (ws, es), (wy, ey) = ref.norm(tail, tail, _f64(w), None, _f64(w), 1e-5, 0.5, 2.0, ref.HALF["bfloat16"], ref.TINY["bfloat16"])
    _within(s[-5:], ws, es, "s")
    _within(y[-5:], wy, ey, "y")
    del s
    db, dr, *_ = norm.join_backward(None, y, stats, b, b, w, None, w, 0.5, 2.0, need=(True, True, False, False, False))
    want = ref.norm_grads(None, _f64(y[-5:]), tail, tail, _f64(w), None, _f64(w), 1e-5, 0.5, 2.0)
    for got, k in ((db, "branch"), (dr, "residual")):
        value, mag = want[k]
        _within(got[-5:], value, 512 * ref.U * mag + ref.HALF["bfloat16"] * np.abs(value) + ref.TINY["bfloat16"], k)
