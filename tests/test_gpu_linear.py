"""GPU parity of the dense product with its epilogue (mi355moe.ffn.linear) and its gradients with their definitions in float64
(oracle/block.py), within bounds computed from the roundings of the sums, the epilogue and the results."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _name(dt):
    return str(dt).replace("torch.", "")


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _within(got, want, tol, what):
    bad = ~(np.abs(_f64(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], int(bad.sum()))


def _inputs(M, K, N, dt, seed, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (new(M, K).to(dt), (new(N, K) * (scale / K ** 0.5)).to(dt), new(N) * 0.5, new(M, N).to(dt), new(M, N).to(dt))


def _hold(M, K, N, dt, act, bias, residual, seed):
    from mi355moe import ffn
    x, w, b, r, dy = _inputs(M, K, N, dt, seed)
    b = None if bias is None else b.to(bias)
    r = r if residual else None
    h, t = ref.HALF[_name(dt)], ref.TINY[_name(dt)]
    out, z = ffn.linear_forward(x, w, b, act, r, save=True)
    want, tol, wz, ez = ref.linear(_f64(x), _f64(w), _f64(b), act, _f64(r), h, t)
    _within(out, want, tol, "out")
    assert (z is None) == (act is None)
    if z is not None:
        _within(z, wz, ez, "z")
    assert torch.equal(ffn.linear(x, w, b, act, r), out)
    dx, dw, db = ffn.linear_backward(dy, z, x, w, act, bias)
    gx, gw, gb = ref.linear_grads(_f64(dy), _f64(z), _f64(x), _f64(w), act, h, t, dt == torch.float16)
    _within(dx, *gx, "dx")
    _within(dw, *gw, "dw")
    if bias is not None:
        hb = ref.HALF[_name(bias)]
        _within(db, gb[0], gb[1] * (1 + hb) + hb * np.abs(gb[0]) + ref.TINY[_name(bias)], "db")
    leaf = [None if v is None else v.clone().requires_grad_() for v in (x, w, b, r)]
    y = ffn.linear(leaf[0], leaf[1], bias=leaf[2], activation=act, residual=leaf[3])
    assert torch.equal(y, out)
    y.backward(dy)
    for v, g in zip(leaf, (dx, dw, db, dy)):
        assert v is None or torch.equal(v.grad, g)


# M, K, N: streamed, every kind of tile, contractions that are cut, sizes that are no multiple of anything
SIZES = [(1, 1, 1), (1, 1024, 4096), (1, 4099, 33), (3, 7, 5), (16, 512, 40), (17, 264, 16), (33, 65, 1030), (64, 128, 100), (129, 72, 300),
         (300, 640, 8), (257, 40, 515), (70, 2056, 4100), (1000, 200, 1032), (333, 131, 2051), (1300, 1096, 1032), (2100, 72, 2056),
         (6000, 24, 1100), (200, 8200, 520), (1541, 33, 72), (97, 4168, 2064)]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_forward_and_gradients(cuda, M, K, N, dt):
    i = SIZES.index((M, K, N)) + (dt == torch.float16) * 2
    _hold(M, K, N, dt, ACTS[i % 5], [None, torch.float32, dt, torch.float16][i % 4], i % 3 != 0, M + K)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
def test_every_epilogue(cuda, act, bias, residual):
    for M, K, N in ((5, 72, 40), (150, 130, 777), (1100, 72, 1048), (130, 4104, 1032)):
        _hold(M, K, N, torch.bfloat16, act, bias, residual, M)


def test_large_tiles(cuda):
    """Sizes that take the largest tiles in the forward and in both gradients, ragged in every dimension: a sample of rows and
    columns in float64 on the GPU."""
    from mi355moe import ffn
    M, K, N, dt, act = 3339, 2056, 4104, torch.bfloat16, "gelu_tanh"
    x, w, b, r, dy = _inputs(M, K, N, dt, 5)
    out, z = ffn.linear_forward(x, w, b, act, r, save=True)
    dx, dw, db = ffn.linear_backward(dy, z, x, w, act, torch.float32)
    h, t = ref.HALF["bfloat16"], ref.TINY["bfloat16"]
    rows = torch.randint(0, M, (30,), generator=torch.Generator().manual_seed(1)).tolist() + [0, M - 1]
    want, tol, wz, ez = ref.linear(_f64(x[rows]), _f64(w), _f64(b), act, _f64(r[rows]), h, t)
    _within(out[rows], want, tol, "out")
    _within(z[rows], wz, ez, "z")
    cols = torch.randint(0, K, (20,), generator=torch.Generator().manual_seed(2)).tolist() + [0, K - 1]
    Z, Wc, X = _f64(z), _f64(w[:, cols]), _f64(x[:, cols])
    gx, gw, gb = ref.linear_grads(_f64(dy), Z, X, Wc, act, h, t, False)
    _within(dx[:, cols], *gx, "dx")
    _within(dw[:, cols], *gw, "dw")
    _within(db, gb[0], gb[1], "db")


def test_gradients_against_differences(cuda):
    """Directional differences of the float64 forward against the kernels' gradients, within the gradients' own bounds; the
    quotient's error is of the order of step^2 = 1e-10 times third derivatives of some tens."""
    from mi355moe import ffn
    M, K, N, dt = 24, 96, 40, torch.float16
    h, t = ref.HALF["float16"], ref.TINY["float16"]
    for act in ("silu", "gelu", "gelu_tanh"):
        x, w, b, _, dy = _inputs(M, K, N, dt, 3)
        _, z = ffn.linear_forward(x, w, b, act, save=True)
        got = ffn.linear_backward(dy, z, x, w, act, torch.float32)
        bounds = ref.linear_grads(_f64(dy), _f64(z), _f64(x), _f64(w), act, h, t, True)
        base = [_f64(v) for v in (x, w, b)]
        rng = np.random.default_rng(4)

        def loss(f):
            return float((ref.linear(*f, act, None, 0.0, 0.0)[0] * _f64(dy)).sum())

        for i in range(3):
            v = rng.standard_normal(base[i].shape)
            ends = [loss([p + (k * 1e-5 * v if j == i else 0.0) for j, p in enumerate(base)]) for k in (1, -1)]
            slope = (ends[0] - ends[1]) / 2e-5
            # (the oracle's gradients go by the kernel's fp32 z, the differences by the exact one: 1e-5 of the slope)
            assert abs(slope - float((_f64(got[i]) * v).sum())) <= float((bounds[i][1] * np.abs(v)).sum()) + 1e-4 * abs(slope) + 1e-4


def test_fp16_gradients_keep_their_range(cuda):
    """dz of a call with small gradients lies among fp16's subnormals, of one with large ones beyond its range; the sums do not."""
    from mi355moe import ffn
    M, K, N, dt = 70, 136, 264, torch.float16
    for act in ("silu", "gelu", "gelu_tanh", "relu"):
        for f in (2.0 ** -22, 60000.0):
            x, w, b, _, dy = _inputs(M, K, N, dt, 6)
            x, w = x * 0.01, (w.float() * (0.1 if f > 1 else 1.0)).half()
            dy = (torch.sign(dy).float() * f).to(dt)
            _, z = ffn.linear_forward(x, w, b, act, save=True)
            dx, dw, _ = ffn.linear_backward(dy, z, x, w, act)
            gx, gw, _ = ref.linear_grads(_f64(dy), _f64(z), _f64(x), _f64(w), act, ref.HALF["float16"], ref.TINY["float16"], True)
            for got, (v, tol) in ((dx, gx), (dw, gw)):
                fits = np.abs(v) < 65000.0
                assert fits.any() and (np.abs(_f64(got) - v) <= tol)[fits].all(), (act, f)


def test_zero_and_non_finite_rows(cuda):
    from mi355moe import ffn
    for M in (6, 200, 2100):
        x, w, b, r, dy = _inputs(M, 200, 264, torch.bfloat16, 2)
        clean = ffn.linear(x, w, b, "silu", r)
        x[2, 5], r[4, 3], x[5] = float("nan"), float("inf"), 0.0
        for act in ACTS:
            out, z = ffn.linear_forward(x, w, b, act, r, save=True)
            assert torch.isnan(out[2]).all() and torch.isinf(out[4, 3]) and torch.isfinite(out[5]).all()
            if act == "silu":
                keep = [m for m in range(M) if m not in (2, 4, 5)]
                assert torch.equal(out[keep], clean[keep])
            dx, _, _ = ffn.linear_backward(dy, z, x, w, act)
            assert torch.isfinite(dx[[m for m in range(M) if m != 2]]).all()
            assert act is None or torch.isnan(dx[2]).all()
        big = torch.full((1, 8), 300.0, device="cuda").bfloat16()
        for act in ACTS[1:]:                                     # z of +-240000, 234.4 steps of 1024: the activations' ends
            y = ffn.linear(big, torch.stack([torch.full((8,), v) for v in (100.0, -100.0)]).bfloat16().cuda(), activation=act)
            assert y[0, 0] == 234 * 1024.0 and y[0, 1] == 0.0


def test_views_and_strides(cuda):
    from mi355moe import ffn
    for M, K, N in ((5, 72, 24), (200, 72, 520), (300, 75, 130)):
        x, w, b, r, dy = _inputs(M, K, N, torch.bfloat16, 9)
        want, z = ffn.linear_forward(x, w, b, "silu", r, save=True)
        grads = ffn.linear_backward(dy, z, x, w, "silu", torch.float32)
        for off in (0, 3, 8):
            def wide(v):
                t = torch.zeros(v.shape[0], v.shape[1] + 18, dtype=v.dtype, device="cuda")
                t[:, off:off + v.shape[1]] = v
                return t[:, off:off + v.shape[1]]

            assert torch.equal(ffn.linear(wide(x), wide(w), b, "silu", wide(r)), want)
            got = ffn.linear_backward(wide(dy), z, wide(x), wide(w), "silu", torch.float32)
            assert all(torch.equal(p, q) for p, q in zip(got, grads))
        t = lambda v: v.t().contiguous().t()  # noqa: E731
        assert torch.equal(ffn.linear(t(x), t(w), torch.stack([b, b], 1)[:, 0], "silu", t(r)), want)
        assert torch.equal(ffn.linear(x.reshape(1, M, K), w, b, "silu", r.reshape(1, M, N))[0], want)
        assert torch.equal(ffn.linear(x[0], w, b, "silu", r[0]), ffn.linear(x[:1], w, b, "silu", r[:1])[0])
        rows = x[:1].expand(M, K)
        assert torch.equal(ffn.linear(rows, w), ffn.linear(rows.contiguous(), w))
        leaf, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        for act in (None, "relu"):
            leaf.grad = wl.grad = None
            ffn.linear(leaf, wl, b, act).sum().backward()        # an expanded gradient, strides 0
            zz = ffn.linear_forward(x, w, b, act, save=True)[1]
            dx, dw, _ = ffn.linear_backward(torch.ones_like(dy), zz, x, w, act)
            assert torch.equal(leaf.grad, dx) and torch.equal(wl.grad, dw)
        for need in ((True, False), (False, True), (False, False)):
            one = ffn.linear_backward(dy, z, x, w, "silu", torch.float32, *need)
            assert all((p is None) == (not n) and (p is None or torch.equal(p, q)) for p, q, n in zip(one, grads, (*need, True)))


def test_no_rows(cuda):
    from mi355moe import ffn
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    w = torch.randn(32, 64, device="cuda").half().requires_grad_()
    b = torch.randn(32, device="cuda", requires_grad=True)
    y = ffn.linear(x, w, b, "gelu")
    assert y.shape == (0, 32)
    y.backward(torch.empty_like(y))
    assert x.grad.shape == (0, 64) and (w.grad == 0).all() and (b.grad == 0).all()


def test_captured_step(cuda):
    """The explicit pair captured and replayed with new inputs, eager work between the replays; the differentiable form is refused
    during capture when it would record a gradient, and the capture survives the refusal."""
    from mi355moe import ffn
    for M, K, N, dt in ((8, 256, 64, torch.bfloat16), (260, 2056, 130, torch.float16), (1600, 75, 264, torch.float16)):
        x, w, b, r, dy = _inputs(M, K, N, dt, 1)
        leaf = x.clone().requires_grad_()
        alive = ffn.linear(leaf, w.clone(), b, "silu", r)

        def step():
            y, z = ffn.linear_forward(x, w, b, "silu", r, save=True)
            return (y, *ffn.linear_backward(dy, z, x, w, "silu", torch.float32))

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="capture"):
                ffn.linear(leaf, w)
            outs = step()
        for seed in range(4):
            for t, new in zip((x, w, b, r, dy), _inputs(M, K, N, dt, 20 + seed)):
                t.copy_(new)
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))
        alive.sum().backward()
        assert torch.isfinite(leaf.grad).all()


def test_two_streams(cuda):
    from mi355moe import ffn
    sets = [_inputs(M, 1032, 130, torch.float16, M) for M in (50, 300)]

    def work(i):
        x, w, b, r, dy = sets[i]
        y, z = ffn.linear_forward(x, w, b, "gelu", r, save=True)
        return (y, *ffn.linear_backward(dy, z, x, w, "gelu", torch.float32))

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
    """More than 2^31 values of the output and of z: the last rows, and their gradients, against float64."""
    from mi355moe import ffn
    M, K, N, dt = 1 << 20, 16, 2056, torch.bfloat16
    x, w, b, _, _ = _inputs(M, K, N, dt, 4)
    out, z = ffn.linear_forward(x, w, b, "silu", save=True)
    h, t = ref.HALF["bfloat16"], ref.TINY["bfloat16"]
    for lo in (0, M // 2, M - 200):
        s = slice(lo, lo + 200)
        want, tol, wz, ez = ref.linear(_f64(x[s]), _f64(w), _f64(b), "silu", None, h, t)
        _within(out[s], want, tol, "out")
        _within(z[s], wz, ez, "z")
    dx, _, db = ffn.linear_backward(out, z, x, w, "silu", torch.float32, True, False)
    s = slice(M - 200, M)
    gx, _, _ = ref.linear_grads(_f64(out[s]), _f64(z[s]), _f64(x[s]), _f64(w), "silu", h, t, False)
    _within(dx[s], *gx, "dx")
    d = out[:, :3].double() * torch.sigmoid(z[:, :3].double()) * (1 + z[:, :3].double() * torch.sigmoid(-z[:, :3].double()))
    assert ((db[:3].double() - d.sum(0)).abs() <= (M / 64 / 16 + 64) * ref.U * d.abs().sum(0) + 2.0 ** -20 * out[:, :3].double().abs().sum(0) * 8).all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_slopes_far_out(cuda, act):
    """Where |z| is far beyond the activation's bend the slope is 1 or 0, also where z^2 passes fp32's range; a NaN stays one."""
    from mi355moe import ffn
    far = torch.tensor([100.0, 1e4, 1e15, 1e20, 3e38], device="cuda")
    z = torch.cat([far, -far]).repeat(8, 1).contiguous()
    g = torch.Generator(device="cuda").manual_seed(1)
    dy = torch.randn(8, 10, generator=g, device="cuda").to(torch.bfloat16)
    x, w = torch.ones(8, 16, device="cuda", dtype=torch.bfloat16), torch.ones(10, 16, device="cuda", dtype=torch.bfloat16)
    _, dw, db = ffn.linear_backward(dy, z, x, w, act, torch.float32)
    want = dy.double().sum(0)
    want[5:] = 0
    mag = dy.double().abs().sum(0)
    assert bool(((db.double() - want).abs() <= 2.0 ** -20 * mag).all()), (db, want)      # (eight values and their sum)
    assert bool(((dw[:, 0].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * mag).all())
    z[3, 2] = float("nan")
    db = ffn.linear_backward(dy, z, x, w, act, torch.float32, need_dx=False, need_dw=False)[2]
    assert bool(db[2].isnan()) and not bool(db[[0, 1, 3, 4, 5, 6, 7, 8, 9]].isnan().any())


def test_long_contraction_beyond_32_bit_offsets(cuda):
    """dW over rows whose bytes pass 32 bits, dx that has as many, and x read there by the forward pass."""
    from mi355moe import ffn
    M, K, N, dt = (1 << 21) + 3, 1032, 24, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(M, K, generator=g, device="cuda", dtype=dt)
    dy = torch.randn(M, N, generator=g, device="cuda", dtype=dt)
    w = torch.randn(N, K, generator=g, device="cuda", dtype=dt)
    dx, dw, db = ffn.linear_backward(dy, None, x, w, None, torch.float32)
    some = [0, 7, 511, 1031]
    d, xs = dy.double(), x[:, some].double()
    want, mag = (d.t().contiguous() @ xs), (d.abs().t().contiguous() @ xs.abs())
    h = ref.HALF["bfloat16"]
    assert bool(((dw[:, some].double() - want).abs() <= (M / 8 + 24) * 2 * ref.U * mag * (1 + h) + h * want.abs()).all())
    assert bool(((db.double() - d.sum(0)).abs() <= (M / 8 + 32) * ref.U * d.abs().sum(0)).all())
    out = ffn.linear_forward(x, w)
    for s in (slice(0, 100), slice(M - 100, M)):
        want, tol, _, _ = ref.linear(_f64(x[s]), _f64(w), None, None, None, h, ref.TINY["bfloat16"])
        _within(out[s], want, tol, "out")
        gx, _, _ = ref.linear_grads(_f64(dy[s]), None, _f64(x[s]), _f64(w), None, h, ref.TINY["bfloat16"], False)
        _within(dx[s], *gx, "dx")
