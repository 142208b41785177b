"""GPU parity of the gated feed-forward block (mi355moe.ffn) and its gradient with their definitions in float64
(oracle/mxfp4.py: gated, gated_grads). Bounds are computed per element from the roundings that the formulas' fp32
evaluation and the single roundings to 16 bits take; none is fitted. The shared expert and the routed MXFP4 experts are
also run together, as a layer has them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def _f64(t):
    return t.detach().double().cpu().numpy()


def _inputs(T, H, I, dt, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").to(dt)
    w = (torch.randn(2 * I, H, generator=g, device="cuda") * (scale / H ** 0.5)).to(dt)
    dh = torch.randn(T, I, generator=g, device="cuda").to(dt)
    return x, w, dh


def _within(got, want, tol, what):
    bad = ~(np.abs(_f64(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], int(bad.sum()))


SIZES = [(1, 8, 8, 0.0), (1, 4096, 64, 10.0), (2, 136, 24, 1.0), (16, 512, 40, 2.0), (17, 264, 8, 10.0), (33, 64, 72, 1.0),
         (40, 1000, 200, 3.0), (129, 328, 136, 0.0), (257, 72, 264, 2.0), (300, 640, 8, 10.0), (64, 8, 128, 1.0),
         (1000, 200, 1032, 2.0), (1300, 1096, 1032, 10.0), (2100, 72, 520, 0.0), (6000, 120, 24, 1.0), (800, 136, 200, 1.0),
         (200, 2056, 520, 10.0), (97, 4168, 1032, 1.0), (400, 8200, 136, 2.0), (130, 2048, 776, 0.0),
         (1541, 264, 72, 0.0)]                                             # streamed, every kind of tile, cut contractions


@pytest.mark.parametrize("T,H,I,limit", SIZES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_forward_and_gradients(cuda, T, H, I, limit, dt):
    from mi355moe import ffn
    x, w, dh = _inputs(T, H, I, dt, T + H)
    X, W = _f64(x), _f64(w)
    h, gu = ffn.gated_forward(x, w, limit, save=True)
    want, tol, z, ez = ref.gated(X, W, limit, EPS[dt])
    _within(gu, z, ez, "gu")
    _within(h, want, tol + TINY[dt], "h")
    assert torch.equal(ffn.gated(x, w, limit), h)
    dx, dw = ffn.gated_backward(dh, gu, x, w, limit)
    (rx, tx), (rw, tw) = ref.gated_grads(_f64(dh), _f64(gu), X, W, limit, EPS[dt], TINY[dt])
    _within(dx, rx, tx, "dx")
    _within(dw, rw, tw, "dw")
    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = ffn.gated(xr, wr, limit)
    assert torch.equal(out, h)
    out.backward(dh)
    assert torch.equal(xr.grad, dx) and torch.equal(wr.grad, dw)


def test_large_tiles(cuda):
    """Sizes that take the largest tiles in the forward and in both gradients, ragged in every dimension."""
    from mi355moe import ffn
    T, H, I, limit, dt = 3339, 4104, 2056, 10.0, torch.bfloat16
    x, w, dh = _inputs(T, H, I, dt, 5)
    h, gu = ffn.gated_forward(x, w, limit, save=True)
    dx, dw = ffn.gated_backward(dh, gu, x, w, limit)
    dev = torch.device("cuda")
    # float64 on the GPU, the bounds for a sample of rows and columns
    X, W = x.double(), w.double()
    z = X @ W.t().contiguous()
    rows = torch.randint(0, T, (40,), generator=torch.Generator().manual_seed(1)).tolist() + [0, T - 1]
    want, tol, _, ez = ref.gated(_f64(x[rows]), _f64(w), limit, EPS[dt])
    _within(h[rows], want, tol + TINY[dt], "h")
    _within(gu[rows], _f64(z[rows]), ez, "gu")
    Z = gu.double()
    g, u = Z[:, :I], Z[:, I:]
    gc, uc = g.clamp(max=limit), u.clamp(-limit, limit)
    s = torch.sigmoid(gc)
    D = torch.cat([dh.double() * uc * s * (1 + gc * (1 - s)) * (g <= limit), dh.double() * gc * s * (u.abs() <= limit)], 1)
    # d carries one rounding of half a step and fp32 evaluation; the same bound on every element of D
    eD = D.abs() * (EPS[dt] / 2 + 2.0 ** -18) + 2.0 ** -18 * dh.double().abs().repeat(1, 2) * limit
    cols = torch.randint(0, H, (64,), generator=torch.Generator().manual_seed(2)).tolist() + [0, H - 1]
    for got, A, eA, B, K, pick in ((dx, D, eD, W, 2 * I, lambda t: t[:, cols]), (dw, D.t().contiguous(), eD.t().contiguous(), X, T, lambda t: t[:, cols])):
        v = A @ B[:, cols]
        t = eA @ B[:, cols].abs() + (A.abs() @ B[:, cols].abs()) * (K / 8 + 24) * 2.0 ** -23
        t = t * (1 + EPS[dt]) + v.abs() * EPS[dt] / 2
        assert ((pick(got).double() - v).abs() <= t).all()
    assert dev.type == dx.device.type


def test_gradients_against_differences(cuda):
    """Directional differences of the float64 forward against the kernels' gradients: the difference quotient's own error
    is O(step^2), and the gradients' bound comes from gated_grads."""
    from mi355moe import ffn
    T, H, I, limit, dt = 24, 96, 40, 6.0, torch.float16
    x, w, dh = _inputs(T, H, I, dt, 3, scale=2.0)
    h, gu = ffn.gated_forward(x, w, limit, save=True)
    dx, dw = ffn.gated_backward(dh, gu, x, w, limit)
    X, W, DH = _f64(x), _f64(w), _f64(dh)
    (_, tx), (_, tw) = ref.gated_grads(DH, _f64(gu), X, W, limit, EPS[dt], TINY[dt])
    rng = np.random.default_rng(4)

    def loss(a, b):
        return float((ref.gated(a, b, limit, 0.0)[0] * DH).sum())

    step = 1e-5
    for _ in range(4):
        vx, vw = rng.standard_normal(X.shape), rng.standard_normal(W.shape)
        nx = (loss(X + step * vx, W) - loss(X - step * vx, W)) / (2 * step)
        nw = (loss(X, W + step * vw) - loss(X, W - step * vw)) / (2 * step)
        # third derivatives of the block are below 50 here: |quotient - derivative| <= step^2 * 50 * |v|^3-ish; 1e-6 of the scale
        assert abs(nx - float((_f64(dx) * vx).sum())) <= float((tx * np.abs(vx)).sum()) + 1e-5 * abs(nx) + 1e-4
        assert abs(nw - float((_f64(dw) * vw).sum())) <= float((tw * np.abs(vw)).sum()) + 1e-5 * abs(nw) + 1e-4


def test_limit_borders(cuda):
    """g and u exactly at the limit pass gradients, beyond it none: one-hot rows make z exact."""
    from mi355moe import ffn
    H, I, L = 8, 8, 2.0
    w = torch.zeros(2 * I, H)
    for i in range(8):
        w[i, 0], w[I + i, 1] = [2.0, 2.0, 3.0, -3.0, 1.0, 2.0, -40.0, 0.0][i], [2.0, -2.0, 1.0, 2.5, -2.5, 3.0, 1.0, 0.5][i]
    x = torch.zeros(1, H)
    x[0, :2] = 1.0
    x, w = x.bfloat16().cuda(), w.bfloat16().cuda()
    dh = torch.ones(1, I, dtype=torch.bfloat16, device="cuda")
    h, gu = ffn.gated_forward(x, w, L, save=True)
    _, dw = ffn.gated_backward(dh, gu, x, w, L)
    (_, _), (rw, tw) = ref.gated_grads(_f64(dh), _f64(gu), _f64(x), _f64(w), L, EPS[torch.bfloat16], TINY[torch.bfloat16])
    _within(dw, rw, tw, "dw")
    g, u = _f64(gu)[0, :I], _f64(gu)[0, I:]
    got = _f64(dw)
    assert ((got[:I, 0] == 0) == ((g > L) | (u == 0))).all()
    assert ((got[I:, 1] == 0) == ((np.abs(u) > L) | (g == 0))).all()


def test_views_strides_and_broadcast_gradients(cuda):
    from mi355moe import ffn
    for T in (5, 70):
        x, w, dh = _inputs(T, 72, 24, torch.bfloat16, 9)
        want = ffn.gated(x, w, 1.0)
        wide = torch.zeros(T, 90, dtype=x.dtype, device="cuda")
        for off in (0, 3, 8):
            wide[:, off:off + 72] = x
            assert torch.equal(ffn.gated(wide[:, off:off + 72], w, 1.0), want)
        assert torch.equal(ffn.gated(x.t().contiguous().t(), w, 1.0), want)
        assert torch.equal(ffn.gated(x, w.t().contiguous().t(), 1.0), want)
        assert torch.equal(ffn.gated(x.reshape(1, T, 72), w, 1.0)[0], want)
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        ffn.gated(xr, wr, 1.0).sum().backward()              # an expanded gradient, strides 0
        _, gu = ffn.gated_forward(x, w, 1.0, save=True)
        dx, dw = ffn.gated_backward(torch.ones_like(dh), gu, x, w, 1.0)
        assert torch.equal(xr.grad, dx) and torch.equal(wr.grad, dw)
        only = x.clone().requires_grad_()
        ffn.gated(only, w, 1.0).backward(dh)
        assert torch.equal(only.grad, ffn.gated_backward(dh, gu, x, w, 1.0, need_dw13=False)[0])


def test_empty_rows(cuda):
    from mi355moe import ffn
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    w = torch.randn(32, 64, device="cuda").half().requires_grad_()
    h = ffn.gated(x, w, 1.0)
    assert h.shape == (0, 16)
    h.backward(torch.empty_like(h))
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()


def test_non_finite_rows_stay_apart(cuda):
    from mi355moe import ffn
    for T in (6, 200, 2100):
        x, w, dh = _inputs(T, 200, 48, torch.bfloat16, 2)
        clean = ffn.gated(x, w, 10.0)
        x[2, 5], x[4, 199] = float("nan"), float("inf")
        h, gu = ffn.gated_forward(x, w, 10.0, save=True)
        keep = [t for t in range(T) if t not in (2, 4)]
        assert torch.isnan(h[2]).all() and torch.equal(h[keep], clean[keep])
        # -inf gates give 0 * inf or NaN as the formula has it; +inf gates are limited
        z = gu[4]
        assert torch.isinf(z[:48]).any() or torch.isnan(z[:48]).any()
        dx, _ = ffn.gated_backward(dh, gu, x, w, 10.0)
        assert torch.isfinite(dx[keep]).all()


def test_captured_forward_and_backward(cuda):
    """The explicit pair captured and replayed with new inputs, eager work between the replays; the differentiable form is
    refused during capture when it would record a gradient, and the capture survives the refusal."""
    from mi355moe import ffn
    for T in (8, 260, 1600):
        x, w, dh = _inputs(T, 256, 64, torch.bfloat16, 1)
        eager_leaf = x.clone().requires_grad_()
        alive = ffn.gated(eager_leaf, w.clone(), 10.0)       # an eager graph that lives on (w itself is refilled below)

        def step():
            h, gu = ffn.gated_forward(x, w, 10.0, save=True)
            return (h, *ffn.gated_backward(dh, gu, x, w, 10.0))

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with pytest.raises(RuntimeError, match="capture"):
                ffn.gated(eager_leaf, w, 10.0)
            outs = step()
        for seed in range(4):
            x2, w2, dh2 = _inputs(T, 256, 64, torch.bfloat16, 20 + seed)
            x.copy_(x2), w.copy_(w2), dh.copy_(dh2)
            g.replay()
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))
        alive.sum().backward()
        assert torch.isfinite(eager_leaf.grad).all()


def test_two_streams(cuda):
    from mi355moe import ffn
    sets = [_inputs(T, 512, 128, torch.bfloat16, T) for T in (50, 300)]

    def work(i):
        x, w, dh = sets[i]
        h, gu = ffn.gated_forward(x, w, 10.0, save=True)
        return (h, *ffn.gated_backward(dh, gu, x, w, 10.0))

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


@pytest.mark.parametrize("T", [3, 150])
def test_layer_with_shared_expert(cuda, T):
    """A layer's feed-forward part as a model runs it: the shared expert (gated block, then its down projection) into
    out, the routed MXFP4 experts folded into it; against float64 within the bounds of the parts."""
    from mi355moe import ffn, mxfp4, ops, synthetic
    n, H, I, topk, dt = 16, 512, 128, 4, torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    ex = mxfp4.Mxfp4Experts.from_dense(torch.randn(n, 2 * I, H, generator=g, device="cuda") * 0.1,
                                       torch.randn(n, H, I, generator=g, device="cuda") * 0.1)
    x, w13, _ = _inputs(T, H, I, dt, 7)
    w2 = (torch.randn(H, I, generator=g, device="cuda") * 0.1).to(dt)
    rw, rb = synthetic.router(n, H, seed=5, device="cuda")
    ids, wts = ops.router_topk(ops.router_logits(x, rw), topk, rb, routed_scale=2.5)
    h = ffn.gated(x, w13, 10.0)
    out = torch.nn.functional.linear(h, w2)
    shared = out.clone()
    mxfp4.moe_forward_ids(ex, x, ids, wts, limit=10.0, out=out, accumulate=True)
    want_h, tol_h, _, _ = ref.gated(_f64(x), _f64(w13), 10.0, EPS[dt])
    _within(h, want_h, tol_h + TINY[dt], "h")
    d13 = ref.values(ex.w13.cpu().numpy(), ex.w13_scale.cpu().numpy(), H)
    d2 = ref.values(ex.w2.cpu().numpy(), ex.w2_scale.cpu().numpy(), I)
    routed, tol = ref.moe(_f64(x), d13, d2, ids.cpu().numpy(), _f64(wts), 10.0, 0.0)
    total = _f64(shared) + routed
    _within(out, total, tol + np.abs(total) * EPS[dt] / 2 + np.abs(_f64(shared)) * 2.0 ** -22, "layer")


def test_rows_beyond_32_bit_offsets(cuda):
    """More than 2^31 values of h and of [g | u]: the last rows, and their gradients, against float64."""
    from mi355moe import ffn
    T, H, I = 1 << 20, 32, 2064
    x, w, dh = _inputs(T, H, I, torch.bfloat16, 4)
    h, gu = ffn.gated_forward(x, w, 2.0, save=True)
    dx, _ = ffn.gated_backward(dh, gu, x, w, 2.0, True, False)
    W = _f64(w)
    for lo in (0, T // 2, T - 300):
        X = _f64(x[lo:lo + 300])
        want, tol, z, ez = ref.gated(X, W, 2.0, EPS[torch.bfloat16])
        _within(h[lo:lo + 300], want, tol + TINY[torch.bfloat16], "h")
        _within(gu[lo:lo + 300], z, ez, "gu")
        (rx, tx), _ = ref.gated_grads(_f64(dh[lo:lo + 300]), _f64(gu[lo:lo + 300]), X, W, 2.0, EPS[torch.bfloat16],
                                      TINY[torch.bfloat16])
        _within(dx[lo:lo + 300], rx, tx, "dx")
