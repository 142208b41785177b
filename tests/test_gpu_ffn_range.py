"""The gated block's gradients in fp16 over its range: [dg | du] is an operand of two products, and a loss-scaled dh takes it
past fp16's largest value, a small one under its smallest, where the gradients themselves are ordinary numbers."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu

F16 = torch.float16
EPS, TINY = 2.0 ** -10, 2.0 ** -24


def _f64(t):
    return t.detach().double().cpu().numpy()


def _inputs(T, H, I, xs, zs, dhs, seed):
    """x of deviation xs, z of about zs, dh of magnitudes up to dhs."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(T, H, generator=g, device="cuda") * xs).half()
    w = (torch.randn(2 * I, H, generator=g, device="cuda") * (zs / xs / H ** 0.5)).half()
    dh = ((torch.rand(T, I, generator=g, device="cuda") * 2 - 1) * dhs).half()
    return x, w, dh


def _bounds(dh, gu, x, w, L):
    """float64 gradients and their bounds. d is held in fp16 times a power of two that brings its largest magnitude into
    [2^14, 2^15): its smallest step is at most 2^-38 of that magnitude (2^-24 of fp16's over 2^14)."""
    z, I = _f64(gu), gu.shape[1] // 2
    g, u = np.minimum(z[:, :I], L), np.clip(z[:, I:], -L, L)
    s = ref.sigmoid(g)
    d = _f64(dh)
    top = max(np.abs(d * u * s * (1 + g * (1 - s)) * (z[:, :I] <= L)).max(), np.abs(d * g * s * (np.abs(z[:, I:]) <= L)).max())
    return ref.gated_grads(d, z, _f64(x), _f64(w), L, EPS, TINY, tiny_d=top * 2.0 ** -38)


# T, H, I: products by small tiles, by every size of tile and in parts
@pytest.mark.parametrize("T,H,I", [(1, 64, 24), (33, 64, 72), (260, 136, 40), (1100, 1096, 520), (97, 72, 1800), (3400, 24, 8)])
@pytest.mark.parametrize("dhs", [60000.0, 1.0, 2.0 ** -18])
def test_gradients_over_the_range(cuda, T, H, I, dhs):
    from mi355moe import ffn
    L = 10.0
    # x large and w13 small, and the other way round: the first keeps dx, the second most of dw13 within fp16
    for which, xs in (("dx", 2000.0), ("dw", 0.02)):
        x, w, dh = _inputs(T, H, I, xs, 6.0, dhs, T + H)
        _, gu = ffn.gated_forward(x, w, L, save=True)
        dx, dw = ffn.gated_backward(dh, gu, x, w, L)
        want = _bounds(dh, gu, x, w, L)
        for name, got, (v, tol) in (("dx", dx, want[0]), ("dw", dw, want[1])):
            out = _f64(got)
            fits = np.abs(v) + tol < 65504
            if name == which:
                assert fits.any()                             # (the others are held to an infinity below)
            bad = fits & ~(np.abs(out - v) <= tol)
            bad |= (np.abs(v) - tol >= 65520) & (out != np.copysign(np.inf, v))   # fp16's largest value and half a step more
            assert not bad.any(), (name, xs, np.argwhere(bad)[:5], int(bad.sum()))


def test_non_finite_rows_stay_apart(cuda):
    """A NaN and an infinity among the rows: the other rows' dx is what it is without them, at magnitudes past fp16's."""
    from mi355moe import ffn
    T, H, I, L = 200, 64, 24, 10.0
    x, w, dh = _inputs(T, H, I, 2000.0, 6.0, 60000.0, 3)
    keep = [t for t in range(T) if t not in (2, 4)]
    _, gu = ffn.gated_forward(x, w, L, save=True)
    (v, tol), _ = _bounds(dh[keep], gu[keep], x[keep], w, L)
    dh[2, 3], x[4, 5] = float("inf"), float("nan")
    _, gu = ffn.gated_forward(x, w, L, save=True)
    dx, _ = ffn.gated_backward(dh, gu, x, w, L)
    assert (np.abs(_f64(dx[keep]) - v) <= tol).all()
    assert not torch.isfinite(dx[2]).any() and torch.isnan(dx[4]).all()


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_zero_gradient_and_repeats(cuda, dt):
    """dh of zeros gives zeros; two runs give the same bits."""
    from mi355moe import ffn
    x, w, dh = (t.to(dt) for t in _inputs(1100, 264, 136, 1.0, 4.0, 3.0, 9))
    _, gu = ffn.gated_forward(x, w, 10.0, save=True)
    dx, dw = ffn.gated_backward(torch.zeros_like(dh), gu, x, w, 10.0)
    assert (dx == 0).all() and (dw == 0).all()
    first = ffn.gated_backward(dh, gu, x, w, 10.0)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ffn.gated_backward(dh, gu, x, w, 10.0)))


def test_captured_gradients_follow_their_inputs(cuda):
    """Replays with dh of other magnitudes, eager work in between: the power of two is the replay's own."""
    from mi355moe import ffn
    x, w, dh = _inputs(300, 264, 72, 1.0, 4.0, 1.0, 4)
    _, gu = ffn.gated_forward(x, w, 10.0, save=True)
    ffn.gated_backward(dh, gu, x, w, 10.0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = ffn.gated_backward(dh, gu, x, w, 10.0)
    for scale in (1.0, 2.0 ** 14, 2.0 ** -20, 0.0, 3.0):
        dh.copy_(_inputs(300, 264, 72, 1.0, 4.0, scale, 5)[2])
        g.replay()
        want = ffn.gated_backward(dh, gu, x, w, 10.0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
