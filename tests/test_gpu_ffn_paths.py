"""The gated-block calls of tests/path_cases.py, which reach every kernel of its forward and gradients, against the float64
definitions (oracle/mxfp4.py) within its per-element bounds."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import path_cases as cases
from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.bfloat16, torch.float16]


def _f64(t):
    return t.detach().double().cpu().numpy()


def _id(c):
    return "-".join(str(v) for v in c if not isinstance(v, list))


def _inputs(T, H, I, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").to(dt)
    w = (torch.randn(2 * I, H, generator=g, device="cuda") * (3.0 / H ** 0.5)).to(dt)
    return x, w, torch.randn(T, I, generator=g, device="cuda").to(dt)


def _within(got, want, tol, what):
    bad = ~(np.abs(_f64(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], int(bad.sum()))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", cases.FORWARD, ids=_id)
def test_forward(cuda, case, dt):
    from mi355moe import ffn
    T, H, I, limit = case[:4]
    x, w, _ = _inputs(T, H, I, dt, T + H)
    h, gu = ffn.gated_forward(x, w, limit, save=True)
    want, tol, z, ez = ref.gated(_f64(x), _f64(w), limit, EPS[dt])
    _within(gu, z, ez, "gu")
    _within(h, want, tol + TINY[dt], "h")
    assert torch.equal(ffn.gated_forward(x, w, limit), h)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case,which", [(c, 0) for c in cases.DX] + [(c, 1) for c in cases.DW], ids=lambda v: _id(v) if isinstance(v, tuple) else str(v))
def test_gradients(cuda, case, which, dt):
    from mi355moe import ffn
    T, H, I, limit = case[:4]
    x, w, dh = _inputs(T, H, I, dt, T + H)
    _, gu = ffn.gated_forward(x, w, limit, save=True)
    got = ffn.gated_backward(dh, gu, x, w, limit, need_dx=which == 0, need_dw13=which == 1)
    assert got[1 - which] is None
    bounds = ref.gated_grads(_f64(dh), _f64(gu), _f64(x), _f64(w), limit, EPS[dt], TINY[dt])
    _within(got[which], *bounds[which], ("dx", "dw13")[which])
    both = ffn.gated_backward(dh, gu, x, w, limit)
    assert torch.equal(both[which], got[which])


@pytest.mark.parametrize("dt", TYPES)
def test_largest_weights(cuda, dt):
    """hidden 65536, intermediate 16384: W13's last row ends at 2^32 bytes. A few columns of h, dx and dw13, the last among them."""
    from mi355moe import ffn
    H, I, limit = 65536, 16384, 2.0
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(2 * I, H, dtype=dt, device="cuda")
    for r in range(0, 2 * I, 4096):                          # (in parts: normal_ in fp32 would take twice the room)
        w[r:r + 4096] = torch.randn(4096, H, generator=g, device="cuda") * (3.0 / H ** 0.5)
    rows = [0, 1, 4095, 8191, I - 2, I - 1]
    cols = [0, 7, 32767, 32768, H - 2, H - 1]
    for T in (3, 43):
        x = torch.randn(T, H, generator=g, device="cuda").to(dt)
        dh = torch.randn(T, I, generator=g, device="cuda").to(dt)
        h, gu = ffn.gated_forward(x, w, limit, save=True)
        pick = torch.tensor(rows + [I + r for r in rows], device="cuda")
        want, tol, z, ez = ref.gated(_f64(x), _f64(w[pick]), limit, EPS[dt])
        _within(gu[:, pick], z, ez, "gu")
        _within(h[:, rows], want, tol + TINY[dt], "h")
        dx, dw = ffn.gated_backward(dh, gu, x, w, limit)
        (rx, tx), (rw, tw) = ref.gated_grads(_f64(dh), _f64(gu), _f64(x[:, cols]), _f64(w[:, cols]), limit, EPS[dt], TINY[dt])
        _within(dx[:, cols], rx, tx, "dx")
        _within(dw[:, cols], rw, tw, "dw13")


def test_most_rows(cuda):
    """2^24 rows, the most a call takes."""
    from mi355moe import ffn
    T, H, I, limit, dt = 1 << 24, 8, 8, 1.0, torch.bfloat16
    x, w, dh = _inputs(T, H, I, dt, 3)
    h, gu = ffn.gated_forward(x, w, limit, save=True)
    dx, dw = ffn.gated_backward(dh, gu, x, w, limit)
    for lo in (0, T // 2 - 100, T - 200):
        s = slice(lo, lo + 200)
        want, tol, z, ez = ref.gated(_f64(x[s]), _f64(w), limit, EPS[dt])
        _within(gu[s], z, ez, "gu")
        _within(h[s], want, tol + TINY[dt], "h")
        (rx, tx), _ = ref.gated_grads(_f64(dh[s]), _f64(gu[s]), _f64(x[s]), _f64(w), limit, EPS[dt], TINY[dt])
        _within(dx[s], rx, tx, "dx")
    # dw13 in 256 parts of the tokens: float64 on the GPU. d carries half a step and fp32 evaluation; a part's sum is rounded at
    # most once per 8 products, the parts' once each
    z = gu.double()
    gr, up = z[:, :I], z[:, I:]
    gc, uc, d = gr.clamp(max=limit), up.clamp(-limit, limit), dh.double()
    s = torch.sigmoid(gc)
    D = torch.cat([d * uc * s * (1 + gc * (1 - s)) * (gr <= limit), d * gc * s * (up.abs() <= limit)], 1)
    eD = D.abs() * (EPS[dt] / 2 + 2.0 ** -18) + 2.0 ** -18 * d.abs().repeat(1, 2) * limit
    X = x.double()
    v, m = D.t().contiguous() @ X, D.abs().t().contiguous() @ X.abs()
    tol = (eD.t().contiguous() @ X.abs() + m * (T / 256 / 8 + 24 + 256) * 2.0 ** -23) * (1 + EPS[dt]) + v.abs() * EPS[dt] / 2
    assert ((dw.double() - v).abs() <= tol).all()
    with pytest.raises(RuntimeError, match="code 3"):
        ffn.gated_forward(x.new_empty(T + 1, H), w, limit)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", [(8192, 4096, 2048), (130, 264, 2056), (8203, 136, 72)], ids=_id)
def test_training_steps_repeat(cuda, size, dt):
    """The same step gives the same bits: on the largest tiles, and where a gradient's sum is cut into parts."""
    from mi355moe import ffn
    x, w, dh = _inputs(*size, dt, 3)

    def step():
        h, gu = ffn.gated_forward(x, w, 10.0, save=True)
        return (h, gu, *ffn.gated_backward(dh, gu, x, w, 10.0))

    first = step()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
