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
