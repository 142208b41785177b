"""Every kernel of the operators around a layer's experts at the sizes that take it (tests/block_cases.py), against float64 within
the bounds of oracle/block.py: samples of rows and columns where the products are large."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import block_cases as cases
from oracle import block as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _name(dt):
    return str(dt).replace("torch.", "")


def _f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _within(got, want, tol, what):
    bad = ~(np.abs(_f64(got) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:5], int(bad.sum()))


def _some(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return sorted({0, n - 1, *torch.randint(0, n, (k,), generator=g).tolist()})


def _inputs(M, K, N, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return new(M, K).to(dt), (new(N, K) * (2.0 / K ** 0.5)).to(dt), new(N), new(M, N).to(dt), new(M, N).to(dt)


@pytest.mark.parametrize("case", cases.LINEAR, ids=lambda c: "x".join(map(str, c[:3])))
@pytest.mark.parametrize("dt", TYPES[:2])
def test_linear(cuda, case, dt):
    from mi355moe import ffn
    M, K, N = case[:3]
    x, w, b, r, _ = _inputs(M, K, N, dt, 1)
    out, z = ffn.linear_forward(x, w, b, "gelu", r, save=True)
    rows = _some(M, 24, 2)
    want, tol, wz, ez = ref.linear(_f64(x[rows]), _f64(w), _f64(b), "gelu", _f64(r[rows]), ref.HALF[_name(dt)], ref.TINY[_name(dt)])
    _within(out[rows], want, tol, "out")
    _within(z[rows], wz, ez, "z")
    assert all(torch.equal(p, q) for p, q in zip(ffn.linear_forward(x, w, b, "gelu", r, save=True), (out, z)))


@pytest.mark.parametrize("which", ["dx", "dw"])
@pytest.mark.parametrize("at", range(len(cases.DX)))
@pytest.mark.parametrize("dt", TYPES[:2])
def test_linear_gradients(cuda, which, at, dt):
    from mi355moe import ffn
    M, K, N = (cases.DX if which == "dx" else cases.DW)[at][:3]
    x, w, _, _, dy = _inputs(M, K, N, dt, 3)
    h, t = ref.HALF[_name(dt)], ref.TINY[_name(dt)]
    cols = _some(K, 16, 4)
    for act in (None, "silu"):
        z = None if act is None else ffn.linear_forward(x, w, None, act, save=True)[1]
        dx, dw, db = ffn.linear_backward(dy, z, x, w, act, torch.float32, which == "dx", which == "dw")
        gx, gw, gb = ref.linear_grads(_f64(dy), _f64(z), _f64(x[:, cols]), _f64(w[:, cols]), act, h, t, dt == torch.float16)
        if which == "dx":
            _within(dx[:, cols], *gx, "dx")
        else:
            _within(dw[:, cols], *gw, "dw")
        _within(db, *gb, "db")
        again = ffn.linear_backward(dy, z, x, w, act, torch.float32, which == "dx", which == "dw")
        assert all(p is None or torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))


@pytest.mark.parametrize("case", cases.NORM, ids=lambda c: "x".join(map(str, c[:2])))
@pytest.mark.parametrize("dt", TYPES)
def test_norm(cuda, case, dt):
    from mi355moe import norm
    R, H = case[:2]
    g = torch.Generator(device="cuda").manual_seed(R)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    args = [new(R, H).to(dt), (2 * new(R, H)).to(dt), 1 + 0.2 * new(H), new(H).to(dt), 1 + 0.2 * new(H)]
    ds, dy = new(R, H).to(dt), new(R, H).to(dt)
    s, y, stats = norm.join_forward(*args, 1e-5, 0.5, 1.25)
    got = norm.join_backward(ds, dy, stats, *args, 0.5, 1.25)
    d = _name(dt)
    h, t = ref.HALF[d], ref.TINY[d]
    rows = _some(R, 12, 5)
    f = [_f64(a if a.dim() == 1 else a[rows]) for a in args]
    (ws, es), (wy, ey) = ref.norm(*f, 1e-5, 0.5, 1.25, h, t)
    _within(s[rows], ws, es, "s")
    _within(y[rows], wy, ey, "y")
    want = ref.norm_grads(_f64(ds[rows]), _f64(dy[rows]), *f, 1e-5, 0.5, 1.25)
    for i, k in ((0, "branch"), (1, "residual")):
        value, mag = want[k]
        _within(got[i][rows], value, 256 * ref.U * mag * (1 + h) + h * np.abs(value) + t, k)
    # the sums over the rows, on the GPU in float64
    b, r, p, c, w = (a.double() for a in args)
    rms = lambda v: 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    nb = b * rms(b)
    a_, b_ = 0.5 * c * nb * p, 1.25 * r
    tot = a_ + b_
    rs = rms(tot)
    ns, mn = tot * rs, (a_.abs() + b_.abs()) * rs
    D, S = dy.double(), ds.double()
    gs = S + rs * (D * w - ns * (ns * D * w).mean(-1, keepdim=True))
    m = S.abs() + rs * ((D * w).abs() + mn * (mn * (D * w).abs()).mean(-1, keepdim=True) * (1 + 2 * (mn * mn).mean(-1, keepdim=True)))
    e = (256 + R) * ref.U
    assert ((got[4].double() - (D * ns).sum(0)).abs() <= e * (D.abs() * mn * (1 + (mn * mn).mean(-1, keepdim=True))).sum(0)).all()
    assert ((got[2].double() - (0.5 * c * gs * nb).sum(0)).abs() <= e * (0.5 * c * m * nb).abs().sum(0)).all()
    v = (0.5 * gs * nb * p).sum(0)
    assert ((got[3].double() - v).abs() <= e * (0.5 * m * nb * p).abs().sum(0) * (1 + h) + h * v.abs() + t).all()
    again = norm.join_backward(ds, dy, stats, *args, 0.5, 1.25)
    assert all(torch.equal(p, q) for p, q in zip(again, got))


@pytest.mark.parametrize("case", cases.ROWS, ids=lambda c: "x".join(map(str, c[:3])))
@pytest.mark.parametrize("dt", TYPES)
def test_rows(cuda, case, dt):
    from mi355moe import dispatch
    T, k, H = case[:3]
    g = torch.Generator(device="cuda").manual_seed(T)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ids = torch.randint(0, 60, (T, k), generator=torch.Generator().manual_seed(1)).cuda()
    plan = dispatch.sort_tokens(ids, 50)                         # a sixth of the pairs is dropped
    row = plan.row.cpu().numpy()
    assert np.array_equal(row, ref.order(ids.cpu().numpy(), 50)[0])
    x, y, w, sh, d = new(T, H).to(dt), new(T * k, H).to(dt), new(T, k), new(T, H).to(dt), new(T, H).to(dt)
    rows = dispatch.to_experts(x, plan)
    assert np.array_equal(_f64(rows), ref.to_rows(_f64(x), row))
    h, t = ref.HALF[_name(dt)], ref.TINY[_name(dt)]
    toks = _some(T, 200, 6)
    out = dispatch.from_experts(y, w, plan, shared=sh)
    Y = _f64(y)
    _within(out[toks], *ref.from_rows(Y, _f64(w[toks]), row[toks], _f64(sh[toks]), h, t), "out")
    dy, dw = dispatch.from_experts_backward(d, y, w, plan)
    (ry, ty), (rw, tw) = ref.from_rows_grads(_f64(d[toks]), Y, _f64(w[toks]), row[toks], h, t)
    _within(dw[toks], rw, tw + ref.HALF["float32"] * np.abs(rw), "dw")
    at = row[toks].reshape(-1)
    at = at[at >= 0]
    _within(dy[at.tolist()], ry[at], ty[at], "dy")
    assert (dy[int(plan.offsets[-1]):] == 0).all()


@pytest.mark.parametrize("case", cases.SORT, ids=lambda c: "x".join(map(str, c[:3])))
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(cuda, case, dtype):
    from mi355moe import dispatch
    T, k, n = case[:3]
    ids = torch.randint(-2, n + 2, (T, k), generator=torch.Generator().manual_seed(T)).to(dtype)
    row, pair, offsets = ref.order(ids.numpy(), n)
    plan = dispatch.sort_tokens(ids.cuda(), n)
    assert np.array_equal(plan.row.cpu().numpy(), row) and np.array_equal(plan.pair.cpu().numpy(), pair)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
