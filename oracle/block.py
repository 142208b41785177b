"""Definitions in float64, with error bounds, of the operators around a layer's experts: tokens sorted by expert and back, the
dense product with its epilogue, and the norms around a block. Numpy, on the host.

A bound counts roundings. U is half a step of fp32 at 1; `half` the result type's half step relative to a value, `tiny` half
its smallest step. A sum of fp32 terms is within (longest chain of additions) * U of the sum of magnitudes. The matrix
cores add at least eight exact products at a time, each partial sum rounded or cut (a whole step): K / 8 + 24 steps.
"""
from __future__ import annotations

import math

import numpy as np

U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


# ---------------------------------------------------------------------------------------------- tokens by expert


def order(ids, n, expert_map=None):
    """(row [T, k], pair [P], offsets [n + 1]) of a router's ids, one pair after the other."""
    ids = np.asarray(ids)
    local = []
    for i in ids.reshape(-1).tolist():
        if expert_map is not None:
            i = int(expert_map[i]) if 0 <= i < len(expert_map) else -1
        local.append(i if 0 <= i < n else n)
    lists = [[] for _ in range(n + 1)]
    for p, e in enumerate(local):
        lists[e].append(p)
    row, pair, offsets, r = [0] * len(local), [0] * len(local), [], 0
    for e, members in enumerate(lists):
        offsets.append(r)
        for p in members:
            row[p], pair[r] = (r, p) if e < n else (~r, ~p)
            r += 1
    return np.array(row, dtype=np.int64).reshape(ids.shape), np.array(pair, dtype=np.int64), np.array(offsets, dtype=np.int64)


def to_rows(x, row):
    out = np.zeros((row.size, x.shape[1]))
    flat = row.reshape(-1)
    live = np.flatnonzero(flat >= 0)
    out[flat[live]] = x[live // row.shape[1]]
    return out


def from_rows(rows, weights, row, shared, half, tiny):
    """(out, bound): a chain of k fused multiply-adds and one rounding."""
    T, k = row.shape
    out = np.zeros((T, rows.shape[1])) if shared is None else shared.astype(np.float64).copy()
    mag = np.abs(out)
    for j in range(k):
        live = row[:, j] >= 0
        w = np.ones(live.sum()) if weights is None else weights[live, j]
        v = w[:, None] * rows[row[live, j]]
        out[live] += v
        mag[live] += np.abs(v)
    e = (k + 1) * U * mag
    return out, e * (1 + half) + half * np.abs(out) + tiny


def from_rows_grads(dout, rows, weights, row, half, tiny):
    """((drows, bound), (dweights, bound before its own rounding)): a product and a rounding; a wave's lanes take every 64th group of
    eight products, then six additions."""
    T, k = row.shape
    drows, dw, ew = np.zeros_like(rows), np.zeros((T, k)), np.zeros((T, k))
    for t, j in np.ndindex(T, k):
        r = row[t, j]
        if r >= 0:
            drows[r] = weights[t, j] * dout[t]
            p = dout[t] * rows[r]
            dw[t, j] = p.sum()
            ew[t, j] = (rows.shape[1] / 64 + 16) * U * np.abs(p).sum()
    return (drows, np.abs(drows) * (half + 2 * U) + tiny), (dw, ew)


# ---------------------------------------------------------------------------------------------- the dense product


def _erf(z):
    return np.vectorize(math.erf, otypes=[float])(z)


def act(name, z):
    """(act(z), act'(z), bound of the fp32 evaluation of either, for an exact z).

    silu: e^-z carries (|z| + 2) U of itself, the reciprocal two steps; |z|^2 s (1 - s) stays under 0.54. gelu: the
    polynomial is within 4.2e-8 of erfc, 0.35 U of Phi, its half-term's evaluation within 12 U of at most 1/2. gelu_tanh: the
    argument v = 1.6 (z + ..) carries 5 U of itself, and |v| s (1 - s) stays under 0.23. Derivatives: the same errors times at
    most (1 + |z|) and, for gelu_tanh, the inner slope 1.6 (1 + 0.134 z^2) where s (1 - s) has not vanished: under 6."""
    if name is None:
        return z, np.ones_like(z), 0.0 * z
    if name == "relu":
        return np.maximum(z, 0.0), (z > 0).astype(float), 0.0 * z
    s = lambda v: 1.0 / (1.0 + np.exp(-np.clip(v, -700, 700)))  # noqa: E731
    e = 2.0 ** -20 * (1.0 + np.abs(z))
    if name == "silu":
        return z * s(z), s(z) * (1 + z * (1 - s(z))), e
    if name == "gelu":
        c = 0.5 * (1 + _erf(z / math.sqrt(2)))
        return z * c, c + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi), e
    a, b = 2 * math.sqrt(2 / math.pi), 0.044715
    v = s(a * (z + b * z ** 3))
    return z * v, v + z * v * (1 - v) * a * (1 + 3 * b * z * z), 4 * e


def linear(x, w, bias, name, residual, half, tiny):
    """(out, bound, z, bound of z): slopes of the activations stay under 1.13."""
    K = x.shape[1]
    z = x @ w.T
    ez = (K / 8 + 24) * 2 * U * (np.abs(x) @ np.abs(w).T)
    if bias is not None:
        z = z + bias
        ez = ez + U * np.abs(z)
    y, _, ey = act(name, z)
    ey = ey + 1.13 * ez
    if residual is not None:
        y = y + residual
        ey = ey + U * np.abs(y)
    return y, ey * (1 + half) + half * np.abs(y) + tiny, z, ez


def linear_grads(dy, z, x, w, name, half, tiny, fp16):
    """((dx, bound), (dw, bound), (dbias, bound before its rounding)) from the z that the kernel kept (None without activation).
    dz rounds once to the operand type; in fp16 it is held times 2^k, the largest in [2^14, 2^15): half the smallest step
    is then 2^-39 of the largest."""
    d, ed = dy, np.zeros_like(dy)
    if name is not None:
        _, slope, es = act(name, z)
        d = dy * slope
        ed = np.abs(dy) * es + 2 * U * np.abs(d)
    er = ed
    if name is not None:
        er = ed * (1 + half) + half * np.abs(d) + (np.abs(d).max(initial=0.0) * 2.0 ** -39 if fp16 and name != "relu" else tiny)
    M, N = dy.shape
    out = []
    for a, e, b, n in ((d, er, w, N), (d.T, er.T, x, M)):
        v = a @ b
        t = e @ np.abs(b) + (n / 8 + 24) * 2 * U * (np.abs(a) @ np.abs(b)) + n * U * 2.0 ** -20
        out.append((v, t * (1 + half) + half * np.abs(v) + tiny))
    db = d.sum(0)
    out.append((db, ed.sum(0) + (M / 8 + 32) * U * np.abs(d).sum(0)))
    return out


# ---------------------------------------------------------------------------------------------- the norms around a block

# The longest chains: a row's sum of squares is 16 values a thread and at most six plus sixteen additions, r(.) takes half its
# relative error and four operations; a value passes r(branch), post, gate, scale, the sum, r(s) and pre.
SUM = 48


def _r(v, eps):
    return 1.0 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)


def norm(branch, residual, post, gate, pre, eps, scale, residual_scale, half, tiny):
    """((s, bound), (y, bound)); y None without pre. gate broadcasts against branch."""
    g = 1.0 if gate is None else gate
    u = branch * (_r(branch, eps) * post) if post is not None else branch
    a = scale * g * u
    b = residual_scale * residual if residual is not None else np.zeros_like(branch)
    s = a + b
    e = (SUM / 2 + 10) * U * np.abs(a) + 2 * U * np.abs(b) + U * np.abs(s)
    out = (s, e * (1 + half) + half * np.abs(s) + tiny)
    if pre is None:
        return out, None
    r = _r(s, eps)
    y = s * r * pre
    # r(s) moves by at most the norm of s' errors over the norm of s, relatively
    er = np.sqrt((e * e).mean(-1, keepdims=True)) * r + (SUM / 2 + 6) * U
    ey = np.abs(r * pre) * e + np.abs(y) * (er + 3 * U)
    return out, (y, ey * (1 + half) + half * np.abs(y) + tiny)


def norm_grads(ds, dy, branch, residual, post, gate, pre, eps, scale, residual_scale):
    """{name: (gradient, magnitude)}: each gradient with the sum of the magnitudes of what it adds up. The kernel's fp32 evaluation
    takes at most 256 roundings on any path to a row's value (three row sums of SUM and the products between), plus the
    additions over the rows for the weights' sums: (256 + rows) * U of the magnitude, before the result's own rounding."""
    H = branch.shape[-1]
    g = 1.0 if gate is None else gate
    rb = _r(branch, eps) if post is not None else 1.0
    p = post if post is not None else 1.0
    nb = branch * rb
    u = nb * p
    b = residual_scale * residual if residual is not None else np.zeros_like(branch)
    s = scale * g * u + b
    gs = np.zeros_like(branch) if ds is None else ds
    mag = np.abs(gs)
    out = {}
    if dy is not None:
        rs = _r(s, eps)
        ns, mn = s * rs, (np.abs(scale * g * u) + np.abs(b)) * rs
        dn = dy * pre
        gs = gs + rs * (dn - ns * (ns * dn).mean(-1, keepdims=True))
        mag = mag + rs * (np.abs(dn) + mn * (mn * np.abs(dn)).mean(-1, keepdims=True) * (1 + 2 * (mn * mn).mean(-1, keepdims=True)))
        out["pre"] = (dy * ns).sum(0), (np.abs(dy) * mn * (1 + (mn * mn).mean(-1, keepdims=True))).sum(0)
    if residual is not None:
        out["residual"] = residual_scale * gs, np.abs(residual_scale) * mag
    if gate is not None:
        d, m = scale * gs * u, np.abs(scale * u) * mag
        axis = None if gate.shape == branch.shape else 0 if gate.ndim == 1 else -1
        out["gate"] = (d, m) if axis is None else (d.sum(axis, keepdims=axis == -1), m.sum(axis, keepdims=axis == -1))
    du, mu = scale * g * gs, np.abs(scale * g) * mag
    if post is not None:
        out["post"] = (du * nb).sum(0), (mu * np.abs(nb)).sum(0)
        du, mu = du * p, mu * np.abs(p)
        du = rb * (du - nb * (nb * du).sum(-1, keepdims=True) / H)
        mu = rb * (mu + np.abs(nb) * (np.abs(nb) * mu).sum(-1, keepdims=True) / H)
    out["branch"] = du, mu
    return out
