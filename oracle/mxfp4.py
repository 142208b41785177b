"""MXFP4 (OCP microscaled e2m1 with e8m0 scales per 32) and the gated feed-forward block in float64: the definitions that
the mxfp4 and ffn kernels are tested against, with bounds on how far fp32 sums and the final roundings may take them.
No counterpart in the reference; parity unpinned beyond the published format."""
from __future__ import annotations

import numpy as np

MAGS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDS = (MAGS[1:] + MAGS[:-1]) / 2


def quant_rows(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [rows, ceil(K/2)], scales uint8 [rows, ceil(K/32)]) of float32 rows."""
    x = np.asarray(x, np.float32)
    rows, K = x.shape
    nb = -(-K // 32)
    b = np.zeros((rows, nb * 32), np.float32)
    b[:, :K] = x
    b = b.reshape(rows, nb, 32)
    E = (np.abs(b).view(np.uint32) >> 23).max(-1).astype(np.int64)
    s = np.where(E == 255, 255, np.maximum(E - 2, 0))
    ok = s != 255
    v = np.where(ok[..., None], b, 0).astype(np.float64) * np.exp2(127.0 - np.where(ok, s, 127))[..., None]
    a = np.abs(v)
    lo, hi = np.searchsorted(MIDS, a, side="left"), np.searchsorted(MIDS, a, side="right")
    code = np.where(lo % 2 == 0, lo, hi) | np.where(np.signbit(v), 8, 0)     # ties to the even code
    code[~ok] = 0
    code = code.reshape(rows, -1)
    code[:, K:] = 0
    code = code[:, :2 * (-(-K // 2))]
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8), s.astype(np.uint8)


def values(q: np.ndarray, s: np.ndarray, K: int) -> np.ndarray:
    """float64 values [..., K]."""
    c = np.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], -1)[..., :K].astype(np.int64)
    v = np.where(c & 8, -1.0, 1.0) * MAGS[c & 7]
    f = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127.0))
    return v * np.repeat(f, 32, -1)[..., :K]


def rounded(x: np.ndarray) -> np.ndarray:
    """float64 rows (within fp32's range) to the nearest MXFP4 values."""
    x = np.asarray(x, np.float64)
    rows, K = x.shape
    b = x.reshape(rows, -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    e = np.maximum(np.floor(np.log2(np.maximum(top, 2.0 ** -126))) - 2, -127)
    a = np.abs(b) * np.exp2(-e)
    lo, hi = np.searchsorted(MIDS, a, side="left"), np.searchsorted(MIDS, a, side="right")
    return (np.sign(b) * MAGS[np.where(lo % 2 == 0, lo, hi)] * np.exp2(e)).reshape(rows, K)


def sigmoid(g):
    return 1.0 / (1.0 + np.exp(-g))


def swiglu(g, u, L):
    """(h, g', u')"""
    if L:
        g, u = np.minimum(g, L), np.clip(u, -L, L)
    return g * sigmoid(g) * u, g, u


def sum_err(terms_abs: np.ndarray, K: int) -> np.ndarray:
    """Bound of a fp32 sum of K products whose magnitudes sum to terms_abs: the accumulator is rounded (or cut) at most
    once per 8 products and once per joined part, by at most 2^-23 of the magnitudes so far."""
    return terms_abs * (K / 8 + 24) * 2.0 ** -23


def swiglu_err(g, u, L, eg, eu):
    """Bound of |h(g + eg, u + eu) - h(g, u)| plus fp32 evaluation: |silu'| <= 1.1, |silu(g)| <= |g|; the exponential's
    argument is off by |g| 2^-23 and five further operations by 2^-23 each."""
    h, gc, uc = swiglu(g, u, L)
    return 1.1 * eg * (np.abs(uc) + eu) + np.abs(gc * sigmoid(gc)) * eu + np.abs(h) * (np.abs(gc) + 8) * 2.0 ** -23


def moe(x, w13, w2, ids, wts, L, out_eps):
    """(out float64 [T, H], bound [T, H]) of the routed layer: x float64 rows (their input type's values), w13 [n, 2I, H]
    and w2 [n, H, I] float64 values, ids [T, k] (outside [0, n): no expert). The bound takes the SwiGLU output through
    its quantisation: where the values within fp32 error of h round to different MXFP4 values, both are allowed."""
    T, H = x.shape
    n, I = w13.shape[0], w13.shape[1] // 2
    out, tol = np.zeros((T, H)), np.zeros((T, H))
    xq = rounded(x)
    for t in range(T):
        for e, w in zip(ids[t], wts[t]):
            if not 0 <= e < n:
                continue
            z = w13[e] @ xq[t]
            ez = sum_err(np.abs(w13[e]) @ np.abs(xq[t]), H)
            g, u = z[:I], z[I:]
            h, _, _ = swiglu(g, u, L)
            eh = swiglu_err(g, u, L, ez[:I], ez[I:])
            q = rounded(h[None])[0]
            # a block's scale may move too: round at both ends of every value, with the block's largest at both ends
            spread = np.zeros(I)
            for sa in (-1, 1):
                for sb in (-1, 1):
                    hb = h.reshape(-1, 32).copy()
                    ebk = eh.reshape(-1, 32)
                    k = np.abs(hb).argmax(-1)
                    r = np.arange(len(hb))
                    top = hb[r, k] + sa * np.sign(hb[r, k]) * ebk[r, k]
                    hb = hb + sb * ebk
                    hb[r, k] = top
                    spread = np.maximum(spread, np.abs(rounded(hb.reshape(1, -1))[0] - q))
            y = w2[e] @ q
            ey = np.abs(w2[e]) @ spread + sum_err(np.abs(w2[e]) @ (np.abs(q) + spread), I)
            out[t] += w * y
            tol[t] += abs(w) * (ey + np.abs(y) * 2.0 ** -23)
    tol += np.abs(out) * (out_eps / 2 + 8 * 2.0 ** -23)
    return out, tol


def gated(x, w13, L, eps):
    """(h, bound, z, bound of z) of float64 x [T, H], w13 [2I, H]."""
    I, H = w13.shape[0] // 2, w13.shape[1]
    z = x @ w13.T
    ez = sum_err(np.abs(x) @ np.abs(w13).T, H)
    h, _, _ = swiglu(z[:, :I], z[:, I:], L)
    tol = swiglu_err(z[:, :I], z[:, I:], L, ez[:, :I], ez[:, I:])
    return h, tol * (1 + eps) + np.abs(h) * eps / 2, z, ez


def gated_grads(dh, z, x, w13, L, eps, tiny, tiny_d=None):
    """((dx, bound), (dw13, bound)) from float64 dh [T, I], the forward's z [T, 2I] as the kernel kept it (so masks and
    factors start from the same numbers), x and w13. d is rounded once to the operand type (eps; tiny_d: the smallest step
    it has there), the sums once more (tiny: the output type's smallest step, and d's unless tiny_d is given). z is finite."""
    tiny_d = tiny if tiny_d is None else tiny_d
    I = w13.shape[0] // 2
    g, u = z[:, :I], z[:, I:]
    mg, mu = (g <= L, np.abs(u) <= L) if L else (np.ones_like(g), np.ones_like(u))
    _, g, u = swiglu(g, u, L)
    s = sigmoid(g)
    dg, du = dh * u * s * (1 + g * (1 - s)) * mg, dh * g * s * mu
    d = np.concatenate([dg, du], -1)
    # fp32 evaluation: s within (|g| + 4) 2^-23 relative; 1 + g (1 - s) within that of 1 + |g|
    e = (np.abs(g) + 10) * 2.0 ** -23
    ed = np.concatenate([np.abs(dh * u * s) * (1 + np.abs(g)) * mg * 2 * e, np.abs(du) * e], -1)
    ed = ed + (np.abs(d) + ed) * eps / 2 + tiny_d
    res = []
    for a, ea, b, K in ((d, ed, w13, 2 * I), (d.T, ed.T, x, x.shape[0])):
        v = a @ b
        t = ea @ np.abs(b) + sum_err((np.abs(a) + ea) @ np.abs(b), K)
        res.append((v, t * (1 + eps) + np.abs(v) * eps / 2 + tiny))
    return res
