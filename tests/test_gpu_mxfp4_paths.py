"""The MXFP4 calls of tests/path_cases.py, which reach every kernel of theirs, against the float64 definitions (oracle/mxfp4.py)
within its per-element bounds: ragged sizes, scales in either order, expert maps, foreign and repeated ids, accumulation,
non-finite rows and NaN blocks, and scale codes over their whole range."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import path_cases as cases
from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.bfloat16, torch.float32, torch.float16]


def _np(t):
    return t.detach().cpu().numpy()


def _f64(t):
    return t.detach().double().cpu().numpy()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _id(c):
    return "-".join(str(v) for v in c if not isinstance(v, list))


# ---------------------------------------------------------------------------------------------- products


def _mx(rows, K, seed, lo=118, hi=124):
    g = _gen(seed)
    q = torch.randint(0, 256, (rows, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    return q, torch.randint(lo, hi, (rows, K // 32), generator=g, device="cuda", dtype=torch.uint8)


@pytest.mark.parametrize("case", cases.PRODUCTS, ids=_id)
def test_product(cuda, case):
    from mi355moe import mxfp4
    M, N, K = case[:3]
    odt = TYPES[(M + K) % 3]
    a, sa = _mx(M, K, M + K)
    w, sw = _mx(N, K, N + 2 * K)
    A, W = ref.values(_np(a), _np(sa), K), ref.values(_np(w), _np(sw), K)
    out = mxfp4.matmul(a, sa, w, sw, out_dtype=odt)
    want = A @ W.T
    tol = ref.sum_err(np.abs(A) @ np.abs(W).T, K) * 2 + np.abs(want) * EPS[odt] / 2 + TINY[odt]
    bad = ~(np.abs(_f64(out) - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], int(bad.sum()))
    # NaN blocks: the row's last block (in a partial stage where K has one) and the column's first one
    sa2, sw2 = sa.clone(), sw.clone()
    sa2[M - 1, -1], sw2[N // 2, 0], sw2[0, -1] = 255, 255, 255
    got = mxfp4.matmul(a, sa2, w, sw2, out_dtype=odt)
    nan = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    nan[M - 1], nan[:, N // 2], nan[:, 0] = True, True, True
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], out[~nan])


SPREAD = [0, 1, 3, 40, 90, 127, 150, 200, 251, 253, 254]


@pytest.mark.parametrize("M,N,K", [(5, 40, 192), (11, 40, 1024), (100, 40, 192), (100, 40, 1152), (200, 257, 384), (500, 4000, 384),
                                   (1100, 2000, 160), (2100, 2500, 128), (100, 70, 8320), (4100, 3400, 288)])
def test_scale_codes_over_their_range(cuda, M, N, K):
    """Each row around one of SPREAD: pairs such as 254 with 0 give ordinary numbers, two large ones infinities and two small
    ones zeros. Rows of zero codes stay zero under any scale."""
    from mi355moe import mxfp4
    rng = np.random.default_rng(M + K)

    def scales(rows):
        base = np.array(SPREAD)[np.arange(rows) % len(SPREAD)][:, None]
        return torch.from_numpy(np.clip(base + rng.integers(-3, 4, (rows, K // 32)), 0, 254).astype(np.uint8)).cuda()

    a, _ = _mx(M, K, 1)
    w, _ = _mx(N, K, 2)
    a[M // 2], w[N // 3] = 0, 0x80                           # zeros, and zeros of either sign
    sa, sw = scales(M), scales(N)
    out = _f64(mxfp4.matmul(a, sa, w, sw, out_dtype=torch.float32))
    A, W = ref.values(_np(a), _np(sa), K), ref.values(_np(w), _np(sw), K)
    want, mags = A @ W.T, np.abs(A) @ np.abs(W).T
    assert (out[M // 2] == 0).all() and (out[:, N // 3] == 0).all()
    # fp32 sums hold what lies above its smallest normal number; each of the K / 64 steps may flush what lies below it
    tol = ref.sum_err(mags, K) * 2 + np.abs(want) * 2.0 ** -24 + (K / 64 + 1) * 2.0 ** -126
    ordinary = mags < 2.0 ** 127                             # no partial sum leaves fp32
    bad = ordinary & ~(np.abs(out - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], int(bad.sum()))
    over = np.abs(want) - tol >= 2.0 ** 128                  # these do, whatever the order of the sum
    assert not np.isfinite(out[over]).any()
    assert (ordinary & (np.abs(want) > 2.0 ** -100)).any() and (over.any() or M < len(SPREAD))


# ---------------------------------------------------------------------------------------------- routed experts


def _layer(n, H, I, seed):
    from mi355moe import mxfp4
    g = _gen(seed)
    w13 = torch.randn(n, 2 * I, H, generator=g, device="cuda") * (3.0 / H ** 0.5)
    w2 = torch.randn(n, H, I, generator=g, device="cuda") * (1.0 / I ** 0.5)
    return mxfp4.Mxfp4Experts.from_dense(w13, w2)


def _dense(ex):
    return ref.values(_np(ex.w13), _np(ex.w13_scale), ex.K), ref.values(_np(ex.w2), _np(ex.w2_scale), ex.N)


def _routing(T, n, topk, seed):
    """Picks without repetition, but for a token of one expert alone, one with no expert and two foreign picks."""
    rng = np.random.default_rng(seed)
    ids = np.argsort(rng.random((T, n)), 1)[:, :topk] if topk <= n else rng.integers(0, n, (T, topk))
    ids = ids.astype(np.int64)
    ids[1] = ids[1, 0]
    ids[3] = -1
    if topk > 1:
        ids[0, 0], ids[T // 2, topk - 1] = -1, n + 1
    w = rng.random((T, topk)).astype(np.float32) + 0.1
    return ids, w / w.sum(-1, keepdims=True) * 2.5


@pytest.mark.parametrize("case", cases.ROUTED, ids=_id)
def test_routed(cuda, case):
    from mi355moe import mxfp4
    n, H, I, T, k, limit = case[:6]
    dt = TYPES[(n + H + T) % 3]
    ex = _layer(n, H, I, 11 + n)
    w13, w2 = _dense(ex)
    wide = torch.randn(T, H + 11, generator=_gen(T), device="cuda").to(dt)
    x = wide[:, 3:3 + H]                                     # rows at odd addresses
    ids, w = _routing(T, n, k, 13 + H)
    tid, tw = torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()
    want, tol = ref.moe(_f64(x), w13, w2, ids, w.astype(np.float64), limit, EPS[dt])
    tol = tol + TINY[dt]

    def check(got, base=0.0, more=0.0):
        bad = ~(np.abs(_f64(got) - (want + base)) <= tol + more)
        assert not bad.any(), (np.argwhere(bad)[:5], int(bad.sum()))

    out = mxfp4.moe_forward_ids(ex, x, tid, tw, limit=limit)
    assert out.dtype == dt and (out[3] == 0).all()
    check(out)
    assert torch.equal(out, mxfp4.moe_forward_ids(ex, x, tid.int(), tw, limit=limit))
    # a strided out: written, then added to, its neighbours left as they were
    buf = torch.full((T + 2, H + 5), 3.0, dtype=dt, device="cuda")
    view = buf[1:T + 1, 2:2 + H]
    mxfp4.moe_forward_ids(ex, x, tid, tw, limit=limit, out=view)
    assert torch.equal(view, out)
    shared = torch.randn(T, H, generator=_gen(5), device="cuda").to(dt)
    view.copy_(shared)
    mxfp4.moe_forward_ids(ex, x, tid, tw, limit=limit, out=view, accumulate=True)
    base = _f64(shared)
    check(view, base, np.abs(base + want) * EPS[dt] / 2 + np.abs(base) * 2.0 ** -22)
    assert torch.equal(view[3], shared[3])
    view.fill_(3.0)
    assert (buf == 3.0).all()
    # a map of two more ids than experts: local ids shuffled, the others foreign
    perm = np.random.default_rng(2).permutation(n + 2)
    emap = np.where(perm < n, perm, -1)
    back = np.argsort(perm)                                  # global id of a local one
    gids = np.where((ids >= 0) & (ids < n), back[np.clip(ids, 0, n - 1)], np.where(ids < 0, back[n], n + 2))
    check(mxfp4.moe_forward_ids(ex, x, torch.from_numpy(gids).cuda(), tw, limit=limit, expert_map=torch.from_numpy(emap).cuda()))
    # non-finite rows stay apart
    bad = x.clone()
    bad[2, H // 2], bad[T - 1, H - 1] = float("nan"), float("inf")
    got = mxfp4.moe_forward_ids(ex, bad, tid, tw, limit=limit)
    rows = [t for t in range(T) if t not in (2, T - 1)]
    assert torch.isnan(got[2]).all() and torch.isnan(got[T - 1]).all() and torch.equal(got[rows], out[rows])


@pytest.mark.parametrize("case", cases.ROUTED[:1] + cases.ROUTED[5:6] + cases.ROUTED[8:9], ids=_id)
def test_one_expert_takes_all(cuda, case):
    """Skewed routing: every token picks the same expert (and itself again), the others none."""
    from mi355moe import mxfp4
    n, H, I, T, k, limit = case[:6]
    ex = _layer(n, H, I, 3)
    w13, w2 = _dense(ex)
    x = torch.randn(T, H, generator=_gen(T), device="cuda").half()
    ids, w = np.full((T, k), n - 1), np.random.default_rng(1).random((T, k)).astype(np.float32)
    out = mxfp4.moe_forward_ids(ex, x, torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), limit=limit)
    want, tol = ref.moe(_f64(x), w13, w2, ids, w.astype(np.float64), limit, EPS[torch.float16])
    assert (np.abs(_f64(out) - want) <= tol + TINY[torch.float16]).all()


@pytest.mark.parametrize("case", cases.STORED, ids=_id)
def test_scales_as_they_come(cuda, case):
    """arrange=False with rows of an odd number of half steps: the same bits as with arranged scales, and within the bounds."""
    from mi355moe import fused_experts_mxfp4, mxfp4
    n, H, I, T, k = case[:5]
    dt = torch.bfloat16
    ex = _layer(n, H, I, 7)
    raw = mxfp4.Mxfp4Experts(ex.w13, ex.w13_scale, ex.w2, ex.w2_scale, arrange=False)
    x = torch.randn(T, H, generator=_gen(T), device="cuda").to(dt)
    ids, w = _routing(T, n, k, 5)
    tid, tw = torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()
    out = mxfp4.moe_forward_ids(raw, x, tid, tw)
    assert torch.equal(out, mxfp4.moe_forward_ids(ex, x, tid, tw))
    assert torch.equal(out, fused_experts_mxfp4(x, ex.w13, ex.w2, tw, tid, (ex.w13_scale, ex.w2_scale)))
    w13, w2 = _dense(ex)
    want, tol = ref.moe(_f64(x), w13, w2, ids, w.astype(np.float64), 10.0, EPS[dt])
    assert (np.abs(_f64(out) - want) <= tol + TINY[dt]).all()


@pytest.mark.parametrize("case", cases.STORED + cases.ROUTED[:1] + cases.ROUTED[5:6] + cases.ROUTED[8:9], ids=_id)
def test_nan_blocks_of_weights(cuda, case):
    """A NaN block in the last, partial step of a down row: that column of its expert's tokens and nothing else. One in a gate
    or up row: its expert's tokens whole."""
    from mi355moe import mxfp4
    n, H, I, T, k = case[:5]
    x = torch.randn(T, H, generator=_gen(T), device="cuda").bfloat16()
    ids, w = _routing(T, n, k, 5)
    tid, tw = torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()
    e2, e13, col = 0, n - 1, H - 3
    for arrange in ((True, False) if H % 128 == 0 and I % 128 == 0 else (True,)):
        ex = _layer(n, H, I, 7)
        out = mxfp4.moe_forward_ids(mxfp4.Mxfp4Experts(ex.w13, ex.w13_scale, ex.w2, ex.w2_scale, arrange=arrange), x, tid, tw)
        assert torch.isfinite(out).all()
        s13, s2 = ex.w13_scale.clone(), ex.w2_scale.clone()
        s13[e13, I + 5, -1], s2[e2, col, -1] = 255, 255
        got = mxfp4.moe_forward_ids(mxfp4.Mxfp4Experts(ex.w13, s13, ex.w2, s2, arrange=arrange), x, tid, tw)
        nan = torch.zeros(T, H, dtype=torch.bool, device="cuda")
        nan[(tid == e2).any(1), col] = True
        nan[(tid == e13).any(1)] = True
        assert torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], out[~nan])


@pytest.mark.parametrize("T,k", [(65536, 1), (2048, 32), (8191, 8)])
def test_most_pairs(cuda, T, k):
    """65536 pairs, the most a call takes, and picks of 32 experts; a sample of the tokens."""
    from mi355moe import mxfp4
    n, H, I, limit, dt = 64, 96, 32, 2.0, torch.bfloat16
    ex = _layer(n, H, I, 9)
    x = torch.randn(T, H, generator=_gen(T), device="cuda").to(dt)
    ids, w = _routing(T, n, k, 3)
    tid, tw = torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()
    out = mxfp4.moe_forward_ids(ex, x, tid, tw, limit=limit)
    some = np.unique(np.concatenate([[0, 1, 2, 3, T // 2, T - 1], np.random.default_rng(1).integers(0, T, 60)]))
    w13, w2 = _dense(ex)
    want, tol = ref.moe(_f64(x)[some], w13, w2, ids[some], w[some].astype(np.float64), limit, EPS[dt])
    # (32 pairs a token: their sum is rounded once a pair, on sums of up to all their magnitudes)
    each = sum(np.abs(ref.moe(_f64(x)[some], w13, w2, ids[some, j:j + 1], w[some, j:j + 1].astype(np.float64), limit, 0.0)[0]) for j in range(k))
    assert (np.abs(_f64(out)[some] - want) <= tol + each * k * 2.0 ** -24 + TINY[dt]).all()
    with pytest.raises(ValueError, match="unsupported size"):
        mxfp4.moe_forward_ids(ex, x.new_zeros(65537, H), torch.zeros(65537, 1, dtype=torch.int32, device="cuda"), torch.zeros(65537, 1, device="cuda"))
