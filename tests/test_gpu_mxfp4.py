"""GPU parity of the MXFP4 operators (mi355moe.mxfp4) with their definitions in float64 (oracle/mxfp4.py):

  - quantisation is bit-exact (codes and scales), reading back exact in fp32;
  - products and routed layers stay within bounds that count roundings: fp32 sums by their length and the magnitudes
    summed, the output type by half a step, and for the routed layer both MXFP4 values where a SwiGLU output lies within
    fp32 error of a tie. The bounds are computed per element, none is fitted.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mxfp4 as ref

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def _np(t):
    return t.detach().cpu().numpy()


def _f64(t):
    return t.detach().double().cpu().numpy()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(rows, K, dt, seed):
    g = _gen(seed)
    x = torch.randn(rows, K, generator=g, device="cuda")
    return (x * torch.logspace(-3, 3, rows, device="cuda")[:, None]).to(dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 1), (3, 33), (5, 31), (37, 4096), (9, 96), (2, 1002), (130, 160), (1, 7)])
def test_quant_rows_bit_exact(cuda, dt, rows, K):
    from mi355moe import mxfp4
    x = _rows(rows, K, dt, 3 + K)
    q, s = mxfp4.quant_rows(x)
    qo, so = ref.quant_rows(_np(x.float()))
    assert np.array_equal(_np(s), so)
    assert np.array_equal(_np(q), qo)
    v = mxfp4.dequant_rows(q, s, K, out_dtype=torch.float32)
    assert np.array_equal(_f64(v), ref.values(qo, so, K))


def test_quant_rows_ties_and_extremes(cuda):
    from mi355moe import mxfp4
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9, 0.0, -0.0, -0.25, -0.75, -5.0, 4.0, 1e-30])
    rows = [torch.cat([ties, -ties]), torch.zeros(32), torch.full((32,), 2.0 ** -149), torch.full((32,), 3.4e38),
            torch.full((32,), 2.0 ** -126), torch.linspace(-2.0 ** -126, 2.0 ** -125, 32)]
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.linspace(-3, 3, 32)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows).cuda()
    q, s = mxfp4.quant_rows(x)
    qo, so = ref.quant_rows(_np(x))
    assert np.array_equal(_np(s), so) and np.array_equal(_np(q), qo)
    v = _f64(mxfp4.dequant_rows(q, s, out_dtype=torch.float32))
    assert np.isnan(v[6:]).all() and np.array_equal(v[:6], ref.values(qo, so, 32)[:6])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_quant_rows_strides_and_offsets(cuda, dt):
    from mi355moe import mxfp4
    base = _rows(9, 300, dt, 5)
    for x in (base[:, 1:257], base[::2, 3:99], base[:, :128], base[4:5, 8:72], base[:, 8:264]):
        q, s = mxfp4.quant_rows(x)
        q2, s2 = mxfp4.quant_rows(x.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("odt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("K", [64, 37, 1001])
def test_dequant_rows_types(cuda, odt, K):
    from mi355moe import mxfp4
    g = _gen(K)
    q = torch.randint(0, 256, (11, (K + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.randint(100, 140, (11, -(-K // 32)), generator=g, device="cuda", dtype=torch.uint8)
    s[3, 0] = 255
    got = mxfp4.dequant_rows(q, s, K, out_dtype=odt)
    want = torch.from_numpy(ref.values(_np(q), _np(s), K)).to(torch.float32).to(odt)
    assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-77.0), torch.nan_to_num(want.float(), nan=-77.0))


def _mx(rows, K, seed, lo=118, hi=124):
    g = _gen(seed)
    q = torch.randint(0, 256, (rows, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.randint(lo, hi, (rows, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    return q, s


def _check_product(a, sa, w, sw, out, K):
    A, W = ref.values(_np(a), _np(sa), K), ref.values(_np(w), _np(sw), K)
    want = A @ W.T
    mags = np.abs(A) @ np.abs(W).T
    tol = ref.sum_err(mags, K) * 2 + np.abs(want) * EPS[out.dtype] / 2 + TINY[out.dtype]
    # a partial sum is at most the sum of magnitudes: below 2^128 none leaves fp32's range, beyond it the fp32 sum may
    over = (mags >= 2.0 ** 128) & ~np.isfinite(_f64(out))
    bad = ~(np.abs(_f64(out) - want) <= tol) & ~over
    assert not bad.any(), (np.argwhere(bad)[:5], bad.sum())


SIZES = [(1, 1, 32), (1, 16, 64), (2, 130, 512), (16, 48, 544), (17, 33, 2048), (64, 300, 1056), (65, 129, 96),
         (128, 128, 256), (200, 257, 288), (333, 2050, 2080), (129, 1, 4096), (300, 40, 1024), (70, 64, 8192),
         (100, 70, 8224), (66, 40, 32768 + 32), (600, 1030, 416), (515, 2049, 992), (1500, 2050, 160), (1100, 2000, 1184),
         (33, 2100, 96), (20, 4200, 160), (64, 33000, 64), (5, 12400, 32), (100, 66000, 96), (40, 1100, 16416)]   # every kind of tile


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("odt", [torch.float32, torch.bfloat16])
def test_matmul(cuda, M, N, K, odt):
    from mi355moe import mxfp4
    a, sa = _mx(M, K, M + K)
    w, sw = _mx(N, K, N + 2 * K)
    _check_product(a, sa, w, sw, mxfp4.matmul(a, sa, w, sw, out_dtype=odt), K)


def test_matmul_largest_tiles(cuda):
    from mi355moe import mxfp4
    M, N, K = 4099, 3333, 1184
    a, sa = _mx(M, K, 1)
    w, sw = _mx(N, K, 2)
    _check_product(a, sa, w, sw, mxfp4.matmul(a, sa, w, sw, out_dtype=torch.float16), K)


def test_matmul_scale_extremes_and_nan_blocks(cuda):
    """Scales over the whole range, a NaN block in one row of each side: NaN in that row or column and nowhere else."""
    from mi355moe import mxfp4
    for M, K in ((5, 192), (100, 192), (5, 1024), (100, 1024)):
        a, sa = _mx(M, K, 7, 60, 190)
        w, sw = _mx(40, K, 8, 60, 190)
        sa[2, K // 32 - 1] = 255
        sw[11, 0] = 255
        out = _f64(mxfp4.matmul(a, sa, w, sw, out_dtype=torch.float32))
        nan = np.isnan(out)
        assert nan[2].all() and nan[:, 11].all() and nan.sum() == 40 + M - 1
        rows, cols = [i for i in range(M) if i != 2], [j for j in range(40) if j != 11]
        _check_product(a[rows], sa[rows], w[cols], sw[cols], torch.from_numpy(out[np.ix_(rows, cols)]).float(), K)


def test_matmul_out_strides_and_untouched_neighbours(cuda):
    from mi355moe import mxfp4
    for M, N, off in ((7, 50, 1), (90, 131, 3), (90, 128, 4)):
        a, sa = _mx(M, 320, 1)
        w, sw = _mx(N, 320, 2)
        buf = torch.full((M + 2, N + 9), 7.0, dtype=torch.bfloat16, device="cuda")
        view = buf[1:M + 1, off:off + N]
        assert mxfp4.matmul(a, sa, w, sw, out=view) is view
        assert torch.equal(view, mxfp4.matmul(a, sa, w, sw))
        keep = buf.clone()
        keep[1:M + 1, off:off + N] = 7.0
        assert (keep == 7.0).all()


def test_matmul_unaligned_views(cuda):
    from mi355moe import mxfp4
    a, sa = _mx(6, 160, 1)
    w, sw = _mx(20, 160, 2)
    want = mxfp4.matmul(a, sa, w, sw)

    def shifted(t):
        b = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        b[1:] = t.reshape(-1)
        return b[1:].reshape(t.shape)

    assert torch.equal(mxfp4.matmul(shifted(a), shifted(sa), shifted(w), shifted(sw)), want)
    wide = torch.cat([w, w], 1)
    assert torch.equal(mxfp4.matmul(a, sa, wide[:, :80], sw), want)


# ---------------------------------------------------------------------------------------------- routed experts


def _layer(n, H, I, seed):
    from mi355moe import mxfp4
    g = _gen(seed)
    w13 = torch.randn(n, 2 * I, H, generator=g, device="cuda") * (3.0 / H ** 0.5)
    w2 = torch.randn(n, H, I, generator=g, device="cuda") * (1.0 / I ** 0.5)
    return mxfp4.Mxfp4Experts.from_dense(w13, w2)


def _dense(ex):
    return ref.values(_np(ex.w13), _np(ex.w13_scale), ex.K), ref.values(_np(ex.w2), _np(ex.w2_scale), ex.N)


def _routing(T, n, topk, seed, bad=False):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(n)[:topk] for _ in range(T)]).astype(np.int64)
    if bad:
        ids[0, 0] = -1
        ids[T // 2, topk - 1] = n + 3
    w = rng.random((T, topk)).astype(np.float32) + 0.1
    return ids, w / w.sum(-1, keepdims=True) * 2.5


CASES = [(8, 512, 256, 40, 4, 10.0, torch.bfloat16), (16, 1024, 512, 33, 8, 0.0, torch.float16),
         (4, 32, 32, 1, 2, 10.0, torch.float32), (6, 544, 96, 70, 6, 1.0, torch.bfloat16),
         (3, 160, 1056, 5, 3, 2.0, torch.float32), (2, 288, 160, 150, 2, 10.0, torch.float16),
         (1, 2080, 64, 130, 1, 1.5, torch.bfloat16), (5, 256, 4160, 2, 1, 10.0, torch.bfloat16),
         # few pairs over many experts: no permutation
         (70, 288, 64, 8, 4, 1.0, torch.bfloat16), (40, 4160, 96, 2, 9, 10.0, torch.float16), (3, 160, 1056, 1, 3, 0.0, torch.float32)]


@pytest.mark.parametrize("n,H,I,T,topk,limit,dt", CASES)
def test_moe_forward(cuda, n, H, I, T, topk, limit, dt):
    from mi355moe import mxfp4
    ex = _layer(n, H, I, 11 + n)
    x = torch.randn(T, H, generator=_gen(T), device="cuda").to(dt)
    ids, w = _routing(T, n, topk, 13 + H, bad=topk > 1)
    out = mxfp4.moe_forward_ids(ex, x, torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda(), limit=limit)
    assert out.dtype == dt
    w13, w2 = _dense(ex)
    want, tol = ref.moe(_f64(x), w13, w2, ids, w.astype(np.float64), limit, EPS[dt])
    bad = np.abs(_f64(out) - want) > tol + TINY[dt]
    assert not bad.any(), (np.argwhere(bad)[:5], bad.sum())
    again = mxfp4.moe_forward_ids(ex, x, torch.from_numpy(ids).int().cuda(), torch.from_numpy(w).cuda(), limit=limit)
    assert torch.equal(out, again)


def test_moe_duplicate_ids_expert_map_strides_and_accumulate(cuda):
    from mi355moe import mxfp4
    n, H, I, T = 4, 256, 128, 21
    ex = _layer(n, H, I, 3)
    w13, w2 = _dense(ex)
    wide = torch.randn(T, H + 8, generator=_gen(9), device="cuda").bfloat16()
    x = wide[:, 5:5 + H]                                   # unaligned rows of an odd base
    gids = np.random.default_rng(1).integers(0, 9, (T, 3))
    gids[4] = 7                                            # the same expert three times
    emap = np.array([2, -1, 0, 3, -1, 1, -1, 2, 3])
    w = np.random.default_rng(2).random((T, 3)).astype(np.float32)
    local = emap[gids]
    for odt in (torch.float32, torch.bfloat16):
        want, tol = ref.moe(_f64(x), w13, w2, local, w.astype(np.float64), 10.0, EPS[odt])
        buf = torch.full((T + 1, H + 3), 3.0, dtype=odt, device="cuda")
        out = buf[:T, 1:1 + H]
        args = (ex, x, torch.from_numpy(gids).cuda(), torch.from_numpy(w).cuda())
        mxfp4.moe_forward_ids(*args, expert_map=torch.from_numpy(emap).cuda(), out=out)
        assert (np.abs(_f64(out) - want) <= tol + TINY[odt]).all()
        assert (buf[T] == 3.0).all() and (buf[:, 0] == 3.0).all() and (buf[:, 1 + H:] == 3.0).all()
        shared = torch.randn(T, H, generator=_gen(4), device="cuda").to(odt)
        base = _f64(shared)
        mxfp4.moe_forward_ids(*args, expert_map=torch.from_numpy(emap).cuda(), out=shared, accumulate=True)
        tol2 = tol + np.abs(base + want) * EPS[odt] / 2 + np.abs(base) * 2.0 ** -22
        assert (np.abs(_f64(shared) - (base + want)) <= tol2).all()


def test_moe_few_pairs_expert_map_and_accumulate(cuda):
    """Calls that take no permutation (few pairs over many experts): expert map, duplicate and foreign ids, int32 and int64
    ids, rows at odd addresses, fp16 weights and accumulation."""
    from mi355moe import mxfp4
    n, H, I, T, k = 48, 256, 128, 4, 5
    ex = _layer(n, H, I, 3)
    w13, w2 = _dense(ex)
    rng = np.random.default_rng(1)
    emap = np.where(rng.random(60) < 0.6, rng.integers(0, n, 60), -1)
    gids = rng.integers(0, 60, (T, k))
    gids[1] = np.flatnonzero(emap >= 0)[0]
    gids[2, :2] = (-1, 77)
    gids[3] = np.flatnonzero(emap < 0)[0]
    w = rng.random((T, k)).astype(np.float16)
    local = np.where((gids >= 0) & (gids < 60), emap[np.clip(gids, 0, 59)], -1)
    wide = torch.randn(T, H + 9, generator=_gen(9), device="cuda").bfloat16()
    for x in (wide[:, :H].contiguous(), wide[:, 3:3 + H]):
        want, tol = ref.moe(_f64(x), w13, w2, local, w.astype(np.float64), 10.0, 0.0)
        for it in (torch.int32, torch.int64):
            args = (ex, x, torch.from_numpy(gids).to("cuda", it), torch.from_numpy(w).cuda())
            buf = torch.full((T, H + 1), 2.0, dtype=torch.float32, device="cuda")
            base = _f64(buf[:, 1:])
            mxfp4.moe_forward_ids(*args, expert_map=torch.from_numpy(emap).cuda(), out=buf[:, 1:], accumulate=True)
            assert (np.abs(_f64(buf[:, 1:]) - (base + want)) <= tol + np.abs(base + want) * 2.0 ** -22 + 2.0 ** -21).all()
            assert (buf[:, 0] == 2.0).all() and (buf[3, 1:] == 2.0).all()
            out = mxfp4.moe_forward_ids(*args, expert_map=torch.from_numpy(emap).cuda())
            assert (np.abs(_f64(out) - want) <= tol + np.abs(want) * 2.0 ** -8 + TINY[torch.bfloat16]).all()


def test_moe_no_local_expert_writes_zero(cuda):
    from mi355moe import mxfp4
    ex = _layer(2, 64, 32, 3)
    x = torch.randn(3, 64, device="cuda").bfloat16()
    ids = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    out = torch.full((3, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    mxfp4.moe_forward_ids(ex, x, ids, torch.ones(3, 2, device="cuda"), out=out)
    assert (out == 0).all()


def test_moe_non_finite_rows_stay_apart(cuda):
    from mi355moe import mxfp4
    for T in (5, 300):
        ex = _layer(3, 256, 128, 3)
        x = torch.randn(T, 256, generator=_gen(1), device="cuda").bfloat16()
        ids, w = _routing(T, 3, 2, 5)
        ids, w = torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()
        clean = mxfp4.moe_forward_ids(ex, x, ids, w)
        x[1, 100], x[3, 7] = float("nan"), float("inf")
        out = mxfp4.moe_forward_ids(ex, x, ids, w)
        keep = [t for t in range(T) if t not in (1, 3)]
        assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
        assert torch.equal(out[keep], clean[keep])


def test_moe_functional_form_and_views(cuda):
    from mi355moe import fused_experts_mxfp4, mxfp4
    for H, I, T in ((160, 96, 6), (384, 128, 6), (384, 128, 90)):   # scales arranged in the call, and used as they are
        ex = _layer(4, H, I, 7)
        x = torch.randn(T, H, device="cuda").half()
        ids, w = _routing(T, 4, 2, 5)
        ids, w = torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()
        want = mxfp4.moe_forward_ids(ex, x, ids, w)
        assert torch.equal(fused_experts_mxfp4(x, ex.w13, ex.w2, w, ids, (ex.w13_scale, ex.w2_scale)), want)
    wide = torch.stack([ids, ids], 2)[..., 0]              # ids with a column stride
    assert torch.equal(mxfp4.moe_forward_ids(ex, x, wide, w.half().float()), mxfp4.moe_forward_ids(ex, x, ids, w.half()))


def test_arranged_scales(cuda):
    from mi355moe import mxfp4
    for n, rows, nb in ((1, 3, 1), (2, 64, 8), (3, 17, 21), (2, 5, 128)):
        s = torch.randint(0, 256, (n, rows, nb), generator=_gen(nb), device="cuda", dtype=torch.uint8)
        want = torch.nn.functional.pad(s, (0, -nb % 8), value=127).reshape(n, rows, -1, 8).transpose(1, 2)
        assert torch.equal(mxfp4._arranged(s), want)


def test_empty_calls(cuda):
    from mi355moe import fused_experts_mxfp4, mxfp4
    q, s = mxfp4.quant_rows(torch.empty(0, 64, device="cuda"))
    assert q.shape == (0, 32) and s.shape == (0, 2)
    assert mxfp4.dequant_rows(q, s).shape == (0, 64)
    w, sw = _mx(8, 64, 1)
    assert mxfp4.matmul(q, s, w, sw).shape == (0, 8)
    ex = _layer(2, 64, 32, 3)
    out = mxfp4.moe_forward_ids(ex, torch.empty(0, 64, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"),
                                torch.empty(0, 2, device="cuda"))
    assert out.shape == (0, 64)
    none = fused_experts_mxfp4(torch.empty(0, 64, device="cuda"), ex.w13, ex.w2, torch.empty(0, 2, device="cuda"),
                               torch.empty(0, 2, dtype=torch.int64, device="cuda"), (ex.w13_scale, ex.w2_scale))
    assert none.shape == (0, 64)


def test_two_streams_and_two_graphs(cuda):
    """Calls on two streams at once, and two captured graphs replayed side by side on two streams with eager calls in
    between, give what each gives alone: no scratch is shared."""
    from mi355moe import mxfp4
    ex = _layer(8, 512, 256, 5)
    calls = []
    for T in (9, 200):
        x = torch.randn(T, 512, generator=_gen(T), device="cuda").bfloat16()
        ids, w = _routing(T, 8, 4, T)
        calls.append((x, torch.from_numpy(ids).cuda(), torch.from_numpy(w).cuda()))
    a, sa = _mx(100, 4096, 3)
    w_, sw = _mx(130, 4096, 4)

    def work(i):
        return mxfp4.moe_forward_ids(ex, *calls[i]), mxfp4.matmul(a, sa, w_, sw), mxfp4.quant_rows(calls[i][0])[0]

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
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(i))
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
        eager = work(1)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, want[1]))
        for i in range(2):
            assert all(torch.equal(p, q) for p, q in zip(outs[i], want[i]))


def test_rows_beyond_32_bit_offsets(cuda):
    """Rows 2^32 bytes and more from the first one."""
    from mi355moe import mxfp4
    K = 128
    stride = (1 << 31) + 64                                # elements; 4 GiB a row in bf16
    buf = torch.empty(2 * stride + K, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, K), (stride, 1))
    x.copy_(_rows(3, K, torch.bfloat16, 2))
    q, s = mxfp4.quant_rows(x)
    qo, so = ref.quant_rows(_np(x.float()))
    assert np.array_equal(_np(q), qo) and np.array_equal(_np(s), so)
    ex = _layer(2, K, 64, 1)
    ids = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    w = torch.ones(3, 1, device="cuda")
    assert torch.equal(mxfp4.moe_forward_ids(ex, x, ids, w), mxfp4.moe_forward_ids(ex, x.contiguous(), ids, w))


def test_outputs_beyond_32_bit_offsets(cuda):
    """More than 2^31 output values: the last rows against the same rows on their own."""
    from mi355moe import mxfp4
    M, N, K = 1 << 20, 2064, 32
    a, sa = _mx(M, K, 1)
    w, sw = _mx(N, K, 2)
    out = mxfp4.matmul(a, sa, w, sw)
    for lo in (0, M // 2, M - 100):
        assert torch.equal(out[lo:lo + 100], mxfp4.matmul(a[lo:lo + 100], sa[lo:lo + 100], w, sw))
    q, s = mxfp4.quant_rows(out)
    back = mxfp4.dequant_rows(q, s, N)
    for lo in (0, M // 2, M - 100):
        q2, s2 = mxfp4.quant_rows(out[lo:lo + 100])
        assert torch.equal(q[lo:lo + 100], q2) and torch.equal(s[lo:lo + 100], s2)
        assert torch.equal(back[lo:lo + 100], mxfp4.dequant_rows(q2, s2, N))
