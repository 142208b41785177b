// The gated feed-forward block of a layer's shared expert, and its gradient, on the 16-bit matrix cores.
//
//   [g | u] = x W13^T (fp32 sums);  h = silu(min(g, L)) clamp(u, -L, L)  (the limit iff L != 0), rounded once
//   dg = dh u' s (1 + g' (1 - s)) [g <= L],  du = dh g' s [|u| <= L],  s = sigmoid(g'), from the fp32 g and u that the
//   forward pass keeps;  dx = [dg | du] W13,  dW13 = [dg | du]^T x  (fp32 sums; [dg | du] is rounded once to the operand
//   type, which the matrix cores take, in fp16 times a power of two that the call's largest value sets)
//
// Forward multiplies two operands whose contraction is contiguous; dx has one, and dW13 both, with the contraction as the
// row index (the tiles' COL layout).
#include <algorithm>

#include "gemm_tile.cuh"
#include "mi355moe_internal.h"

namespace mi355moe {

template <int DT>
struct KindOf {
    static constexpr int value = DT == DT_BF16 ? MM_BF16 : MM_F16;
};
template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (DT == DT_BF16) return pack_bf16x2(lo, hi);
    else return h_as_u16((_Float16)lo) | (h_as_u16((_Float16)hi) << 16);
}
template <int DT>
__device__ __forceinline__ float value16(uint32_t b) {
    if constexpr (DT == DT_BF16) return bf16_to_f32((uint16_t)b);
    else return (float)u16_as_h(b & 0xFFFFu);
}

// ------------------------------------------------------------------------------------------------ forward, few rows

template <int DT>
__device__ __forceinline__ f32x4 few_mma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// grid (N / 8, ceil(T / 16)), 1024 threads: 8 gate and the same 8 up columns as one 16-row MFMA operand, for 16 tokens.
// Lane (c = lane % 16, g = lane / 16) holds the chunks g, 4 + g, 8 + g, 12 + g of weight row c and of token c, so that a load
// takes 64 bytes in a row (128 of the contraction a wave step, in the same order on both sides); the contraction is cut over
// the sixteen waves, whose sums join in LDS in wave order. Bound: the latency of the two or three loads a wave makes and the
// join (one token, 4096 -> 1024, 16.8 MB of weights by 128 workgroups, two rounds of loads each: 7.1 us, 2.4 TB/s; 4096 -> 4096: 13.4 us, 5.0 TB/s); more than one group
// of tokens reads the weights and the tokens through L2 again, 16.8 us at 512 workgroups, all that the card holds at once.
// Two or four groups a workgroup, which read the weights once: 13.7 us for 32 tokens (9.9 by two workgroups), 21 for 64 (16.8).
template <int DT>
__global__ __launch_bounds__(1024) void gated_few_kernel(GatedArgs a) {
    __shared__ __align__(16) float red[16][256];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 8;
    const int64_t m0 = (int64_t)blockIdx.y * 16;
    const int rows = (int)min((int64_t)16, a.T - m0);
    const int chunks = a.K >> 3;                                     // 16-byte chunks of a row
    const u32x4* w = reinterpret_cast<const u32x4*>(a.w13 + ((size_t)(c < 8 ? 0 : a.N) + n0 + (c & 7)) * a.K);
    const u32x4* x = reinterpret_cast<const u32x4*>(a.x + (size_t)(m0 + min(c, rows - 1)) * a.x_stride);
    f32x4 acc = {};
    for (int b0 = wv * 16; b0 < chunks; b0 += 256) {
        const int b = b0 + g;
        u32x4 wv4[4], xv4[4];
        if (b0 + 16 <= chunks) {                                     // (uniform)
#pragma unroll
            for (int i = 0; i < 4; ++i) wv4[i] = w[b + 4 * i];
#pragma unroll
            for (int i = 0; i < 4; ++i) xv4[i] = x[b + 4 * i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool ok = b + 4 * i < chunks;
                wv4[i] = w[min(b + 4 * i, chunks - 1)];
                xv4[i] = x[min(b + 4 * i, chunks - 1)];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    wv4[i][j] = ok ? wv4[i][j] : 0u;
                    xv4[i][j] = ok ? xv4[i][j] : 0u;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = few_mma16<DT>(wv4[i], xv4[i], acc);
    }
    *reinterpret_cast<f32x4*>(&red[wv][lane * 4]) = acc;
    __syncthreads();
    if (tid >= 128) return;
    const int m = tid >> 3, n = tid & 7;
    if (m >= rows) return;
    const int ag = (((n >> 2) << 4) + m) * 4 + (n & 3), au = ag + 128;   // (up: n + 8, two lane groups on)
    float gs = 0.f, us = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        gs += red[i][ag];
        us += red[i][au];
    }
    const size_t t = (size_t)(m0 + m);
    a.h[t * a.h_stride + n0 + n] = (uint16_t)pack16<DT>(swiglu(gs, us, a.limit), 0.f);
    if (a.gu) {
        a.gu[t * 2 * a.N + n0 + n] = gs;
        a.gu[t * 2 * a.N + a.N + n0 + n] = us;
    }
}

// ------------------------------------------------------------------------------------------------ forward, tiles

// Workgroup tiles of BP / 2 columns x BQ tokens; a wave's P rows are its gate columns, then the same up columns, so the SwiGLU
// is local to a lane. 8192 tokens, 4096 -> 2048, 275 GFLOP with g and u kept: 267 us, 1.03 PFLOP/s (without them 235 us, 1.17; a
// library product alone takes 218): the matrix cores, busy in half of the cycles at 2.0 GHz, then 134 MB of fp32 sums. 1791 tokens
// -> 1024: 36 us, 0.83 PFLOP/s, 224 tiles on 256 CUs at 0.57 us a stage, of which the matrix cores work half and LDS 38 %, and
// waves wait 39 %, next to nothing of it for LDS: the stage's loads and its barrier. Few tokens: the latency of a stage, 0.33 us
// whatever the tile (4096 -> 1024, 700 tokens: 24 us).
template <int DT, int BP, int BQ, int WP, int WQ, int ST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void gated_kernel(GatedArgs a, int nt, int mt) {
    using G = GemmTile<KindOf<DT>::value, LAY_ROW, LAY_ROW, BP, BQ, WP, WQ, ST>;
    static_assert(G::TP % 2 == 0, "");
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int HALF = BP / WP / 2;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int2 tile = tile_order(blockIdx.x, nt, mt);
    const int n0 = tile.x * (BP / 2);
    const int64_t m0 = (int64_t)tile.y * BQ;
    const int ql = (int)min((int64_t)BQ, a.T - m0) - 1;
    const uint32_t wp = 2u * a.K, xp = 2u * (uint32_t)a.x_stride;
    G t;
    t.p.init_row(a.w13, wv, lane, [&](int r) {
        const int w = r / (2 * HALF), i = r % (2 * HALF);
        return (uint32_t)(min(n0 + w * HALF + (i % HALF), a.N - 1) + (i < HALF ? 0 : a.N)) * wp;
    });
    t.q.init_row(uniform_ptr(a.x + (size_t)m0 * a.x_stride), wv, lane, [&](int r) { return (uint32_t)min(r, ql) * xp; });
    const int tail = a.K % (SB / 2) / 8;
    t.run(lds, 0, (a.K + SB / 2 - 1) / (SB / 2), tail, tail, 0, 0);
    const int p0 = (wv % WP) * HALF, q0 = (wv / WP) * (BQ / WQ);
    constexpr int TN = G::TP / 2;
    const int64_t m1 = m0 + q0, rows = a.T - m1;
    const int n1 = n0 + p0, cols = a.N - n1;
    auto exists = [&](int r) { return r < rows; };
    if (a.gu) {                                                      // (uniform) g and u before the limit
#pragma unroll
        for (int half = 0; half < 2; ++half)
            t.template store_rows<TN>(lds, a.gu + (size_t)m1 * 2 * a.N + half * a.N + n1, 2 * (int64_t)a.N, cols, exists,
                                      [&](int i, int j, int r) {
                                          const f32x16& v = t.acc[half * TN + i][j];
                                          return f32x4{v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]};
                                      });
    }
    t.template store_rows<TN>(lds, a.h + (size_t)m1 * a.h_stride + n1, a.h_stride, cols, exists, [&](int i, int j, int r) {
        float h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = swiglu(t.acc[i][j][4 * r + k], t.acc[TN + i][j][4 * r + k], a.limit);
        return pack4(DT, h[0], h[1], h[2], h[3]);
    });
}

// h (and gu) from the sums of the contraction's parts [splits][T][2N], added in order: eight columns a thread. Bound: a launch's
// latency and memory (the parts come mostly from cache).
template <int DT>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedArgs a, int splits) {
    const int per = a.N / 8;
    const int64_t items = a.T * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per;
        const int c = (int)(i - t * per) * 8;
        const float* p = a.part + (size_t)t * 2 * a.N + c;
        f32x4 g[2] = {}, u[2] = {};
        for (int s = 0; s < splits; ++s, p += (size_t)a.T * 2 * a.N) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                g[k] += reinterpret_cast<const f32x4*>(p)[k];
                u[k] += reinterpret_cast<const f32x4*>(p + a.N)[k];
            }
        }
        u32x4 h;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            h[k] = pack16<DT>(swiglu(g[k >> 1][2 * (k & 1)], u[k >> 1][2 * (k & 1)], a.limit),
                              swiglu(g[k >> 1][2 * (k & 1) + 1], u[k >> 1][2 * (k & 1) + 1], a.limit));
        *reinterpret_cast<u32x4*>(a.h + (size_t)t * a.h_stride + c) = h;
        if (a.gu) {
            f32x4* o = reinterpret_cast<f32x4*>(a.gu + (size_t)t * 2 * a.N + c);
            o[0] = g[0], o[1] = g[1];
            o = reinterpret_cast<f32x4*>(a.gu + (size_t)t * 2 * a.N + a.N + c);
            o[0] = u[0], o[1] = u[1];
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward

// dg and du of eight columns of token t, in fp32.
template <int DT>
__device__ __forceinline__ void gate_grads(const GatedArgs& a, int64_t t, int c, float (&dg)[8], float (&du)[8]) {
    const float L = a.limit;
    const f32x4* gp = reinterpret_cast<const f32x4*>(a.gu + (size_t)t * 2 * a.N + c);
    const f32x4* up = reinterpret_cast<const f32x4*>(a.gu + (size_t)t * 2 * a.N + a.N + c);
    const u32x4 dv = *reinterpret_cast<const u32x4*>(a.dh + (size_t)t * a.dh_stride + c);
    const f32x4 g4[2] = {gp[0], gp[1]}, u4[2] = {up[0], up[1]};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float dh = value16<DT>(dv[j >> 1] >> (16 * (j & 1)));
        float g = g4[j >> 2][j & 3], u = u4[j >> 2][j & 3];
        const bool gout = L != 0.0f && g > L, uout = L != 0.0f && fabsf(u) > L;
        if (L != 0.0f) {
            g = gout ? L : g;
            u = uout ? (u > 0.f ? L : -L) : u;
        }
        const float s = __fdiv_rn(1.0f, 1.0f + __expf(-g));
        dg[j] = gout ? 0.0f : dh * u * s * (1.0f + g * (1.0f - s));
        du[j] = uout ? 0.0f : dh * g * s;
    }
}

// The largest finite magnitude of d, as fp32 bits, of each workgroup's share. fp16 only: at dh = 60000 and the layer's limit d
// reaches 660000, and where dh is small d lies among fp16's subnormals, while the sums over it are ordinary fp16 numbers; d is
// therefore held times a power of two that goes by this maximum. Bound: memory and the exponentials; 8192 x 2048, 168 MB: 44 us,
// 3.8 TB/s (of 590 for both gradients); 64 x 1024: 3.6 us.
template <int DT>
__global__ __launch_bounds__(256) void gated_top_kernel(GatedArgs a) {
    __shared__ uint32_t red[4];
    const int per = a.N / 8;
    const int64_t items = a.T * per;
    uint32_t top = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per;
        float d[2][8];
        gate_grads<DT>(a, t, (int)(i - t * per) * 8, d[0], d[1]);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t b = __builtin_bit_cast(uint32_t, d[j >> 3][j & 7]) & 0x7FFFFFFFu;
            top = max(top, b < 0x7F800000u ? b : 0u);
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) a.tops[blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
}

// 2^k that brings the largest of `n` maxima into [2^14, 2^15) (k between -113 and 120, 0 where all are zero): every thread of the
// workgroup gets it. An exact factor: d keeps its bits, apart from what it would lose at the ends of fp16's range.
__device__ __forceinline__ int gated_shift(const uint32_t* tops, int n) {
    __shared__ uint32_t red[4];
    uint32_t top = 0;
    for (int i = threadIdx.x; i < n; i += 256) top = max(top, tops[i]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
    return top ? min(14 - ((int)(top >> 23) - 127), 120) : 0;
}
__device__ __forceinline__ float power_of_two(int k) { return __builtin_bit_cast(float, (uint32_t)(127 + k) << 23); }

// d = [dg | du], eight columns a thread. Bound: memory; 8192 x 2048, 235 MB: 35 us, 6.7 TB/s (part of it from cache). Rounded
// once to the operand type, which the matrix cores take; unrounded, the two products would be fp32 ones, at a tenth of the rate
// (the gradients' error against float64 grows from 0.0017 to 0.0024 of their norm in bf16, their own last rounding's share 0.0017).
// fp16: times 2^k by the maxima of gated_top_kernel, and 2^-k left for the products.
template <int DT>
__global__ __launch_bounds__(256) void gated_d_kernel(GatedArgs a) {
    const int per = a.N / 8;
    const int64_t items = a.T * per;
    float f = 1.0f;
    if constexpr (DT == DT_F16) {
        const int k = gated_shift(a.tops, a.ntops);
        f = power_of_two(k);
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.unscale = power_of_two(-k);
    }
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / per;
        const int c = (int)(i - t * per) * 8;
        float dg[8], du[8];
        gate_grads<DT>(a, t, c, dg, du);
        u32x4 og, ou;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            og[k] = pack16<DT>(dg[2 * k] * f, dg[2 * k + 1] * f);
            ou[k] = pack16<DT>(du[2 * k] * f, du[2 * k + 1] * f);
        }
        *reinterpret_cast<u32x4*>(a.d + (size_t)t * 2 * a.N + c) = og;
        *reinterpret_cast<u32x4*>(a.d + (size_t)t * 2 * a.N + a.N + c) = ou;
    }
}

struct Gemm16Args {
    const uint16_t* p;      // ROW: [N][ldp], COL: [C][ldp]
    const uint16_t* q;      // ROW: [M][ldq], COL: [C][ldq]
    int64_t ldp, ldq;       // elements
    int64_t M;
    int N;
    int64_t C;              // contraction
    void* out;
    int64_t out_stride;
    int splits;
    float* part;
    const float* unscale;   // fp16: the factor of the sums (nullptr: none)
};

// out[m][n] = sum over k of P Q, dtype DT, or fp32 partials of the contraction's splits (grid y). Bound: the matrix cores, busy
// in 60 and 64 % of the cycles at 1.8 GHz (memory-bound kernels run at 2.2); 8192 tokens, 4096 -> 2048, 275 GFLOP each: dx (8192 x
// 4096 from 4096) 235 us, dw (4096 x 4096 from 8192) 230, 1.17 and 1.19 PFLOP/s (library products of these sizes and layouts: 238
// and 256). Of few tiles (dx below 2000 tokens): a stage's latency, 0.6 us on the small tiles.
template <int DT, int PL, int QL, int BP, int BQ, int WP, int WQ, int ST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void gemm16_kernel(Gemm16Args a, int nt, int mt) {
    using G = GemmTile<KindOf<DT>::value, PL, QL, BP, BQ, WP, WQ, ST>;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int2 tile = tile_order(blockIdx.x, nt, mt);
    const int n0 = tile.x * BP;
    const int64_t m0 = (int64_t)tile.y * BQ;
    const int stages = (int)((a.C + SB / 2 - 1) / (SB / 2)), per = (stages + a.splits - 1) / a.splits;
    const int kb0 = blockIdx.y * per, kb1 = min(stages, kb0 + per);
    const uint32_t ldp = 2u * (uint32_t)a.ldp, ldq = 2u * (uint32_t)a.ldq;
    const int pl = min(BP, a.N - n0), ql = (int)min((int64_t)BQ, a.M - m0);
    G t;
    if constexpr (PL == LAY_ROW)
        t.p.init_row(uniform_ptr(a.p + (size_t)n0 * a.ldp + (size_t)kb0 * (SB / 2)), wv, lane, [&](int r) { return (uint32_t)min(r, pl - 1) * ldp; });
    else t.p.init_col(uniform_ptr(a.p + (size_t)kb0 * (SB / 2) * a.ldp + n0), wv, lane, ldp, pl);
    if constexpr (QL == LAY_ROW)
        t.q.init_row(uniform_ptr(a.q + (size_t)m0 * a.ldq + (size_t)kb0 * (SB / 2)), wv, lane, [&](int r) { return (uint32_t)min(r, ql - 1) * ldq; });
    else t.q.init_col(uniform_ptr(a.q + (size_t)kb0 * (SB / 2) * a.ldq + m0), wv, lane, ldq, ql);
    const int left = kb1 == stages ? (int)(a.C % (SB / 2)) : 0;
    if (kb0 < kb1) t.run(lds, kb0, kb1, PL == LAY_ROW ? left >> 3 : left, QL == LAY_ROW ? left >> 3 : left, ldp, ldq);
    else
#pragma unroll
        for (int i = 0; i < G::TP; ++i)
#pragma unroll
            for (int j = 0; j < G::TQ; ++j) t.acc[i][j] = f32x16{};
    if constexpr (DT == DT_F16)
        if (a.unscale) {                                             // (uniform)
            const float f = *a.unscale;
#pragma unroll
            for (int i = 0; i < G::TP; ++i)
#pragma unroll
                for (int j = 0; j < G::TQ; ++j) t.acc[i][j] *= f;
        }
    const int p0 = (wv % WP) * (BP / WP), q0 = (wv / WP) * (BQ / WQ);
    if (a.splits == 1) {                                             // (uniform)
        const int64_t rows = a.M - m0 - q0;
        t.template store_rows<G::TP>(lds, static_cast<uint16_t*>(a.out) + (size_t)(m0 + q0) * a.out_stride + n0 + p0, a.out_stride,
                                     a.N - n0 - p0, [&](int r) { return r < rows; }, [&](int i, int j, int r) {
                                         return pack4(DT, t.acc[i][j][4 * r], t.acc[i][j][4 * r + 1], t.acc[i][j][4 * r + 2],
                                                      t.acc[i][j][4 * r + 3]);
                                     });
        return;
    }
    float* part = a.part + (size_t)blockIdx.y * a.M * a.N;
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
        const int64_t m = m0 + q0 + 32 * j + (lane & 31);
        if (m >= a.M) continue;
#pragma unroll
        for (int i = 0; i < G::TP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + p0 + 32 * i + 8 * r + 4 * (lane >> 5);
                if (n < a.N)                                         // (N % 8 == 0)
                    *reinterpret_cast<f32x4*>(part + (size_t)m * a.N + n) =
                        f32x4{t.acc[i][j][4 * r], t.acc[i][j][4 * r + 1], t.acc[i][j][4 * r + 2], t.acc[i][j][4 * r + 3]};
            }
    }
}

// ------------------------------------------------------------------------------------------------ launchers

// Parts of the contraction for few 64 x 64 tiles: at least 16 stages each, of at least 48 (a stage takes 0.33 us, the join and its
// launch 5). us whole / in parts: 4096 -> 1024, 200 tokens (4 parts) 23.8 / 15.8; 8192 -> 512, 200 (4) 42.5 / 15.5; 4096 ->
// 2048, 128 (2) 23.5 / 15.0; 2048 -> 768, 200 (2) 13.5 / 15.0. Two parts also where that makes two workgroups a CU, which wait
// for their stages by turns: 4096 -> 1024, 512 23.7 / 19.9; 5120 -> 1536, 256 28.1 / 22.6; 4096 -> 2048, 300 23.8 / 23.3 (four or
// eight instead of two or four to that end: 8192 -> 512, 200 tokens 15.0 / 16.4).
static int gated_parts(int64_t T, int64_t K, int64_t N) {
    const int64_t tiles = (2 * N + 63) / 64 * ((T + 63) / 64), stages = (K + 63) / 64;
    int s = 1;
    while (stages >= 48 && tiles * s * 2 <= (s == 1 ? 512 : 256) && stages / (s * 2) >= 16) s *= 2;
    return s;
}
// The forward streams the weights for one group of 16 tokens, and for more while their workgroups are at most three a CU, or, where
// the contraction would be cut, two of 4096 values. us streamed / by tiles, cold weights: 4096 -> 1024, T = 16 9.7 / 26, 64
// 16.8 / 30, 96 23.5 / 29 (in parts 15), 128 30.5 / 29; 4096 -> 4096, 16 18 / 28, 32 31.7 / 29.5; 4096 -> 12288, 1 34 / 44, 16
// 50 / 45; 2048 -> 768, 128 13.1 / 16.6; 8192 -> 512, 64 16.6 / 53 (in parts 15.5), 100 31 / 53 (in parts 15.5). What so simple a
// rule leaves by these figures: 5 us at 12288 columns and 16 tokens, 1 at 8192 -> 512 and 64.
static bool gated_streams(int64_t T, int64_t K, int64_t N) {
    const int64_t wgs = (T + 15) / 16 * (N / 8);
    return T <= 16 || (wgs <= 768 && (wgs * K <= 512 * 4096 || gated_parts(T, K, N) == 1));
}
static int gated_splits(int64_t T, int64_t K, int64_t N) { return gated_streams(T, K, N) ? 1 : gated_parts(T, K, N); }
int64_t gated_forward_floats(int64_t T, int64_t K, int64_t N) {
    const int s = T > 0 ? gated_splits(T, K, N) : 1;
    return s > 1 ? s * T * 2 * N : 0;
}

struct Gemm16Plan {
    int tile, splits;
};
// By the rule of plan_mx_matmul. us by kind 256 / 128 / 128 deep / 64, dx of 4096 columns from 2048: T = 128 42 / 29 / 20.7 /
// 20.4, 512 46 / 32 / 24.0 / 22.5 (512 tiles of 64: the deep one is taken), 1791 51 / 41.8 / 47.7 / 61.7, 4096 71 / 83 / 95 / 120.
// A long contraction of few tiles (128 x 512 x 8192): 36 us, in 4 parts 21.
static Gemm16Plan plan_gemm16(int64_t M, int64_t N, int64_t C) {
    Gemm16Plan p{TILE_256, 1};
    auto tiles = [&](int64_t b) { return ((N + b - 1) / b) * ((M + b - 1) / b); };
    const int64_t t64 = tiles(64), stages = (C + 63) / 64;
    if (t64 <= 256) {
        p.tile = TILE_64;
        while (t64 * p.splits * 2 <= 256 && stages / (p.splits * 2) >= 24) p.splits *= 2;
    } else if (tiles(128) <= 256) p.tile = TILE_128_DEEP;
    else if (tiles(256) < 192) p.tile = TILE_128;
    return p;
}

template <int DT, int PL, int QL, int BP, int BQ, int WP, int WQ, int ST>
static int run_gemm16(const Gemm16Args& a, hipStream_t st) {
    using G = GemmTile<KindOf<DT>::value, PL, QL, BP, BQ, WP, WQ, ST>;
    if (!allow_lds<gemm16_kernel<DT, PL, QL, BP, BQ, WP, WQ, ST>>(G::LDS)) return -1;
    const int nt = (a.N + BP - 1) / BP, mt = (int)((a.M + BQ - 1) / BQ);
    hipLaunchKernelGGL((gemm16_kernel<DT, PL, QL, BP, BQ, WP, WQ, ST>), dim3(nt * mt, a.splits), dim3(G::THREADS), G::LDS, st, a, nt, mt);
    return 0;
}
template <int DT, int PL, int QL>
static int gemm16(Gemm16Args a, hipStream_t st) {
    const Gemm16Plan p = plan_gemm16(a.M, a.N, a.C);
    a.splits = p.splits;
    const int r = p.tile == TILE_256        ? run_gemm16<DT, PL, QL, 256, 256, 2, 4, 2>(a, st)
                  : p.tile == TILE_128      ? run_gemm16<DT, PL, QL, 128, 128, 2, 2, 2>(a, st)
                  : p.tile == TILE_128_DEEP ? run_gemm16<DT, PL, QL, 128, 128, 2, 4, 4>(a, st)
                                            : run_gemm16<DT, PL, QL, 64, 64, 2, 2, 4>(a, st);
    if (r) return r;
    if (hipGetLastError() != hipSuccess) return -1;
    if (p.splits > 1) return launch_join(a.part, p.splits, a.M, a.N, a.out, DT, a.out_stride, st);
    return 0;
}

int64_t gated_part_floats(int64_t T, int64_t K, int64_t N) {
    const Gemm16Plan px = plan_gemm16(T, K, 2 * N), pw = plan_gemm16(2 * N, K, T);
    int64_t f = 0;
    if (px.splits > 1) f = std::max(f, px.splits * T * K);
    if (pw.splits > 1) f = std::max(f, pw.splits * 2 * N * K);
    return f;
}

template <int DT, int BP, int BQ, int WP, int WQ, int ST>
static int run_gated(const GatedArgs& a, hipStream_t st) {
    using G = GemmTile<KindOf<DT>::value, LAY_ROW, LAY_ROW, BP, BQ, WP, WQ, ST>;
    if (!allow_lds<gated_kernel<DT, BP, BQ, WP, WQ, ST>>(G::LDS)) return -1;
    const int nt = (a.N + BP / 2 - 1) / (BP / 2), mt = (int)((a.T + BQ - 1) / BQ);
    hipLaunchKernelGGL((gated_kernel<DT, BP, BQ, WP, WQ, ST>), dim3(nt * mt), dim3(G::THREADS), G::LDS, st, a, nt, mt);
    return 0;
}

template <int DT>
static int gated_forward(const GatedArgs& a, hipStream_t st) {
    if (gated_streams(a.T, a.K, a.N)) {
        hipLaunchKernelGGL(gated_few_kernel<DT>, dim3(a.N / 8, (unsigned)((a.T + 15) / 16)), dim3(1024), 0, st, a);
    } else if (const int splits = gated_splits(a.T, a.K, a.N); splits > 1) {
        Gemm16Args g{};
        g.p = a.w13, g.ldp = a.K, g.q = a.x, g.ldq = a.x_stride;
        g.M = a.T, g.N = 2 * a.N, g.C = a.K, g.part = a.part, g.splits = splits;
        if (int r = run_gemm16<DT, LAY_ROW, LAY_ROW, 64, 64, 2, 2, 4>(g, st)) return r;
        if (hipGetLastError() != hipSuccess) return -1;
        const int64_t items = a.T * (a.N / 8);
        hipLaunchKernelGGL(gated_join_kernel<DT>, dim3((unsigned)std::min<int64_t>((items + 255) / 256, 8192)), dim3(256), 0, st, a, splits);
    } else {
        // tiles of n columns (and as many gate as up rows of W13) x b tokens, by the rule of plan_mx_matmul. us by kind 256 /
        // 128 / 128 deep / 64 (4096 -> 1024): T = 128 72 / 35 / 28 / 23, 512 85 / 49 / 29 / 23, 1791 87 / 52 / 36 / 50, 4096 95 /
        // 75 / 85 / 108; 8192 (2048 columns) 235 / 272 / 312 / 395
        auto tiles = [&](int64_t n, int64_t b) { return ((a.N + n - 1) / n) * ((a.T + b - 1) / b); };
        const int r = tiles(64, 64) <= 256    ? run_gated<DT, 128, 64, 2, 2, 4>(a, st)
                      : tiles(64, 128) <= 256 ? run_gated<DT, 128, 128, 2, 4, 4>(a, st)
                      : tiles(128, 256) < 192 ? run_gated<DT, 128, 128, 2, 2, 2>(a, st)
                                              : run_gated<DT, 256, 256, 2, 4, 2>(a, st);
        if (r) return r;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_gated_forward(const GatedArgs& a, hipStream_t st) {
    return a.dt == DT_BF16 ? gated_forward<DT_BF16>(a, st) : gated_forward<DT_F16>(a, st);
}

template <int DT>
static int gated_backward(GatedArgs a, hipStream_t st) {
    const int64_t items = a.T * (a.N / 8);
    if constexpr (DT == DT_F16) {
        a.ntops = (int)std::min<int64_t>((items + 255) / 256, GATED_TOPS);
        hipLaunchKernelGGL(gated_top_kernel<DT>, dim3(a.ntops), dim3(256), 0, st, a);
        if (hipGetLastError() != hipSuccess) return -1;
    }
    hipLaunchKernelGGL(gated_d_kernel<DT>, dim3((unsigned)std::min<int64_t>((items + 255) / 256, 8192)), dim3(256), 0, st, a);
    if (hipGetLastError() != hipSuccess) return -1;
    const float* unscale = DT == DT_F16 ? a.unscale : nullptr;
    if (a.dx) {
        Gemm16Args g{};
        g.unscale = unscale;
        g.p = a.w13, g.ldp = a.K, g.q = a.d, g.ldq = 2 * a.N;
        g.M = a.T, g.N = a.K, g.C = 2 * a.N, g.out = a.dx, g.out_stride = a.K, g.part = a.part;
        if (int r = gemm16<DT, LAY_COL, LAY_ROW>(g, st)) return r;
    }
    if (a.dw) {
        Gemm16Args g{};
        g.unscale = unscale;
        g.p = a.x, g.ldp = a.x_stride, g.q = a.d, g.ldq = 2 * a.N;
        g.M = 2 * a.N, g.N = a.K, g.C = a.T, g.out = a.dw, g.out_stride = a.K, g.part = a.part;
        if (int r = gemm16<DT, LAY_COL, LAY_COL>(g, st)) return r;
    }
    return 0;
}
int launch_gated_backward(const GatedArgs& a, hipStream_t st) {
    return a.dt == DT_BF16 ? gated_backward<DT_BF16>(a, st) : gated_backward<DT_F16>(a, st);
}

}  // namespace mi355moe
