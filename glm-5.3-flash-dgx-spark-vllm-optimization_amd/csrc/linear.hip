// The dense product with its epilogue, and its gradients, on the 16-bit matrix cores.
//
//   z = x W^T + bias (fp32 sums);   out = act(z) + residual, rounded once
//   dz = dy act'(z) from the fp32 z that the forward pass keeps;   dx = dz W,   dW = dz^T x,   dbias = sum over rows of dz
//   (fp32 sums; dbias sums the unrounded dz, the products take it rounded once to the operand type, in fp16 times a power of
//   two that the call's largest value sets where the activation has a slope other than 0 and 1)
//
//   relu max(z, 0);   silu z s(z);   gelu z Phi(z), Phi the normal distribution's integral;   gelu_tanh z s(2 sqrt(2/pi) (z +
//   0.044715 z^3)), which is z (1 + tanh(half of that)) / 2;   s(v) = 1 / (1 + e^-v)
#include <algorithm>

#include "gemm_tile.cuh"
#include "rows.cuh"

namespace mi355moe {

// One product with its epilogue, as the kernels take it: out [M][N], out[m][n] = act(sum over k of P Q + bias) + res.
struct ProductArgs {
    const uint16_t* p;      // ROW: [N][ldp], COL: [K][ldp]
    const uint16_t* q;      // ROW: [M][ldq], COL: [K][ldq]
    int64_t ldp, ldq;       // elements
    int pcols, qcols;       // COL: how many of a row's values may be read (multiples of 8)
    int64_t M, K;
    int N;
    const void* bias;       // optional [N] of type bdt
    int bdt, act;
    const void* res;        // optional [M][res_stride]
    int64_t res_stride;
    float* z;               // optional [M][N]: before the activation
    const float* unscale;   // optional: a factor of the sums
    void* out;
    int64_t out_stride;
    int splits;             // parts of the contraction
    float* part;            // [splits][M][part_stride] (splits > 1)
    int64_t part_stride;
};
// What the gradient's own kernels take beside the call's arguments.
struct SlopeArgs {
    LinearArgs a;
    uint16_t* dz;           // optional [M][dz_stride]
    int64_t dz_stride;
    uint32_t* tops;
    int ntops;
    float* unscale;
    float* part;            // [row blocks][part_stride]
    int64_t part_stride;
};

template <int DT>
struct LinearKind {
    static constexpr int value = DT == DT_BF16 ? MM_BF16 : MM_F16;
};

// ------------------------------------------------------------------------------------------------ activations

__device__ __forceinline__ float sigmoid_rcp(float v) { return __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }
// Phi(z) from erfc(x) = t (a1 + t (a2 + ... + t a7)) e^(-x^2), t = 1 / (1 + 0.3625 x), x = |z| / sqrt(2). The coefficients (here
// halved) and 0.3625 are a minimax fit made for this: up to x = 9.6, where e^(-x^2) leaves fp32, within 2^-18 of erfc itself and
// within 4.2e-8 absolutely, so that the tail z Phi(z) at z << 0 keeps its own leading bits (in fp32: 8e-6 of itself at -12.5; a
// formula that is good to 1.5e-7 absolutely alone, with five terms, is off by 0.4 % at -6, a bf16 half step, and by 3.2 % at
// -12.5). The library's erfcf takes three times the instructions. e: e^(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    e = __expf(-0.5f * z * z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3625f * 0.70710678118654752f, fabsf(z), 1.0f));
    float p = __builtin_fmaf(0.5f * -0.1574683f, t, 0.5f * 0.5264033f);
    p = __builtin_fmaf(p, t, 0.5f * -0.30249074f);
    p = __builtin_fmaf(p, t, 0.5f * 0.391264f);
    p = __builtin_fmaf(p, t, 0.5f * 0.12326955f);
    p = __builtin_fmaf(p, t, 0.5f * 0.21518677f);
    p = __builtin_fmaf(p, t, 0.5f * 0.20383538f);
    const float half = p * t * e;
    return z < 0.0f ? half : 1.0f - half;
}
constexpr float GELU_A = 1.5957691216057308f;                        // 2 sqrt(2 / pi)

template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
    if (act == ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];       // (NaN stays)
    } else if (act == ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] *= sigmoid_rcp(v[j]);
    } else if (act == ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float e;
            v[j] *= normal_cdf(v[j], e);
        }
    } else if (act == ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] *= sigmoid_rcp(GELU_A * (v[j] + 0.044715f * v[j] * v[j] * v[j]));
    }
}
__device__ __forceinline__ float act_slope(int act, float z) {
    if (act == ACT_RELU) return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;     // (NaN stays)
    if (act == ACT_SILU) {
        const float s = sigmoid_rcp(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (act == ACT_GELU) {
        float e;
        const float c = normal_cdf(z, e);
        return __builtin_fmaf(z * 0.3989422804014327f, e, c);
    }
    if (act == ACT_GELU_TANH) {
        const float s = sigmoid_rcp(GELU_A * (z + 0.044715f * z * z * z));
        const float c = __builtin_amdgcn_fmed3f(z, -64.0f, 64.0f);    // (beyond, s is 0 or 1, and z^2 may not be a number)
        return s + z * s * (1.0f - s) * GELU_A * (1.0f + 3.0f * 0.044715f * c * c);
    }
    return 1.0f;
}

// Columns c .. of row m from their sums: bias (b: theirs), activation, residual (r: theirs) and the one rounding.
template <int DT>
__device__ __forceinline__ void product_out8(const ProductArgs& a, int64_t m, int c, float (&v)[8], const float (&b)[8], const Raw8<DT>& r8) {
    const int n = a.N - c;
    if (a.bias)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += b[j];
    if (a.z) store8<DT_F32>(a.z, (size_t)m * a.N + c, n, v);
    activate(a.act, v);
    if (a.res) {
        float r[8];
        r8.get(r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
    }
    store8<DT>(a.out, (size_t)m * a.out_stride + c, n, v);
}

// ------------------------------------------------------------------------------------------------ few rows

template <int DT>
__device__ __forceinline__ f32x4 linear_mma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (DT == DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// Chunk (eight values) i of a row of K values, what lies behind the row's end as zero.
__device__ __forceinline__ u32x4 row_chunk(const uint16_t* row, int i, int K) {
    Raw8<DT_BF16> v;                                                 // (the bits of either type)
    v.load(row, 8 * i, K - 8 * i);
    return v.w[0];
}

// grid (ceil(N / 16), ceil(M / 16)), eight waves: 16 weight rows as one 16-row MFMA operand, for 16 rows of x; any K, stride and
// address. Lane (c = lane % 16, g = lane / 16) holds the chunks g, 4 + g, 8 + g, 12 + g of weight row c and of row c of x, so
// that a load takes 64 bytes in a row (128 of the contraction a wave step, in the same order on both sides); the contraction is
// cut over the waves, whose sums join in LDS in wave order. Bound: the weights' way through a CU, 7 us for 4096 of the contraction (M = 1,
// 4096 from 1024: 8.4 MB in 4.0 us, of which 2.6 are the launch and the chain of two loads); sixteen waves spilled.
constexpr int FEW_WAVES = 8;
template <int DT>
__global__ __launch_bounds__(64 * FEW_WAVES) void linear_few_kernel(ProductArgs a) {
    constexpr int W = FEW_WAVES;
    __shared__ __align__(16) float red[W][256];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = blockIdx.x * 16;
    const int64_t m0 = (int64_t)blockIdx.y * 16;
    const int rows = (int)min((int64_t)16, a.M - m0);
    const int K = (int)a.K, chunks = (K + 7) >> 3;
    const uint16_t* w = a.p + (size_t)min(n0 + c, a.N - 1) * a.ldp;
    const uint16_t* x = a.q + (size_t)(m0 + min(c, rows - 1)) * a.ldq;
    f32x4 acc = {};
    for (int b0 = wv * 16; b0 < chunks; b0 += 16 * W) {
        u32x4 p[4], q[4];
        if ((b0 + 16) * 8 <= K) {                                  // (uniform)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const rows_u32x4*>(w + 8 * (b0 + g + 4 * i));
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const rows_u32x4*>(x + 8 * (b0 + g + 4 * i));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = row_chunk(w, b0 + g + 4 * i, K);
                q[i] = row_chunk(x, b0 + g + 4 * i, K);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = linear_mma16<DT>(p[i], q[i], acc);
    }
    *reinterpret_cast<f32x4*>(&red[wv][lane * 4]) = acc;
    __syncthreads();
    if (tid >= 256) return;
    const int m = tid >> 4, n = tid & 15, col = n0 + n;
    if (m >= rows || col >= a.N) return;
    float v[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < W; ++i) v[0] += red[i][((n >> 2) * 16 + m) * 4 + (n & 3)];
    if (a.bias) v[0] += any_value(a.bias, a.bdt, col);
    if (a.z) a.z[(size_t)(m0 + m) * a.N + col] = v[0];
    activate(a.act, v);
    if (a.res) v[0] += row_value<DT>(a.res, (size_t)(m0 + m) * a.res_stride + col);
    store_any(a.out, DT, (size_t)(m0 + m) * a.out_stride + col, v[0]);
}

// ------------------------------------------------------------------------------------------------ tiles

// What a wave does with its sums (32 TP columns from c0, 32 TQ rows from r0): they pass through LDS in fp32 (`mine`, 32 rows of 128 TP
// bytes of the wave's own), 32 rows at a time, so that a lane ends up with eight columns of a row: bias, residual and output
// are whole 16-byte accesses in whole lines, and the residual is added before the one rounding; it is requested before the sums
// go to LDS.
template <int DT, int TP, int TQ>
__device__ __forceinline__ void linear_finish(const ProductArgs& a, const f32x16 (&acc)[TP][TQ], unsigned char* mine, int lane, int64_t r0, int c0) {
    constexpr int UNITS = 8 * TP, CH = UNITS / 2;                    // 16-byte units and 8-column chunks of a wave's row
    const int64_t m1 = r0 + lane / CH;
    const int c = c0 + 8 * (lane % CH), n = a.N - c;
    const int m = lane & 31, h = lane >> 5;
    float b[8] = {};
    if (a.bias && a.splits == 1) load8_any(a.bias, a.bdt, c, n, b);
    const float f = a.unscale ? *a.unscale : 1.0f;
    float* part = a.splits > 1 ? a.part + (size_t)blockIdx.y * a.M * a.part_stride : nullptr;
#pragma unroll
    for (int j = 0; j < TQ; ++j) {
        Raw8<DT> r8[CH / 2];
        if (a.res && !part)                                          // (uniform)
#pragma unroll
            for (int s = 0; s < CH / 2; ++s) {
                const int64_t mm = m1 + 32 * j + s * (64 / CH);
                r8[s].load(a.res, (size_t)mm * a.res_stride + c, mm < a.M ? n : 0);
            }
        unsigned char* row = mine + m * (16 * UNITS);
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x16& v = acc[i][j];
                *reinterpret_cast<f32x4*>(row + (((8 * i + 2 * r + h) ^ (m & (UNITS - 1))) << 4)) =
                    f32x4{v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]};
            }
        asm volatile("" ::: "memory");                               // (a wave's LDS accesses are performed in order)
#pragma unroll
        for (int s = 0; s < CH / 2; ++s) {
            const int rr = s * (64 / CH) + lane / CH, u = 2 * (lane % CH), x = rr & (UNITS - 1);
            const unsigned char* from = mine + rr * (16 * UNITS);
            const f32x4 lo = *reinterpret_cast<const f32x4*>(from + ((u ^ x) << 4)), hi = *reinterpret_cast<const f32x4*>(from + (((u + 1) ^ x) << 4));
            float v[8] = {lo[0] * f, lo[1] * f, lo[2] * f, lo[3] * f, hi[0] * f, hi[1] * f, hi[2] * f, hi[3] * f};
            const int64_t mm = m1 + 32 * j + s * (64 / CH);
            if (mm >= a.M || n <= 0) continue;
            if (part) store8<DT_F32>(part, (size_t)mm * a.part_stride + c, 8, v);
            else product_out8<DT>(a, mm, c, v, b, r8[s]);
        }
        asm volatile("" ::: "memory");
    }
}

// A workgroup's BP columns x BQ rows, the contraction in a.splits parts (grid y). Bound: the matrix cores
// while the contraction runs and memory at its ends, which do not overlap where one workgroup has the CU (M = 8192, 4096 from 2048, bf16:
// the product with relu 123 us, 1.1 PFLOP/s; + residual 146, + gelu_tanh 154, + z, 134 MB of fp32, 184 to 200; its gradients dx 124
// to 150, dw 131 to 150). Gained nothing there: the residual requested before the product (206, for its registers), z in whole
// lines by a second pass over LDS or marked as not read again (202, 210).
template <int DT, int PL, int QL, int BP, int BQ, int WP, int WQ, int ST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void linear_kernel(ProductArgs a, int nt, int mt) {
    using G = GemmTile<LinearKind<DT>::value, PL, QL, BP, BQ, WP, WQ, ST>;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int2 tile = tile_order(blockIdx.x, nt, mt);
    const int n0 = tile.x * BP;
    const int64_t m0 = (int64_t)tile.y * BQ;
    const int stages = (int)((a.K + SB / 2 - 1) / (SB / 2)), per = (stages + a.splits - 1) / a.splits;
    const int kb0 = blockIdx.y * per, kb1 = min(stages, kb0 + per);
    const uint32_t ldp = 2u * (uint32_t)a.ldp, ldq = 2u * (uint32_t)a.ldq;
    const int pl = min(BP, a.N - n0) - 1, ql = (int)min((int64_t)BQ, a.M - m0) - 1;
    G t;
    if constexpr (PL == LAY_ROW)
        t.p.init_row(uniform_ptr(a.p + (size_t)n0 * a.ldp + (size_t)kb0 * (SB / 2)), wv, lane, [&](int r) { return (uint32_t)min(r, pl) * ldp; });
    else t.p.init_col(uniform_ptr(a.p + (size_t)kb0 * (SB / 2) * a.ldp + n0), wv, lane, ldp, min(BP, a.pcols - n0));
    if constexpr (QL == LAY_ROW)
        t.q.init_row(uniform_ptr(a.q + (size_t)m0 * a.ldq + (size_t)kb0 * (SB / 2)), wv, lane, [&](int r) { return (uint32_t)min(r, ql) * ldq; });
    else t.q.init_col(uniform_ptr(a.q + (size_t)kb0 * (SB / 2) * a.ldq + m0), wv, lane, ldq, (int)min((int64_t)BQ, a.qcols - m0));
    const int left = kb1 == stages ? (int)(a.K % (SB / 2)) : 0;      // (ROW operands hold whole chunks of eight, zeros in the last)
    if (kb0 < kb1) t.run(lds, kb0, kb1, PL == LAY_ROW ? (left + 7) >> 3 : left, QL == LAY_ROW ? (left + 7) >> 3 : left, ldp, ldq);
    else
#pragma unroll
        for (int i = 0; i < G::TP; ++i)
#pragma unroll
            for (int j = 0; j < G::TQ; ++j) t.acc[i][j] = f32x16{};

    static_assert(G::NW * 32 * 128 * G::TP <= G::LDS, "the stages hold the waves' rows");
    __syncthreads();                                                 // no wave reads a stage any more
    linear_finish<DT, G::TP, G::TQ>(a, t.acc, lds + wv * (32 * 128 * G::TP), lane, m0 + (wv / WP) * (BQ / WQ), n0 + (wv % WP) * (BP / WP));
}

// 64 columns x 64 rows of operands whose rows lie at any address (K no multiple of 8: the loads to LDS above take whole 16 bytes), so
// that they need no copies: four stages of 64 are on their way to registers, from which a stage goes to one of two LDS buffers,
// its 16-byte chunks exchanged by the row (lanes of one chunk then read different banks). The last, part stage is requested first.
// Bound: the loads' way, which addresses off 16 bytes double (0.35 us a stage and workgroup of a CU, however many it has). us with the
// copies and the tiles above / so: M = 130, 2051 from 1027 21.8 / 11.1, 333 15.4 / 10.3, 700 20.2 / 16.3, 1791 26.0 / 31.1; 1024 from
// 4099, 130 20.6 / 13.5 (in parts), 1791 41 / 48.
constexpr int ANY_AHEAD = 4;
template <int DT>
__global__ __launch_bounds__(256, 1) void linear_any_kernel(ProductArgs a, int nt, int mt) {
    __shared__ __align__(16) unsigned char lds[2][2][64 * 128];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int2 tile = tile_order(blockIdx.x, nt, mt);
    const int n0 = tile.x * 64, K = (int)a.K;
    const int64_t m0 = (int64_t)tile.y * 64;
    const int stages = (K + 63) / 64, per = (stages + a.splits - 1) / a.splits;
    const int kb0 = blockIdx.y * per, kb1 = min(min(stages, kb0 + per), K / 64);       // (whole stages)
    const bool tail = kb0 < stages && kb0 + per >= stages && K % 64;
    const int row = threadIdx.x >> 2, c4 = threadIdx.x & 3;          // what this thread loads: chunks c4 and c4 + 4 of a row of each
    const uint16_t* p = a.p + (size_t)min(n0 + row, a.N - 1) * a.ldp;
    const uint16_t* q = a.q + (size_t)min(m0 + row, a.M - 1) * a.ldq;
    const int to0 = row * 128 + ((c4 ^ ((row >> 1) & 7)) << 4), to1 = row * 128 + (((c4 + 4) ^ ((row >> 1) & 7)) << 4);
    u32x4 last[4], set[ANY_AHEAD][4];
    if (tail)
#pragma unroll
        for (int i = 0; i < 4; ++i) last[i] = row_chunk(i < 2 ? p : q, K / 64 * 8 + c4 + 4 * (i & 1), K);
    auto load = [&](u32x4 (&v)[4], int kb) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const rows_u32x4*>((i < 2 ? p : q) + kb * 64 + 8 * (c4 + 4 * (i & 1)));
    };
    f32x16 acc[1][1] = {};
    int cur = 0;
    // one stage from registers, into which stage `next` is requested
    auto step = [&](auto more, u32x4 (&v)[4], int next) {
        unsigned char(*buf)[64 * 128] = lds[cur];
        *reinterpret_cast<u32x4*>(buf[0] + to0) = v[0];
        *reinterpret_cast<u32x4*>(buf[0] + to1) = v[1];
        *reinterpret_cast<u32x4*>(buf[1] + to0) = v[2];
        *reinterpret_cast<u32x4*>(buf[1] + to1) = v[3];
        if constexpr (more) load(v, next);
        __syncthreads();                                             // (the buffer before it is free: all have passed its reads)
        const int pr = 32 * (wv & 1) + (lane & 31), qr = 32 * (wv >> 1) + (lane & 31), h = lane >> 5;
        u32x4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = *reinterpret_cast<const u32x4*>(buf[0] + pr * 128 + (((2 * i + h) ^ ((pr >> 1) & 7)) << 4));
            y[i] = *reinterpret_cast<const u32x4*>(buf[1] + qr * 128 + (((2 * i + h) ^ ((qr >> 1) & 7)) << 4));
        }
        SCHED_FENCE();                                               // (all reads requested before the first multiplication)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[0][0] = mma16(std::integral_constant<int, LinearKind<DT>::value>{}, x[i], y[i], acc[0][0]);
        cur ^= 1;
    };
    if (kb0 < kb1) {
#pragma unroll
        for (int i = 0; i < ANY_AHEAD; ++i) load(set[i], min(kb0 + i, kb1 - 1));
        for (int kb = kb0;;) {                                       // (uniform; beyond the last stage the loads repeat it)
#pragma unroll
            for (int i = 0; i < ANY_AHEAD; ++i) {
                step(std::true_type{}, set[i], min(kb + ANY_AHEAD, kb1 - 1));
                if (++kb == kb1) break;
            }
            if (kb == kb1) break;
        }
    }
    if (tail) step(std::false_type{}, last, 0);
    __syncthreads();                                                 // no wave reads a stage any more
    linear_finish<DT, 1, 1>(a, acc, &lds[0][0][0] + wv * (32 * 128), lane, m0 + 32 * (wv >> 1), n0 + 32 * (wv & 1));
}

// out from the sums of the contraction's parts [splits][M][part_stride], added in order: eight columns a thread. Bound: memory
// (M = 1791, N = 1024 from two parts: 18 MB in 4.7 us).
template <int DT>
__global__ __launch_bounds__(256) void linear_join_kernel(ProductArgs a) {
    const int per = (a.N + 7) / 8;
    const int64_t items = a.M * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / per;
        const int c = (int)(i - m * per) * 8;
        float v[8] = {}, b[8] = {};
        Raw8<DT> r8;
        if (a.res) r8.load(a.res, (size_t)m * a.res_stride + c, a.N - c);
        if (a.bias) load8_any(a.bias, a.bdt, c, a.N - c, b);
        for (int s = 0; s < a.splits; ++s) {
            float p[8];
            load8<DT_F32>(a.part, ((size_t)s * a.M + m) * a.part_stride + c, 8, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += p[j];
        }
        product_out8<DT>(a, m, c, v, b, r8);
    }
}

// ------------------------------------------------------------------------------------------------ copies

// Up to two matrices of `cols` columns copied to rows of whole 16 bytes ([rows][wide], the columns behind `cols` zero), as the
// tiles read them.
struct PadArgs {
    const uint16_t* src[2];
    int64_t stride[2], rows[2];
    uint16_t* dst[2];
    int cols, wide;
};
// A wave a row. Bound: latency and rows that begin at odd addresses (333 and 2051 rows of 1027: 10 MB in 7.2 us).
__global__ __launch_bounds__(256) void linear_pad_kernel(PadArgs a) {
    const int lane = threadIdx.x & 63;
    int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r >= a.rows[0] + a.rows[1]) return;
    const int k = r >= a.rows[0];
    r -= k ? a.rows[0] : 0;
    const uint16_t* src = (k ? a.src[1] : a.src[0]) + (size_t)r * (k ? a.stride[1] : a.stride[0]);
    uint16_t* dst = (k ? a.dst[1] : a.dst[0]) + (size_t)r * a.wide;
    for (int c0 = lane * 8; c0 < a.wide; c0 += 2048) {
        Raw8<DT_BF16> v[4];                                          // (on their way together)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i].load(src, c0 + 512 * i, a.cols - c0 - 512 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c0 + 512 * i < a.wide) *reinterpret_cast<u32x4*>(dst + c0 + 512 * i) = v[i].w[0];
    }
}

// ------------------------------------------------------------------------------------------------ gradient

constexpr int DZ_ROWS = 64;                                          // rows of a workgroup of linear_dz_kernel

template <int DT>
__device__ __forceinline__ void slope8(const LinearArgs& a, int64_t m, int c, float (&d)[8]) {
    const int n = a.N - c;
    Raw8<DT> d8;
    d8.load(a.dy, (size_t)m * a.dy_stride + c, n);
    if (a.act != ACT_NONE) {
        Raw8<DT_F32> z8;
        z8.load(a.z, (size_t)m * a.N + c, n);
        float z[8];
        z8.get(z);
        d8.get(d);
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] *= act_slope(a.act, z[j]);
    } else d8.get(d);
}

// The largest finite magnitude of dz, as fp32 bits, of each workgroup's share (fp16 only: dz = dy act'(z) can lie among fp16's
// subnormals, or beyond its range, where the sums over it are ordinary fp16 numbers). Bound: HBM, a pass over dy and z that the
// next kernel makes again (8192 x 4096: 201 MB in 41 to 47 us, 4.6 TB/s; the next one then takes what it takes in bf16).
template <int DT>
__global__ __launch_bounds__(256) void linear_top_kernel(SlopeArgs g) {
    const LinearArgs& a = g.a;
    __shared__ uint32_t red[4];
    const int per = (a.N + 7) / 8;
    const int64_t items = a.M * per;
    uint32_t top = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / per;
        float d[8];
        slope8<DT>(a, m, (int)(i - m * per) * 8, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = __builtin_bit_cast(uint32_t, d[j]) & 0x7FFFFFFFu;
            top = max(top, b < 0x7F800000u ? b : 0u);
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) g.tops[blockIdx.x] = max(max(red[0], red[1]), max(red[2], red[3]));
}
// k of the 2^k that brings the largest of `n` maxima into [2^14, 2^15) (0 where all are zero): every thread gets it.
__device__ __forceinline__ int linear_shift(const uint32_t* tops, int n) {
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

// dz of 256 columns and DZ_ROWS rows: 32 threads across the columns, eight values each, eight down the rows. dz [M][dz_stride] in
// the operand type (its columns behind N zero), where g.dz is set; the sums of the unrounded dz over the workgroup's rows to part
// [grid x][part_stride] where that is set. A kernel of its own, because two products read dz and the tiles take 16-bit operands
// from memory as they lie. This rounding of dz is the one place where a gradient holds less than fp32 before its own: dx and dW err
// by 0.0023 of their norm in bf16 where their own rounding alone is 0.0017. The rest of dz as a second term would bring them there,
// for both products again: 280 of 500 us at 8192 x 4096 from 2048. Bound: HBM (8192 x 4096: 268 MB in 47 to 52 us, 5.3 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void linear_dz_kernel(SlopeArgs g) {
    const LinearArgs& a = g.a;
    __shared__ __align__(16) float red[8][256];
    float f = 1.0f;
    if constexpr (DT == DT_F16)
        if (g.ntops) {                                               // (uniform)
            const int k = linear_shift(g.tops, g.ntops);
            f = __builtin_bit_cast(float, (uint32_t)(127 + k) << 23);
            if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *g.unscale = __builtin_bit_cast(float, (uint32_t)(127 - k) << 23);
        }
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int c = blockIdx.y * 256 + tx * 8;
    const int64_t m0 = (int64_t)blockIdx.x * DZ_ROWS, m1 = min(a.M, m0 + DZ_ROWS);
    float sum[8] = {};
    if (c < a.N)
        for (int64_t m = m0 + ty; m < m1; m += 8) {
            float d[8];
            slope8<DT>(a, m, c, d);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += d[j];
            if (g.dz) {
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = c + j < a.N ? d[j] * f : 0.0f;
                store8<DT>(g.dz, (size_t)m * g.dz_stride + c, 8, d);
            }
        }
    if (!a.dbias) return;                                            // (uniform)
    store8<DT_F32>(red[ty], tx * 8, 8, sum);
    __syncthreads();
    const int col = blockIdx.y * 256 + threadIdx.x;
    if (col >= a.N) return;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
    g.part[(size_t)blockIdx.x * g.part_stride + col] = s;
}
// dbias: the parts' sums in order, 64 columns a workgroup, the parts cut over its sixteen waves. Bound: latency (128 parts of 4096
// columns: 5 us).
__global__ __launch_bounds__(1024) void linear_dbias_kernel(SlopeArgs g, int parts) {
    const LinearArgs& a = g.a;
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const int per = (parts + 15) / 16, g0 = wv * per, g1 = min(parts, g0 + per);
    float v = 0.0f;
    if (c < a.N) {
#pragma unroll 8
        for (int i = g0; i < g1; ++i) v += g.part[(size_t)i * g.part_stride + c];
    }
    red[wv][lane] = v;
    __syncthreads();
    if (wv || c >= a.N) return;
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += red[w][lane];
    store_any(a.dbias, a.bdt, c, v);
}

// ------------------------------------------------------------------------------------------------ launchers

static unsigned linear_grid(int64_t items) { return (unsigned)std::min<int64_t>((items + 255) / 256, 8192); }
static int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }

// Which kernel, and in how many parts of the contraction, by an estimate of each one's time in us. Measured per stage of 64 (one
// workgroup a CU; 64 x 64 also two): 64 x 64 0.30 (0.49 for two), 128 x 128 0.54, 256 x 128 0.91, 256 x 256 1.56, and per tile for
// its ends 0.9 (2.8), 6, 11, 24: small tiles bring more workgroups, large ones read less. Parts pay a second launch and their
// fp32 sums' way through memory. us measured, 64 / 128 / 256 x 128 / 256 (N = 4096 from 1024): M = 256 8.7 / 13.0 / 19.9 / 35, 768 19.7
// / 16.5 / 24.3 / 44, 2048 43.7 / 32.6 / 27.4 / 46, 8192 - / 127 / 106 / 101; N = 1024 from 4096, M = 128 19.3, in four parts 11.9.
struct ProductPlan {
    int tile, splits;
    double us;
};
static double tiles_us(int tile, int64_t tiles, int64_t stages) {
    if (tile == TILE_ANY) return 3.5 + (double)((tiles + 255) / 256) * (0.35 * stages + 1.3);
    if (tile == TILE_64) {
        const double one = 0.30 * stages + 0.9, two = 0.49 * stages + 2.8;
        const int64_t rest = tiles % 512;
        return 3.0 + (tiles / 512) * two + (rest == 0 ? 0.0 : rest <= 256 ? one : two);
    }
    const int64_t rounds = (tiles + 255) / 256;
    return 3.0 + rounds * (tile == TILE_128_DEEP ? 0.54 * stages + 6.0 : tile == TILE_256_128 ? 0.91 * stages + 11.0 : 1.56 * stages + 24.0);
}
static double join_us(int s, int64_t M, int64_t N) { return 2.0 + s * (double)(M * N) * 8.0 / 6e6; }
// any: the operands lie at any address, so linear_any_kernel, or copies of them for the others.
static ProductPlan plan_product(int64_t M, int64_t N, int64_t K, bool any = false) {
    auto count = [&](int64_t p, int64_t q) { return ((N + p - 1) / p) * ((M + q - 1) / q); };
    const int64_t stages = (K + 63) / 64;
    ProductPlan best{TILE_64, 1, 1e30};
    const struct {
        int tile;
        int64_t tiles;
    } kinds[] = {{TILE_64, count(64, 64)}, {TILE_128_DEEP, count(128, 128)}, {TILE_256_128, count(256, 128)}, {TILE_256, count(256, 256)}};
    for (const auto& k : kinds)
        for (int s = 1; s <= 16; s *= 2) {
            if (s > 1 && (k.tile == TILE_256 || k.tile == TILE_256_128 || stages / s < 8 || k.tiles * s > 512)) break;
            double us = tiles_us(k.tile, k.tiles * s, (stages + s - 1) / s);
            if (s > 1) us += join_us(s, M, N);
            if (us < best.us) best = {k.tile, s, us};
        }
    if (any) {
        best.us += 4.0 + (double)((M + N) * K) * 4.0 / 4e6;         // (the copies)
        for (int s = 1; s <= 16 && (s == 1 || (stages / s >= 8 && count(64, 64) * s <= 512)); s *= 2) {
            const double us = tiles_us(TILE_ANY, count(64, 64) * s, (stages + s - 1) / s) + (s > 1 ? join_us(s, M, N) : 0.0);
            if (us < best.us) best = {TILE_ANY, s, us};
        }
    }
    return best;
}
// Few rows stream the weights. The streaming kernel takes about 3 us and, for every 256 workgroups of 16 columns and 16 rows, what
// one CU takes to read its rows of both operands (7 us for 4096 of the contraction). us streamed / by tiles: 1024 from 4096, M = 64
// 9.6 / 11.3, 96 16.5 / 11.6; 4096 from 1024, 16 4.6 / 7.3, 32 6.4 / 8.1, 64 9.9 / 8.2; 4096 from 4096, 16 10.7 / 12.8, 32 17 /
// 13.2. Rows at odd addresses (K no multiple of 8) take 1.7 times as long to read (us streamed / by linear_any_kernel, M = 65: 515 from
// 131 4.4 / 6.0, 2051 from 1027 14.4 / 10.0).
static bool linear_streams(int64_t M, int64_t N, int64_t K) {
    const int64_t wgs = (M + 15) / 16 * ((N + 15) / 16);
    const double few = 2.6 + (double)((wgs + 255) / 256) * (0.5 + 1.75e-3 * (double)K) * (K % 8 ? 1.7 : 1.0);
    return M <= 4096 && few <= plan_product(M, N, K, K % 8 != 0).us;
}
static int64_t part_bytes(int64_t M, int64_t N, int64_t K, bool any = false) {
    const int s = plan_product(M, N, K, any).splits;
    return s > 1 ? 4 * s * M * up8(N) : 0;
}

template <int DT, int PL, int QL, int BP, int BQ, int WP, int WQ, int ST>
static int run_tiles(const ProductArgs& a, hipStream_t st) {
    using G = GemmTile<LinearKind<DT>::value, PL, QL, BP, BQ, WP, WQ, ST>;
    if (!allow_lds<linear_kernel<DT, PL, QL, BP, BQ, WP, WQ, ST>>(G::LDS)) return -1;
    const int nt = (a.N + BP - 1) / BP, mt = (int)((a.M + BQ - 1) / BQ);
    hipLaunchKernelGGL((linear_kernel<DT, PL, QL, BP, BQ, WP, WQ, ST>), dim3(nt * mt, a.splits), dim3(G::THREADS), G::LDS, st, a, nt, mt);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int DT>
static int run_any(const ProductArgs& a, hipStream_t st) {
    const int nt = (a.N + 63) / 64, mt = (int)((a.M + 63) / 64);
    hipLaunchKernelGGL(linear_any_kernel<DT>, dim3(nt * mt, a.splits), dim3(256), 0, st, a, nt, mt);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
template <int DT, int PL, int QL>
static int run_product(ProductArgs a, const ProductPlan& p, float* part, hipStream_t st) {
    a.splits = p.splits;
    a.part = part;
    a.part_stride = up8(a.N);
    const int r = p.tile == TILE_ANY        ? run_any<DT>(a, st)
                  : p.tile == TILE_256      ? run_tiles<DT, PL, QL, 256, 256, 2, 4, 2>(a, st)
                  : p.tile == TILE_256_128  ? run_tiles<DT, PL, QL, 256, 128, 2, 4, 3>(a, st)
                  : p.tile == TILE_128_DEEP ? run_tiles<DT, PL, QL, 128, 128, 2, 4, 4>(a, st)
                                            : run_tiles<DT, PL, QL, 64, 64, 2, 2, 4>(a, st);
    if (r || a.splits == 1) return r;
    hipLaunchKernelGGL(linear_join_kernel<DT>, dim3(linear_grid(a.M * ((a.N + 7) / 8))), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
static int run_pad(const PadArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(linear_pad_kernel, dim3((unsigned)((a.rows[0] + a.rows[1] + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// Where the parts of a workspace begin, in bytes (256-byte steps); -1: not there.
struct LinearSpace {
    int64_t x = -1, w = -1, part = -1, dz = -1, tops = -1, bytes = 0;
    int64_t take(int64_t n) {
        const int64_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
};
static LinearSpace forward_space(int64_t M, int64_t N, int64_t K) {
    LinearSpace s;
    if (M == 0 || linear_streams(M, N, K)) return s;
    if (K % 8 && plan_product(M, N, K, true).tile != TILE_ANY) s.x = s.take(M * up8(K) * 2), s.w = s.take(N * up8(K) * 2);
    if (const int64_t n = part_bytes(M, N, K, K % 8 != 0)) s.part = s.take(n);
    return s;
}
int64_t linear_forward_bytes(int64_t M, int64_t N, int64_t K) { return forward_space(M, N, K).bytes; }

template <int DT>
static int linear_forward(LinearArgs a, char* ws, hipStream_t st) {
    ProductArgs g{};
    g.M = a.M, g.N = a.N, g.K = a.K;
    g.p = a.w, g.ldp = a.w_stride, g.q = a.x, g.ldq = a.x_stride;
    g.bias = a.bias, g.bdt = a.bdt, g.act = a.act, g.res = a.res, g.res_stride = a.res_stride;
    g.z = a.z, g.out = a.out, g.out_stride = a.out_stride;
    if (linear_streams(a.M, a.N, a.K)) {
        const dim3 grid((a.N + 15) / 16, (unsigned)((a.M + 15) / 16));
        hipLaunchKernelGGL(linear_few_kernel<DT>, grid, dim3(64 * FEW_WAVES), 0, st, g);
        return hipGetLastError() == hipSuccess ? 0 : -1;
    }
    const LinearSpace s = forward_space(a.M, a.N, a.K);
    if (s.x >= 0) {
        uint16_t *x = reinterpret_cast<uint16_t*>(ws + s.x), *w = reinterpret_cast<uint16_t*>(ws + s.w);
        const int64_t K8 = up8(a.K);
        if (int r = run_pad(PadArgs{{a.x, a.w}, {a.x_stride, a.w_stride}, {a.M, a.N}, {x, w}, a.K, (int)K8}, st)) return r;
        g.p = w, g.q = x, g.ldp = g.ldq = K8;
    }
    return run_product<DT, LAY_ROW, LAY_ROW>(g, plan_product(a.M, a.N, a.K, a.K % 8 != 0), s.part >= 0 ? reinterpret_cast<float*>(ws + s.part) : nullptr, st);
}
int launch_linear(const LinearArgs& a, void* ws, hipStream_t st) {
    return a.dt == DT_BF16 ? linear_forward<DT_BF16>(a, static_cast<char*>(ws), st) : linear_forward<DT_F16>(a, static_cast<char*>(ws), st);
}

// What a gradient's call puts in its workspace: dz unless dy serves as it is, its largest values (tops), the copies and parts of
// the products that are asked for, the sums of dbias.
struct LinearUse {
    bool dz, tops, dx, dw, dbias;
};
// Whether the products can take dy as it is (its rows then lie as an operand's do: aligned).
static bool dz_is_dy(int act, int64_t N, bool aligned) { return act == ACT_NONE && N % 8 == 0 && aligned; }
static LinearUse linear_use(int dt, int act, int64_t N, bool aligned, bool dx, bool dw, bool dbias) {
    const bool dz = (dx || dw) && !dz_is_dy(act, N, aligned);
    return {dz, dz && dt == DT_F16 && act != ACT_NONE && act != ACT_RELU, dx, dw, dbias};
}
static LinearSpace backward_space(int64_t M, int64_t N, int64_t K, const LinearUse& u) {
    LinearSpace s;
    if (u.dz) s.dz = s.take(M * up8(N) * 2);
    if (u.tops) s.tops = s.take(4 * (LINEAR_TOPS + 1));
    if (K % 8 && u.dw) s.x = s.take(M * up8(K) * 2);
    if (K % 8 && u.dx) s.w = s.take(N * up8(K) * 2);
    const int64_t part = std::max({u.dx ? part_bytes(M, K, N) : 0, u.dw ? part_bytes(N, K, M) : 0,
                                   u.dbias ? 4 * ((M + DZ_ROWS - 1) / DZ_ROWS) * up8(N) : 0});
    if (part) s.part = s.take(part);
    return s;
}
int64_t linear_backward_bytes(int64_t M, int64_t N, int64_t K) { return backward_space(M, N, K, {true, true, true, true, true}).bytes; }
// A workspace of up to 1 MB for all gradients is laid out for all of them whatever is asked for: one size for a shape, and nothing
// to gain (an allocator's own step is of that order).
static LinearSpace call_space(int64_t M, int64_t N, int64_t K, const LinearUse& u) {
    const LinearSpace all = backward_space(M, N, K, {true, true, true, true, true});
    return all.bytes <= 1 << 20 ? all : backward_space(M, N, K, u);
}
int64_t linear_backward_call_bytes(int dt, int act, int64_t M, int64_t N, int64_t K, bool aligned, bool dx, bool dw, bool dbias) {
    return call_space(M, N, K, linear_use(dt, act, N, aligned, dx, dw, dbias)).bytes;
}

template <int DT>
static int linear_backward(const LinearArgs& a, char* ws, hipStream_t st) {
    const LinearUse use = linear_use(a.dt, a.act, a.N, linear_dy_aligned(a.dy, a.dy_stride), a.dx, a.dw, a.dbias);
    const LinearSpace s = call_space(a.M, a.N, a.K, use);
    const int64_t N8 = up8(a.N), K8 = up8(a.K);
    auto at = [&](int64_t o) { return o < 0 ? nullptr : reinterpret_cast<uint16_t*>(ws + o); };
    float* part = reinterpret_cast<float*>(at(s.part));
    SlopeArgs g{};
    g.a = a;
    g.part = part;
    g.part_stride = N8;
    g.dz = use.dz ? at(s.dz) : nullptr;
    g.dz_stride = N8;
    if constexpr (DT == DT_F16)
        if (use.tops) {
            g.tops = reinterpret_cast<uint32_t*>(at(s.tops));
            g.unscale = reinterpret_cast<float*>(g.tops + LINEAR_TOPS);
            g.ntops = (int)std::min<int64_t>((a.M * ((a.N + 7) / 8) + 255) / 256, LINEAR_TOPS);
            hipLaunchKernelGGL(linear_top_kernel<DT>, dim3(g.ntops), dim3(256), 0, st, g);
            if (hipGetLastError() != hipSuccess) return -1;
        }
    if (g.dz || a.dbias) {
        const int parts = (int)((a.M + DZ_ROWS - 1) / DZ_ROWS);
        hipLaunchKernelGGL(linear_dz_kernel<DT>, dim3(parts, (a.N + 255) / 256), dim3(256), 0, st, g);
        if (hipGetLastError() != hipSuccess) return -1;
        if (a.dbias) {
            hipLaunchKernelGGL(linear_dbias_kernel, dim3((a.N + 63) / 64), dim3(1024), 0, st, g, parts);
            if (hipGetLastError() != hipSuccess) return -1;
        }
    }
    ProductArgs p{};
    p.q = g.dz ? g.dz : static_cast<const uint16_t*>(a.dy);
    p.ldq = g.dz ? N8 : a.dy_stride;
    p.qcols = (int)N8;
    p.pcols = (int)K8;
    p.N = a.K;
    p.out_stride = a.K;
    p.unscale = g.ntops ? g.unscale : nullptr;
    const uint16_t *x = a.x, *w = a.w;
    int64_t ldx = a.x_stride, ldw = a.w_stride;
    if (a.K % 8 && (a.dx || a.dw)) {
        const PadArgs pad{{a.x, a.w}, {ldx, ldw}, {a.dw ? a.M : 0, a.dx ? a.N : 0}, {at(s.x), at(s.w)}, a.K, (int)K8};
        if (int r = run_pad(pad, st)) return r;
        x = at(s.x), w = at(s.w), ldx = ldw = K8;
    }
    if (a.dx) {
        p.p = w, p.ldp = ldw, p.M = a.M, p.K = a.N, p.out = a.dx;
        if (int r = run_product<DT, LAY_COL, LAY_ROW>(p, plan_product(p.M, p.N, p.K), part, st)) return r;
    }
    if (a.dw) {
        p.p = x, p.ldp = ldx, p.M = a.N, p.K = a.M, p.out = a.dw;
        if (int r = run_product<DT, LAY_COL, LAY_COL>(p, plan_product(p.M, p.N, p.K), part, st)) return r;
    }
    return 0;
}
int launch_linear_backward(const LinearArgs& a, void* ws, hipStream_t st) {
    return a.dt == DT_BF16 ? linear_backward<DT_BF16>(a, static_cast<char*>(ws), st) : linear_backward<DT_F16>(a, static_cast<char*>(ws), st);
}

}  // namespace mi355moe
