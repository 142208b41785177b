// Microscaled 4-bit floating point (OCP MXFP4): e2m1 elements, element 2i of a row in the low four bits of byte i, and
// one e8m0 scale (2^(code - 127), 255 = NaN) per 32 consecutive elements of a row.
//
//   quant    per block: E = the exponent field of max|v|, s = max(E - 2, 0), q = e2m1(v 2^(127 - s)), to nearest even,
//            saturating at 6 (a block's largest element lies in [4, 8) after scaling); a block that holds an infinity or
//            a NaN gets s = 255 and reads back as NaN
//   product  out[m][n] = sum over blocks of 2^(sa + sw - 254) (sum of the block's 32 products), on the scaled matrix
//            instructions: the products are exact (multiples of 1/4 up to 36), and against float64 their sums of 128 came
//            out within 3e-8 of the sum of magnitudes, whatever the scales' spread
//   experts  z = q(x) W13^T; h = silu(min(g, L)) clamp(u, -L, L) in fp32, quantised without a rounding to 16 bits;
//            y = q(h) W2^T; out[token] = the token's w y in slot order (fp32), then the output type
#include <algorithm>

#include "gemm_tile.cuh"
#include "mi355moe_internal.h"

namespace mi355moe {

// ------------------------------------------------------------------------------------------------ quantisation

// The scale code of a block whose largest magnitude has these fp32 bits (sign cleared; NaN above infinity).
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t top) {
    const uint32_t E = top >> 23;
    return E == 255u ? 255u : (E > 2u ? E - 2u : 0u);
}
// 2^(127 - code); 0 for a NaN block, whose codes are then all zero (inf * 0 and NaN convert to some code: masked)
__device__ __forceinline__ float mx_inv_scale(uint32_t code) {
    return __builtin_bit_cast(float, code == 255u ? 0u : (254u - code) << 23);
}
// Eight values as eight e2m1 codes (round to nearest even, saturating), value 0 in the low bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8], float inv) {
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[0] * inv, v[1] * inv, 1.0f, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[2] * inv, v[3] * inv, 1.0f, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[4] * inv, v[5] * inv, 1.0f, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[6] * inv, v[7] * inv, 1.0f, 3);
    return inv == 0.0f ? 0u : d;
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// Vectors at any address of their element (the hardware takes global accesses at any byte address).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// Eight consecutive values.
template <int XDT>
__device__ __forceinline__ void mx_load8(const void* x, size_t i, float (&v)[8]) {
    if constexpr (XDT == DT_F32) {
        const u32x4_any* p = reinterpret_cast<const u32x4_any*>(static_cast<const float*>(x) + i);
        const f32x4 a = __builtin_bit_cast(f32x4, (u32x4)p[0]), b = __builtin_bit_cast(f32x4, (u32x4)p[1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(x) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (XDT == DT_BF16) {
                v[2 * j] = bf16_to_f32((uint16_t)w[j]);
                v[2 * j + 1] = bf16_to_f32((uint16_t)(w[j] >> 16));
            } else {
                v[2 * j] = (float)u16_as_h(w[j] & 0xFFFFu);
                v[2 * j + 1] = (float)u16_as_h(w[j] >> 16);
            }
        }
    }
}

// Where the scale of row r, block b goes among `rows` rows: rows of nb bytes, or arranged by steps of eight blocks.
__device__ __forceinline__ int64_t scale_place(int64_t r, int b, int nb, int64_t rows, int steps) {
    return steps ? ((b >> 3) * rows + r) * 8 + (b & 7) : r * nb + b;
}
// The bytes behind a row's last scale in its last step.
__device__ __forceinline__ void scale_pad(uint8_t* s, int64_t r, int nb, int64_t rows) {
#pragma unroll 1
    for (int b = nb; b & 7; ++b) s[scale_place(r, b, nb, rows, 1)] = 127;
}

// Four lanes a block, eight values a lane, the lanes of a wave on consecutive places of a row (rows of 4 nb such groups, the
// last ones partly or wholly behind the row's end); any row length, stride and address. Ix: 32 bits where the groups of the
// call fit them (the division by the groups of a row is the kernel's longest instruction sequence). Bound: memory; 32768 x
// 4096 bf16, 268 MB read and 71 written: 68 us, 5.0 TB/s (a large copy: 5.2); 8 x 4096: 2.8 us, a launch's latency.
template <int XDT, typename Ix>
__global__ __launch_bounds__(256) void mx_quant_kernel(const void* __restrict__ x, int64_t stride, Ix items, int K,
                                                       uint8_t* __restrict__ q, uint8_t* __restrict__ s, int64_t rows, int steps) {
    const int nb = (K + 31) / 32, qp = (K + 1) / 2;
    const Ix per_row = (Ix)nb * 4;
    for (Ix i = (Ix)blockIdx.x * 256 + threadIdx.x; i < items; i += (Ix)gridDim.x * 256) {
        const Ix r = i / per_row;
        const int c = (int)(i - r * per_row), n = min(8, K - 8 * c);   // this group's values
        const size_t at = (size_t)r * (size_t)stride + 8 * (size_t)c;
        float v[8];
        if (n == 8) mx_load8<XDT>(x, at, v);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < n ? load_value(x, XDT, at + j) : 0.0f;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
        top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));       // (items % 4 == 0: a block's lanes are all here)
        top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
        const uint32_t code = mx_scale_code(top);
        const uint32_t d = e2m1x8(v, mx_inv_scale(code));
        uint8_t* o = q + (size_t)r * qp + 4 * (size_t)c;
        if (n == 8) *reinterpret_cast<u32_any*>(o) = d;
        else
            for (int b = 0; 2 * b < n; ++b) o[b] = (uint8_t)(d >> (8 * b));
        if ((c & 3) == 0) {
            s[scale_place(r, c >> 2, nb, rows, steps)] = (uint8_t)code;
            if (steps && c + 4 == 4 * nb) scale_pad(s, r, nb, rows);
        }
    }
}

__device__ __forceinline__ float e2m1_value(uint32_t c) {
    // exponent and mantissa bits of 1.x values moved into an fp32's fields; 0 and 0.5 apart
    const uint32_t m = c & 7u;
    const float v = m < 2u ? 0.5f * (float)m : __builtin_bit_cast(float, (126u << 23) + (m << 22));
    return (c & 8u) ? -v : v;
}
__device__ __forceinline__ float mx_scale_value(uint32_t code) {
    return __builtin_bit_cast(float, code == 255u ? 0x7FC00000u : code ? code << 23 : 0x00400000u);
}

// Eight values a thread, laid out as for quantisation: out = e2m1(q) 2^(s - 127), rounded once for 16 bits. Bound: memory;
// 32768 x 4096 to bf16: 66 us, 5.1 TB/s.
template <int ODT, typename Ix>
__global__ __launch_bounds__(256) void mx_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s, Ix items, int K,
                                                         void* __restrict__ out) {
    const int nb = (K + 31) / 32, qp = (K + 1) / 2, per_row = (K + 7) / 8;
    for (Ix i = (Ix)blockIdx.x * 256 + threadIdx.x; i < items; i += (Ix)gridDim.x * 256) {
        const Ix r = i / (Ix)per_row;
        const int c = (int)(i - r * (Ix)per_row), n = min(8, K - 8 * c);
        const uint8_t* p = q + (size_t)r * qp + 4 * (size_t)c;
        const float f = mx_scale_value(s[(size_t)r * nb + (c >> 2)]);
        uint32_t d = 0;
        if (n == 8) d = *reinterpret_cast<const u32_any*>(p);
        else
            for (int b = 0; 2 * b < n; ++b) d |= (uint32_t)p[b] << (8 * b);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = e2m1_value(d >> (4 * j)) * f;
        const size_t o = (size_t)r * K + 8 * (size_t)c;
        if constexpr (ODT == DT_F32) {
            float* w = static_cast<float*>(out) + o;
            if (n == 8) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    reinterpret_cast<u32x4_any*>(w)[k] =
                        __builtin_bit_cast(u32x4, f32x4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]});
            } else
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) w[j] = v[j];
        } else {
            uint16_t* w = static_cast<uint16_t*>(out) + o;
            u32x4 h;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint2 t = pack4(ODT, v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                h[2 * k] = t.x, h[2 * k + 1] = t.y;
            }
            if (n == 8) *reinterpret_cast<u32x4_any*>(w) = h;
            else
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) w[j] = (uint16_t)(h[j >> 1] >> (16 * (j & 1)));
        }
    }
}

// Scales of rows of nb bytes arranged by steps, the bytes behind a row's last one 127: `mats` matrices of `rows` rows, and a
// second matrix of rb rows. One thread a row and step. Bound: memory and a launch's latency (8192 + 4096 rows of 4096: 3.5
// us; a layer's 288 x 2048 rows of 4096, once as it is loaded: 16 us).
__global__ __launch_bounds__(256) void mx_arrange_kernel(const uint8_t* __restrict__ a, int64_t mats, int64_t rows, uint2* __restrict__ ao,
                                                         const uint8_t* __restrict__ b, int64_t rb, uint2* __restrict__ bo, int nb) {
    const int ns = (nb + 7) / 8;
    const int64_t first = mats * rows * ns, total = first + rb * ns;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const bool second = i >= first;
        const int64_t j = second ? i - first : i, nr = second ? rb : rows;
        // consecutive threads take consecutive steps of a row: they read its bytes together
        const int64_t r = j / ns, mat = r / nr;
        const int k = (int)(j - r * ns);
        const uint8_t* src = (second ? b : a) + r * nb + 8 * k;
        uint2 v = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
        if ((nb & 7) == 0 && (reinterpret_cast<uintptr_t>(src) & 7) == 0) v = *reinterpret_cast<const uint2*>(src);
        else {
            uint8_t c[8];
#pragma unroll
            for (int t = 0; t < 8; ++t) c[t] = 8 * k + t < nb ? src[t] : 127;
            v.x = c[0] | c[1] << 8 | c[2] << 16 | (uint32_t)c[3] << 24;
            v.y = c[4] | c[5] << 8 | c[6] << 16 | (uint32_t)c[7] << 24;
        }
        (second ? bo : ao)[(mat * ns + k) * nr + (r - mat * nr)] = v;
    }
}

// ------------------------------------------------------------------------------------------------ few rows

// Weights for at most 16 rows are streamed once, straight from memory into MFMA operands: lane (c = lane % 16, g = lane
// / 16) holds 64 consecutive bytes (four blocks, one a step) of weight row c and the dword of their scales, a wave 16
// rows x 512 of the contraction. A = weights, so lane l's accumulator holds columns n = 4 (l / 16) .. + 3 of row m = l %
// 16. The contraction is cut over waves; their sums join in LDS in wave order. Every weight byte is read once and used for
// 16 rows at most, so memory bounds these kernels; loads go past LDS since nothing in a workgroup shares them.
struct FewRow {
    const uint8_t* q;
    const uint8_t* s;
    uint32_t step;
};
__device__ __forceinline__ FewRow few_row(const uint8_t* q, size_t pitch, const MxScales& s, size_t r) {
    return {q + r * pitch, s.p + r * s.row, s.step};
}
// the four steps' operand bytes and scales of 512 values from block b0 on (nblk blocks in a row; blocks past them: zero
// codes for ZERO, else those of the last one, and scales of 2^0)
template <bool ZERO>
__device__ __forceinline__ void few_load(const FewRow& r, int b0, int g, int nblk, u32x4 (&v)[4], int& sc) {
    const int b = b0 + 4 * g;
    if (b0 + 16 <= nblk) {                                           // (uniform)
        const u32x4* p = reinterpret_cast<const u32x4*>(r.q + (size_t)b * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[i];
        sc = (int)*reinterpret_cast<const u32_any*>(r.s + (size_t)(b >> 3) * r.step + (b & 4));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x4 t = *reinterpret_cast<const u32x4*>(r.q + (size_t)min(b + i, nblk - 1) * 16);
            const bool ok = b + i < nblk || !ZERO;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = ok ? t[j] : 0u;
        }
        uint32_t c = 0x7F7F7F7Fu;                                    // (rows end at any byte: the last dword in single ones)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (b + i < nblk) c ^= (uint32_t)(r.s[(size_t)(b >> 3) * r.step + (b & 4) + i] ^ 127) << (8 * i);
        sc = (int)c;
    }
}
template <int S>
__device__ __forceinline__ f32x4 few_mma(u32x4 a, u32x4 b, f32x4 c, int sa, int sb) {
    const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, S, sa, S, sb);
}
template <int T>
__device__ __forceinline__ void few_product(const FewRow (&w)[T], const FewRow& x, int b0, int g, int nblk, f32x4 (&acc)[T]) {
    u32x4 wv[T][4], xv[4];
    int ws[T], xs;
#pragma unroll
    for (int t = 0; t < T; ++t) few_load<false>(w[t], b0, g, nblk, wv[t], ws[t]);
    few_load<true>(x, b0, g, nblk, xv, xs);
#pragma unroll
    for (int t = 0; t < T; ++t) {
        acc[t] = few_mma<0>(wv[t][0], xv[0], acc[t], ws[t], xs);
        acc[t] = few_mma<1>(wv[t][1], xv[1], acc[t], ws[t], xs);
        acc[t] = few_mma<2>(wv[t][2], xv[2], acc[t], ws[t], xs);
        acc[t] = few_mma<3>(wv[t][3], xv[3], acc[t], ws[t], xs);
    }
}

// grid (N / 32, segments), 64 NW threads: 32 columns of gate and up for a segment of at most 16 rows, the contraction over
// the waves, then SwiGLU and the quantisation of the 32 columns (one block) by a half wave a row. Four waves, so that three
// or more workgroups a CU keep loads in flight through each other's joins: 64 tokens, top 8 of 288 experts (about 240 of them
// hit, 4096 -> 1024, 1.07 GB): 173 us, 6.1 TB/s, more than a copy reaches, since next to nothing is written.
template <int NW>
__global__ __launch_bounds__(64 * NW, 3) void mx_gateup_few_kernel(Mxfp4Args a) {
    __shared__ __align__(16) float red[NW][4][256];
    const int cb = blockIdx.x, s = blockIdx.y;
    if (s >= a.nseg[0]) return;
    const int e = a.seg_expert[s], row0 = a.seg_row0[s], rn = a.seg_rows[s];
    if (rn <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = a.K >> 5;
    FewRow w[4], x;
    const MxScales ws = {a.w13s.p + (size_t)e * a.w13se, a.w13s.row, a.w13s.step};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const size_t r = (size_t)(t >> 1) * a.N + cb * 32 + (t & 1) * 16 + c;
        w[t] = few_row(a.w13 + (size_t)e * 2 * a.N * (a.K / 2), a.K / 2, ws, r);
    }
    x = few_row(a.qx, a.K / 2, MxScales{a.sx, 8, 8u * a.T}, a.tok[row0 + min(c, rn - 1)]);
    f32x4 acc[4] = {};
    for (int b0 = wv * 16; b0 < nblk; b0 += 16 * NW) few_product(w, x, b0, g, nblk, acc);
#pragma unroll
    for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4*>(&red[wv][t][lane * 4]) = acc[t];
    __syncthreads();
    const int n = tid & 31, t = n >> 4;
    for (int m = tid >> 5; m < rn; m += 2 * NW) {
        const int at = ((((n & 15) >> 2) << 4) + m) * 4 + (n & 3);
        float gs = 0.f, us = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            gs += red[i][t][at];
            us += red[i][2 + t][at];
        }
        const float h = swiglu(gs, us, a.limit);
        uint32_t top = abs_bits(h);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
        const uint32_t code = mx_scale_code(top);
        const uint32_t nib =
            code == 255u ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, h * mx_inv_scale(code), 0.0f, 1.0f, 0) & 15u;
        uint32_t d = nib << (4 * (n & 7));
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) d |= (uint32_t)__shfl_xor((int)d, o, 64);
        const size_t r = (size_t)row0 + m;
        if ((n & 7) == 0) *reinterpret_cast<uint32_t*>(a.qh + r * (a.N / 2) + cb * 16 + (n >> 1)) = d;
        if (n == 0) {
            a.sh[scale_place(r, cb, 0, a.P, 1)] = (uint8_t)code;
            if ((cb + 1) * 32 == a.N) scale_pad(a.sh, r, cb + 1, a.P);
        }
    }
}

// ------------------------------------------------------------------------------------------------ few pairs

// A call of few pairs (mxfp4_direct) takes two launches and no tables: every pair is a segment of its own, read from the
// router's ids; gate/up quantises the pair's token itself, and down sums a token's pairs. Pairs that share an expert read
// its weights each for itself (from the caches, where they run together).
__device__ __forceinline__ int pair_expert(const Mxfp4Args& a, int j) {
    int64_t id = a.ids64 ? reinterpret_cast<const int64_t*>(a.ids)[j] : (int64_t)reinterpret_cast<const int32_t*>(a.ids)[j];
    if (a.emap) id = id >= 0 && id < a.n_global ? a.emap[id] : -1;
    return id >= 0 && id < a.n ? (int)id : -1;
}

// grid (N / 32, pairs), 64 NW threads: mx_gateup_few_kernel for one row, which every wave quantises as far as it multiplies it
// (512 values a step: eight a lane, four lanes a block, through 272 bytes of LDS into the lanes that hold the blocks). Bound:
// memory and the latency of the ids, the row and the weights in turn; one token's 8 pairs, 35.7 MB: 10.5 us, 3.4 TB/s.
template <int XDT, int NW>
__global__ __launch_bounds__(64 * NW, 3) void mx_gateup_direct_kernel(Mxfp4Args a) {
    __shared__ __align__(16) float red[NW][4][16];
    __shared__ __align__(16) uint8_t xq[NW][272];
    const int cb = blockIdx.x, j = blockIdx.y;
    const int e = __builtin_amdgcn_readfirstlane(pair_expert(a, j));
    if (e < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = a.K >> 5;
    FewRow w[4];
    const MxScales ws = {a.w13s.p + (size_t)e * a.w13se, a.w13s.row, a.w13s.step};
#pragma unroll
    for (int t = 0; t < 4; ++t)
        w[t] = few_row(a.w13 + (size_t)e * 2 * a.N * (a.K / 2), a.K / 2, ws, (size_t)(t >> 1) * a.N + cb * 32 + (t & 1) * 16 + c);
    const size_t x0 = (size_t)(j / a.topk) * a.x_stride;
    f32x4 acc[4] = {};
    for (int b0 = wv * 16; b0 < nblk; b0 += 16 * NW) {
        u32x4 wv4[4][4];
        int wsc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) few_load<false>(w[t], b0, g, nblk, wv4[t], wsc[t]);
        const int b = b0 + (lane >> 2);                              // this lane's block, and its eighth
        float v[8];
        if (b < nblk) mx_load8<XDT>(a.x, x0 + 32 * (size_t)b + 8 * (lane & 3), v);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
        top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
        const uint32_t code = mx_scale_code(top);
        asm volatile("" ::: "memory");                               // (a wave's LDS accesses are performed in order)
        *reinterpret_cast<uint32_t*>(xq[wv] + 4 * lane) = e2m1x8(v, mx_inv_scale(code));
        if ((lane & 3) == 0) xq[wv][256 + (lane >> 2)] = b < nblk ? (uint8_t)code : (uint8_t)127;
        asm volatile("" ::: "memory");
        u32x4 xv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = *reinterpret_cast<const u32x4*>(xq[wv] + 64 * g + 16 * i);
        const int xs = *reinterpret_cast<const int*>(xq[wv] + 256 + 4 * g);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            acc[t] = few_mma<0>(wv4[t][0], xv[0], acc[t], wsc[t], xs);
            acc[t] = few_mma<1>(wv4[t][1], xv[1], acc[t], wsc[t], xs);
            acc[t] = few_mma<2>(wv4[t][2], xv[2], acc[t], wsc[t], xs);
            acc[t] = few_mma<3>(wv4[t][3], xv[3], acc[t], wsc[t], xs);
        }
    }
    // all sixteen columns of an accumulator are this row's: lane 16 g holds n = 4 g .. + 3
    if (c == 0)
#pragma unroll
        for (int t = 0; t < 4; ++t) *reinterpret_cast<f32x4*>(&red[wv][t][4 * g]) = acc[t];
    __syncthreads();
    if (tid >= 32) return;
    float gs = 0.f, us = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        gs += red[i][tid >> 4][tid & 15];
        us += red[i][2 + (tid >> 4)][tid & 15];
    }
    const float h = swiglu(gs, us, a.limit);
    uint32_t top = abs_bits(h);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    const uint32_t code = mx_scale_code(top);
    const uint32_t nib = code == 255u ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, h * mx_inv_scale(code), 0.0f, 1.0f, 0) & 15u;
    uint32_t d = nib << (4 * (tid & 7));
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) d |= (uint32_t)__shfl_xor((int)d, o, 64);
    if ((tid & 7) == 0) *reinterpret_cast<uint32_t*>(a.qh + (size_t)j * (a.N / 2) + cb * 16 + (tid >> 1)) = d;
    if (tid == 0) {
        a.sh[scale_place(j, cb, 0, a.P, 1)] = (uint8_t)code;
        if ((cb + 1) * 32 == a.N) scale_pad(a.sh, j, cb + 1, a.P);
    }
}

// grid (ceil(K / 16), tokens), 512 threads: 16 columns of one token, a pair a wave at a time, summed in slot order. One token's
// 8 pairs, 17.8 MB: 6.0 us, 3.0 TB/s, the latency of a launch and of two loads in turn (the ids, the weights).
__global__ __launch_bounds__(512) void mx_down_direct_kernel(Mxfp4Args a) {
    __shared__ __align__(16) float sum[MX_MAX_TOPK][16];
    const int t = blockIdx.y, n0 = blockIdx.x * 16;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = a.N >> 5;
    for (int k = wv; k < a.topk; k += 8) {
        const int j = t * a.topk + k;
        const int e = __builtin_amdgcn_readfirstlane(pair_expert(a, j));
        f32x4 acc[1] = {};
        if (e >= 0) {
            const FewRow w[1] = {few_row(a.w2 + (size_t)e * a.K * (a.N / 2), a.N / 2,
                                         MxScales{a.w2s.p + (size_t)e * a.w2se, a.w2s.row, a.w2s.step}, min(n0 + c, a.K - 1))};
            const FewRow x = few_row(a.qh, a.N / 2, MxScales{a.sh, 8, 8u * a.P}, j);
#pragma unroll 2
            for (int b0 = 0; b0 < nblk; b0 += 16) few_product(w, x, b0, g, nblk, acc);
        }
        const float rw = e < 0 ? 0.0f : load_value(a.wts, a.wdt, j);
        if (c == 0) *reinterpret_cast<f32x4*>(&sum[k][4 * g]) = acc[0] * f32x4{rw, rw, rw, rw};
    }
    __syncthreads();
    if (tid >= 4) return;
    f32x4 v = {};
    for (int k = 0; k < a.topk; ++k)
        if (pair_expert(a, t * a.topk + k) >= 0) v += *reinterpret_cast<const f32x4*>(&sum[k][4 * tid]);
    const int n = n0 + 4 * tid;
    const size_t o = (size_t)t * a.out_stride + n;
    if (a.accumulate)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.K) v[i] += load_value(a.out, a.odt, o + i);
    if (n < a.K) store4(a.out, a.odt, o, a.K - n, v);
}

// The eight waves of a workgroup as KS cuts of the contraction x 8 / KS groups of 16 T columns. Store(m, n, four sums of
// columns n ..): called for columns of this wave's own sums (after the join) and rows m < rows.
template <int T, int KS, typename Store>
__device__ __forceinline__ void few_columns(const uint8_t* wq, size_t wqp, const MxScales& ws, int cols, int n0,
                                            const FewRow& x, int nblk, float* red, const Store& store) {
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = wv % KS, grp = wv / KS;
    const int nw = n0 + grp * 16 * T;
    FewRow w[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const size_t r = min(nw + 16 * t + c, cols - 1);
        w[t] = few_row(wq, wqp, ws, r);
    }
    f32x4 acc[T] = {};
    for (int b0 = ks * 16; b0 < nblk; b0 += 16 * KS) few_product(w, x, b0, g, nblk, acc);
    if constexpr (KS > 1) {
#pragma unroll
        for (int t = 0; t < T; ++t) *reinterpret_cast<f32x4*>(red + ((wv * T + t) * 64 + lane) * 4) = acc[t];
        __syncthreads();
        // tile t of a group is summed by the group's wave t % KS
#pragma unroll
        for (int t = 0; t < T; ++t)
            if (t % KS == ks) {
                f32x4 v = {};
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const f32x4 p = *reinterpret_cast<const f32x4*>(red + (((grp * KS + i) * T + t) * 64 + lane) * 4);
                    v += p;
                }
                store(c, nw + 16 * t + 4 * g, v);
            }
    } else {
#pragma unroll
        for (int t = 0; t < T; ++t) store(c, nw + 16 * t + 4 * g, acc[t]);
    }
}

// grid (ceil(K / (16 T 8 / KS)), segments), 512 threads: down projection of a segment of at most 16 rows. Bound: memory; 64
// tokens as above, 0.53 GB: 94 us, 5.7 TB/s.
template <int T, int KS>
__global__ __launch_bounds__(512) void mx_down_few_kernel(Mxfp4Args a) {
    __shared__ __align__(16) float red[KS > 1 ? 8 * T * 256 : 4];
    const int s = blockIdx.y;
    if (s >= a.nseg[0]) return;
    const int e = a.seg_expert[s], row0 = a.seg_row0[s], rn = a.seg_rows[s];
    if (rn <= 0) return;
    const int c = threadIdx.x & 15;
    const size_t xr = (size_t)row0 + min(c, rn - 1);
    const FewRow x = few_row(a.qh, a.N / 2, MxScales{a.sh, 8, 8u * a.P}, xr);
    const float rw = a.w32[xr];
    const int pe = a.pe[xr];
    few_columns<T, KS>(a.w2 + (size_t)e * a.K * (a.N / 2), a.N / 2, MxScales{a.w2s.p + (size_t)e * a.w2se, a.w2s.row, a.w2s.step}, a.K,
                       (int)blockIdx.x * (16 * T * 8 / KS), x, a.N >> 5, red, [&](int m, int n, f32x4 v) {
                           if (m < rn && n < a.K && pe >= 0)
                               *reinterpret_cast<f32x4*>(a.contrib + xr * a.K + n) = v * f32x4{rw, rw, rw, rw};
                       });
}

// grid (ceil(N / (16 T 8 / KS)), ceil(M / 16)), 512 threads: the dense product for few rows. Bound: a launch's latency for small
// weights (1 x 4096 x 4096, 8.9 MB, from cache: 4.0 us), memory for large ones (1 x 131072 x 4096, 285 MB: 52 us, 5.5 TB/s).
template <int T, int KS>
__global__ __launch_bounds__(512) void mx_matmul_few_kernel(MxMatmulArgs a) {
    __shared__ __align__(16) float red[KS > 1 ? 8 * T * 256 : 4];
    const int c = threadIdx.x & 15;
    const int64_t m0 = (int64_t)blockIdx.y * 16;
    const int64_t xr = min(m0 + c, a.M - 1);
    const FewRow x = few_row(a.q, a.K / 2, a.qs, xr);
    few_columns<T, KS>(a.w, a.K / 2, a.ws, a.N, (int)blockIdx.x * (16 * T * 8 / KS), x, a.K >> 5, red,
                       [&](int m, int n, f32x4 v) {
                           if (m0 + m < a.M && n < a.N)
                               store4(a.out, a.odt, (size_t)(m0 + m) * a.out_stride + n, a.N - n, v);
                       });
}

// ------------------------------------------------------------------------------------------------ tiles

template <int BP, int BQ, int WP, int WQ, int ST>
using MxTile = GemmTile<MM_MX4, LAY_ROW, LAY_ROW, BP, BQ, WP, WQ, ST>;

constexpr int MX_SCALES_AHEAD_K = 8192;              // contractions whose scales a 64 x 64 tile takes up front (32 KB)
__device__ __forceinline__ int mx_stages(int K) { return (K + 2 * SB - 1) / (2 * SB); }
__device__ __forceinline__ int mx_tail(int K) { return K % (2 * SB) / 32; }

// The scales of a tile's rows (row r: tile row min(r, last) of the matrix from row0 on, nb bytes each, at any address) for
// stages kb0 .. kb1 - 1, into LDS: 8 bytes of row r for stage k at (k - kb0) * step + 8 r, those behind the row's end 127.
// Published by the barrier before the first stage.
__device__ __forceinline__ void scales_ahead(const MxScales& s, int64_t row0, int last, int rows, int nb, int kb0, int kb1,
                                             unsigned char* lds, int step, int threads) {
    // whole stages first, several loads in flight
    const int n = kb1 - kb0, whole = min(n, nb / 8 - kb0);
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * whole; i += threads) {
        const int r = i / whole, k = i - r * whole;
        const u32_any* p = reinterpret_cast<const u32_any*>(s.p + (size_t)(row0 + min(r, last)) * s.row + 8 * (kb0 + k));
        *reinterpret_cast<uint2*>(lds + k * step + 8 * r) = make_uint2(p[0], p[1]);
    }
    if (whole == n) return;                                          // (uniform; else the last stage is a partial one)
    for (int r = threadIdx.x; r < rows; r += threads) {
        const uint8_t* p = s.p + (size_t)(row0 + min(r, last)) * s.row;
        uint32_t v[2] = {0x7F7F7F7Fu, 0x7F7F7F7Fu};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (8 * whole + 8 * kb0 + j < nb) v[j >> 2] ^= (uint32_t)(p[8 * (kb0 + whole) + j] ^ 127) << (8 * (j & 3));
        *reinterpret_cast<uint2*>(lds + whole * step + 8 * r) = make_uint2(v[0], v[1]);
    }
}

// Dense product: workgroup tiles of BP columns x BQ rows, out or (splits > 1) fp32 partials [split][M][N]. Bound: the largest
// tiles by the matrix cores' clock and the waits at a stage's barrier (8192 x 4096 x 4096: 72 us, 3.8 PFLOP/s of a rate of about
// 5.5; the matrix cores are busy in 54 % of the cycles, at 1.6 GHz where memory-bound kernels run at 2.2, LDS in 30 %, waves
// wait 36 %); the small ones by the latency of a stage, 0.5 us (333 x 2050 x 2080, nine stages: 8.8 us).
template <int BP, int BQ, int WP, int WQ, int ST, bool AHEAD>
__global__ __launch_bounds__(64 * WP * WQ, 2) void mx_matmul_kernel(MxMatmulArgs a, int nt, int mt) {
    using G = GemmTile<MM_MX4, LAY_ROW, LAY_ROW, BP, BQ, WP, WQ, ST, AHEAD>;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int2 tile = tile_order(blockIdx.x, nt, mt);
    const int n0 = tile.x * BP;
    const int64_t m0 = (int64_t)tile.y * BQ;
    const int stages = mx_stages(a.K), per = (stages + a.splits - 1) / a.splits;
    const int kb0 = blockIdx.y * per, kb1 = min(stages, kb0 + per);
    const uint32_t pitch = a.K / 2;
    const int pl = min(BP, a.N - n0) - 1;
    const int ql = (int)min((int64_t)BQ, a.M - m0) - 1;
    G t;
    t.p.init_row(uniform_ptr(a.w + (size_t)n0 * pitch + (size_t)kb0 * SB), wv, lane, [&](int r) { return min(r, pl) * pitch; });
    t.q.init_row(uniform_ptr(a.q + (size_t)m0 * pitch + (size_t)kb0 * SB), wv, lane, [&](int r) { return min(r, ql) * pitch; });
    if constexpr (AHEAD) {
        const int nb = a.K / 32;
        scales_ahead(a.ws, n0, pl, BP, nb, kb0, kb1, lds + G::LDS, (BP + BQ) * 8, G::THREADS);
        scales_ahead(a.qs, m0, ql, BQ, nb, kb0, kb1, lds + G::LDS + BP * 8, (BP + BQ) * 8, G::THREADS);
    } else {
        t.xp.init(a.ws, n0, (a.K + 127) / 128, wv, lane, [&](int r) { return (uint32_t)min(r, pl); });
        t.xq.init(a.qs, m0, (a.K + 127) / 128, wv, lane, [&](int r) { return (uint32_t)min(r, ql); });
    }
    const int tail = kb1 == stages ? mx_tail(a.K) : 0;
    if (kb0 < kb1) t.run(lds, kb0, kb1, tail, tail, 0, 0);
    else
#pragma unroll
        for (int i = 0; i < G::TP; ++i)
#pragma unroll
            for (int j = 0; j < G::TQ; ++j) t.acc[i][j] = f32x16{};
    const int p0 = (wv % WP) * (BP / WP), q0 = (wv / WP) * (BQ / WQ);
    if (a.rows16) {                                                  // (uniform: 16-bit rows at 16-byte addresses)
        const int64_t rows = a.M - m0 - q0;
        t.template store_rows<G::TP>(lds, static_cast<uint16_t*>(a.out) + (size_t)(m0 + q0) * a.out_stride + n0 + p0, a.out_stride,
                                     a.N - n0 - p0, [&](int r) { return r < rows; }, [&](int i, int j, int r) {
                                         return pack4(a.odt, t.acc[i][j][4 * r], t.acc[i][j][4 * r + 1], t.acc[i][j][4 * r + 2],
                                                      t.acc[i][j][4 * r + 3]);
                                     });
        return;
    }
    void* out = a.splits > 1 ? static_cast<void*>(a.part + (size_t)blockIdx.y * a.M * a.N) : a.out;
    const int odt = a.splits > 1 ? (int)DT_F32 : a.odt;
    const int64_t stride = a.splits > 1 ? a.N : a.out_stride;
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
        const int64_t m = m0 + q0 + 32 * j + (lane & 31);
        if (m >= a.M) continue;
#pragma unroll
        for (int i = 0; i < G::TP; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + p0 + 32 * i + 8 * r + 4 * (lane >> 5);
                if (n < a.N)
                    store4(out, odt, (size_t)m * stride + n, a.N - n,
                              f32x4{t.acc[i][j][4 * r], t.acc[i][j][4 * r + 1], t.acc[i][j][4 * r + 2], t.acc[i][j][4 * r + 3]});
            }
    }
}

// out = the splits' partials in order. Bound: memory (partials mostly still in cache).
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int splits, int64_t M, int N, void* out, int odt,
                                                   int64_t stride) {
    const int64_t total = M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += part[(size_t)s * total + i];
        const int64_t m = i / N;
        const size_t o = (size_t)m * stride + (i - m * N);
        if (odt == DT_F32) static_cast<float*>(out)[o] = v;
        else static_cast<uint16_t*>(out)[o] = odt == DT_BF16 ? f32_to_bf16(v) : (uint16_t)h_as_u16((_Float16)v);
    }
}

// Gate/up of a segment: grid (ceil(N / (BP / 2)), segments). A wave's P rows are its gate columns, then the same up
// columns, so the SwiGLU is local to a lane; a 32-column block of a row lies in lanes l and l ^ 32. 2047 tokens, top 8 of 288
// experts, 57 rows an expert (128 x 64 tiles, two workgroups a CU): 274 us. Memory bounds it: 1.28 GB of weights take 217 us
// at the rate that few rows reach, and each 64-column group of an expert reads the expert's tokens again through L2.
template <int BP, int BQ, int WP, int WQ, int ST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void mx_gateup_kernel(Mxfp4Args a) {
    using G = MxTile<BP, BQ, WP, WQ, ST>;
    static_assert(G::TP % 2 == 0, "");
    extern __shared__ __align__(16) unsigned char lds[];
    constexpr int HALF = BP / WP / 2;                                // gate (and up) columns of a wave
    const int s = blockIdx.y;
    if (s >= a.nseg[0]) return;
    const int e = a.seg_expert[s], row0 = a.seg_row0[s], rn = a.seg_rows[s];
    if (rn <= 0) return;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * (BP / 2);
    const uint32_t pitch = a.K / 2;
    auto wrow = [&](int r) {                                         // tile row -> row of w13[e]
        const int w = r / (2 * HALF), i = r % (2 * HALF);
        const int col = min(n0 + w * HALF + (i % HALF), a.N - 1);
        return (uint32_t)(col + (i < HALF ? 0 : a.N));
    };
    auto trow = [&](int r) { return (uint32_t)a.tok[row0 + min(r, rn - 1)]; };
    G t;
    t.p.init_row(uniform_ptr(a.w13 + (size_t)e * 2 * a.N * pitch), wv, lane, [&](int r) { return wrow(r) * pitch; });
    t.q.init_row(a.qx, wv, lane, [&](int r) { return trow(r) * pitch; });
    t.xp.init(MxScales{a.w13s.p + (size_t)e * a.w13se, a.w13s.row, a.w13s.step}, 0, (a.K + 127) / 128, wv, lane, wrow);
    t.xq.init(MxScales{a.sx, 8, 8u * a.T}, 0, (a.K + 127) / 128, wv, lane, trow);
    t.run(lds, 0, mx_stages(a.K), mx_tail(a.K), mx_tail(a.K), 0, 0);
    const int p0 = (wv % WP) * HALF, q0 = (wv / WP) * (BQ / WQ), hl = lane >> 5;
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) {
        const int m = q0 + 32 * j + (lane & 31);
#pragma unroll
        for (int i = 0; i < G::TP / 2; ++i) {
            float h[16];
            uint32_t top = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                h[r] = swiglu(t.acc[i][j][r], t.acc[i + G::TP / 2][j][r], a.limit);
                top = max(top, abs_bits(h[r]));
            }
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            const uint32_t code = mx_scale_code(top);
            const float inv = mx_inv_scale(code);
            // this lane's codes: columns 8 r + 4 hl .. + 3 for r = 0 .. 3, 16 bits each
            uint32_t d[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float v[8] = {h[8 * k], h[8 * k + 1], h[8 * k + 2], h[8 * k + 3],
                                    h[8 * k + 4], h[8 * k + 5], h[8 * k + 6], h[8 * k + 7]};
                d[k] = e2m1x8(v, inv);
            }
            // lane l (hl 0) takes bytes 0 .. 7 of the block, lane l ^ 32 bytes 8 .. 15
            const uint32_t other = (uint32_t)__shfl_xor((int)(hl ? d[0] : d[1]), 32, 64);
            const uint32_t lo = hl ? other : d[0], hi = hl ? d[1] : other;   // columns 8 r .. + 3 and + 4 .. + 7
            const uint2 v = make_uint2((lo & 0xFFFFu) | (hi << 16), (lo >> 16) | (hi & 0xFFFF0000u));
            const int col = n0 + p0 + 32 * i;
            if (m < rn && col < a.N) {
                const size_t rr = (size_t)row0 + m;
                *reinterpret_cast<uint2*>(a.qh + rr * (a.N / 2) + col / 2 + 8 * hl) = v;
                if (hl == 0) {
                    a.sh[scale_place(rr, col / 32, 0, a.P, 1)] = (uint8_t)code;
                    if (col + 32 == a.N) scale_pad(a.sh, rr, a.N / 32, a.P);
                }
            }
        }
    }
}

// Down of a segment: grid (ceil(K / BP), segments), weighted contributions in fp32 (2047 tokens as above: 0.64 GB of weights
// and 268 MB of contributions, 156 us, 5.8 TB/s).
template <int BP, int BQ, int WP, int WQ, int ST>
__global__ __launch_bounds__(64 * WP * WQ, 2) void mx_down_kernel(Mxfp4Args a) {
    using G = MxTile<BP, BQ, WP, WQ, ST>;
    extern __shared__ __align__(16) unsigned char lds[];
    const int s = blockIdx.y;
    if (s >= a.nseg[0]) return;
    const int e = a.seg_expert[s], row0 = a.seg_row0[s], rn = a.seg_rows[s];
    if (rn <= 0) return;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * BP;
    const uint32_t pitch = a.N / 2;
    auto wrow = [&](int r) { return (uint32_t)min(n0 + r, a.K - 1); };
    auto xrow = [&](int r) { return (uint32_t)min(r, rn - 1); };
    const int p0 = (wv % WP) * (BP / WP), q0 = (wv / WP) * (BQ / WQ);
    float rw[G::TQ];                                                 // the weights of this lane's rows
#pragma unroll
    for (int j = 0; j < G::TQ; ++j) rw[j] = a.w32[row0 + min(q0 + 32 * j + (lane & 31), rn - 1)];
    G t;
    t.p.init_row(uniform_ptr(a.w2 + (size_t)e * a.K * pitch), wv, lane, [&](int r) { return wrow(r) * pitch; });
    t.q.init_row(uniform_ptr(a.qh + (size_t)row0 * pitch), wv, lane, [&](int r) { return xrow(r) * pitch; });
    t.xp.init(MxScales{a.w2s.p + (size_t)e * a.w2se, a.w2s.row, a.w2s.step}, 0, (a.N + 127) / 128, wv, lane, wrow);
    t.xq.init(MxScales{a.sh, 8, 8u * a.P}, row0, (a.N + 127) / 128, wv, lane, xrow);
    t.run(lds, 0, mx_stages(a.N), mx_tail(a.N), mx_tail(a.N), 0, 0);
    // (rows of no valid pair get a value too, which the combine does not read)
    t.template store_rows<G::TP>(lds, a.contrib + (size_t)(row0 + q0) * a.K + n0 + p0, a.K, a.K - n0 - p0,
                                 [&](int r) { return q0 + r < rn; }, [&](int i, int j, int r) {
                                     const f32x16& v = t.acc[i][j];
                                     return f32x4{rw[j] * v[4 * r], rw[j] * v[4 * r + 1], rw[j] * v[4 * r + 2], rw[j] * v[4 * r + 3]};
                                 });
}

// grid (T, ceil(K / 1024)), 256 threads: four columns a thread, a token's valid pairs in slot order (accumulate: added
// to out's values, one rounding). Bound: memory; 2047 tokens x 8 x 4096 fp32, 268 MB: 54 us, 5.2 TB/s (summing in the down
// kernel by atomics would leave the order of the sum to chance).
__global__ __launch_bounds__(256) void mx_combine_kernel(Mxfp4Args a) {
    const int t = blockIdx.x, col = blockIdx.y * 1024 + 4 * threadIdx.x;
    if (col >= a.K) return;
    f32x4 sum = {};
    for (int k0 = 0; k0 < a.topk; k0 += 4) {
        f32x4 c[4];
        bool ok[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int pos = a.inv[t * a.topk + min(k0 + k, a.topk - 1)];
            ok[k] = k0 + k < a.topk && a.pe[pos] >= 0;
            c[k] = ok[k] ? *reinterpret_cast<const f32x4*>(a.contrib + (size_t)pos * a.K + col) : f32x4{};
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (ok[k]) sum += c[k];
    }
    const size_t o = (size_t)t * a.out_stride + col;
    if (a.accumulate) {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += load_value(a.out, a.odt, o + j);
    }
    store4(a.out, a.odt, o, 4, sum);
}

// ------------------------------------------------------------------------------------------------ launchers

static unsigned grid_for(int64_t items) { return (unsigned)std::min<int64_t>((items + 255) / 256, 256 * 32); }

template <int XDT>
static void run_mx_quant(const void* x, int64_t stride, int64_t rows, int K, uint8_t* q, uint8_t* s, int steps, hipStream_t st) {
    const int64_t items = rows * 4 * ((K + 31) / 32);
    const dim3 g(grid_for(items)), d(256);
    if (items + 256 * 256 * 32 < (int64_t(1) << 32))
        hipLaunchKernelGGL((mx_quant_kernel<XDT, uint32_t>), g, d, 0, st, x, stride, (uint32_t)items, K, q, s, rows, steps);
    else hipLaunchKernelGGL((mx_quant_kernel<XDT, int64_t>), g, d, 0, st, x, stride, items, K, q, s, rows, steps);
}

int launch_mx_quant(const void* x, int xdt, int64_t stride, int64_t rows, int K, uint8_t* q, uint8_t* s, int steps,
                    hipStream_t st) {
    if (rows <= 0) return 0;
    if (xdt == DT_F32) run_mx_quant<DT_F32>(x, stride, rows, K, q, s, steps, st);
    else if (xdt == DT_F16) run_mx_quant<DT_F16>(x, stride, rows, K, q, s, steps, st);
    else run_mx_quant<DT_BF16>(x, stride, rows, K, q, s, steps, st);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int ODT>
static void run_mx_dequant(const uint8_t* q, const uint8_t* s, int64_t rows, int K, void* out, hipStream_t st) {
    const int64_t items = rows * ((K + 7) / 8);
    const dim3 g(grid_for(items)), d(256);
    if (items + 256 * 256 * 32 < (int64_t(1) << 32))
        hipLaunchKernelGGL((mx_dequant_kernel<ODT, uint32_t>), g, d, 0, st, q, s, (uint32_t)items, K, out);
    else hipLaunchKernelGGL((mx_dequant_kernel<ODT, int64_t>), g, d, 0, st, q, s, items, K, out);
}

int launch_mx_dequant(const uint8_t* q, const uint8_t* s, int64_t rows, int K, void* out, int odt, hipStream_t st) {
    if (rows <= 0) return 0;
    if (odt == DT_F32) run_mx_dequant<DT_F32>(q, s, rows, K, out, st);
    else if (odt == DT_F16) run_mx_dequant<DT_F16>(q, s, rows, K, out, st);
    else run_mx_dequant<DT_BF16>(q, s, rows, K, out, st);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_join(const float* part, int splits, int64_t M, int N, void* out, int odt, int64_t stride, hipStream_t st) {
    hipLaunchKernelGGL(join_kernel, dim3(grid_for(M * N)), dim3(256), 0, st, part, splits, M, N, out, odt, stride);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// Few rows stream the weights: always up to four, up to 16 while the workgroups (16 columns x 16 rows) are at most three a CU,
// up to 64 at one a CU, since every group of 16 rows reads the weights and its rows through L2 again. us streamed / by tiles,
// cold weights, K = 4096: N = 1024, M = 16 4.8 / 8.3, 64 4.9 / 8.4; N = 4096, 16 5.3 / 9.4, 32 7.7 / 9.6, 64 12.1 / 10.0; N =
// 12288, 8 9.0 / 10.1, 16 10.2 / 10.2, 32 16.7 / 10.3; N = 32768, 1 16.8 / 18.2, 16 23.5 / 18.3; N = 131072, 1 52 / 66, 16 80 / 68;
// 4096 from 16384, 16 12.7 / 14.0, 32 21.4 / 15.7.
static bool mx_streams(int64_t M, int64_t N) {
    return M <= 4 || (M <= 64 && (M + 15) / 16 * ((N + 15) / 16) <= (M <= 16 ? 768 : 256));
}
// The smallest tile that leaves at most one workgroup a CU (its stages deep enough to keep the memory busy), else 128 x 128
// with two a CU, else 256 x 256 from 192 of them on (no tile of mostly absent rows: 131072 columns of 4096 for 16 rows 91 us by
// the largest tiles, 68 by 128 x 64). us by kind 256 / 128 / 128 deep / 128 x 64 / 64 (N = K = 4096):
// M = 200 27 / 16.1 / 13.3 / 11.1 / 10.8, 512 29 / 18.3 / 14.7 / 12.4 / 15.9, 1024 30 / 20.9 / 16.9 / 22.8 / 27.3,
// 2048 32.7 / 28.0 / 30.3 / 42 / 49, 8192 80 / 108 / 124 / - / 184. Long contractions of few tiles are cut (128 x 512 x
// 32768, 16 tiles: 47 us, in 4 parts 19.5); a cut of fewer than 16 stages costs more than it gains.
MxMatmulPlan plan_mx_matmul(int64_t M, int64_t N, int64_t K) {
    MxMatmulPlan p{};
    p.few = mx_streams(M, N);
    p.splits = 1;
    if (p.few) return p;
    auto tiles = [&](int64_t bp, int64_t bq) { return ((N + bp - 1) / bp) * ((M + bq - 1) / bq); };
    const int64_t stages = (K + 255) / 256, t64 = tiles(64, 64);
    if (t64 <= 256) {
        p.tile = TILE_64;
        while (t64 * p.splits * 2 <= 256 && stages / (p.splits * 2) >= 16) p.splits *= 2;
    } else if (tiles(128, 64) <= 256 || M <= 64) p.tile = TILE_128_64;
    else if (tiles(128, 128) <= 256) p.tile = TILE_128_DEEP;
    else if (tiles(256, 256) < 192 || M <= 128) p.tile = TILE_128;
    else p.tile = TILE_256;
    // scales in an order of their own: for rows of no whole dwords, except where a workgroup reads a tile's scales up front;
    // and for the largest tiles, which would touch as many lines for their scales as for their codes
    p.arrange = p.tile == TILE_256 || (K % 128 != 0 && !(p.tile == TILE_64 && K <= MX_SCALES_AHEAD_K));
    return p;
}

template <int BP, int BQ, int WP, int WQ, int ST, bool AHEAD = false>
static int run_mx_matmul(MxMatmulArgs a, hipStream_t st) {
    a.rows16 = a.splits == 1 && a.odt != DT_F32 && a.N % 8 == 0 && a.out_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    using G = GemmTile<MM_MX4, LAY_ROW, LAY_ROW, BP, BQ, WP, WQ, ST, AHEAD>;
    constexpr int most = G::LDS + (AHEAD ? (BP + BQ) * 8 * (MX_SCALES_AHEAD_K / 256) : 0);
    if (!allow_lds<mx_matmul_kernel<BP, BQ, WP, WQ, ST, AHEAD>>(most)) return -1;
    const int nt = (a.N + BP - 1) / BP, mt = (int)((a.M + BQ - 1) / BQ);
    const int per = ((a.K + 255) / 256 + a.splits - 1) / a.splits;
    const int bytes = G::LDS + (AHEAD ? (BP + BQ) * 8 * per : 0);
    hipLaunchKernelGGL((mx_matmul_kernel<BP, BQ, WP, WQ, ST, AHEAD>), dim3(nt * mt, a.splits), dim3(G::THREADS), bytes, st, a, nt, mt);
    return 0;
}

int launch_mx_matmul(const MxMatmulArgs& a, const MxMatmulPlan& p, hipStream_t st) {
    if (p.few) {
        const int nblk = a.K >> 5;
        const unsigned my = (unsigned)((a.M + 15) / 16);
        auto grid = [&](int cols) { return dim3((a.N + cols - 1) / cols, my); };
        if (nblk > 64) hipLaunchKernelGGL((mx_matmul_few_kernel<1, 8>), grid(16), dim3(512), 0, st, a);
        else if (nblk > 32) hipLaunchKernelGGL((mx_matmul_few_kernel<1, 4>), grid(32), dim3(512), 0, st, a);
        else if (nblk > 16) hipLaunchKernelGGL((mx_matmul_few_kernel<1, 2>), grid(64), dim3(512), 0, st, a);
        else hipLaunchKernelGGL((mx_matmul_few_kernel<1, 1>), grid(128), dim3(512), 0, st, a);
    } else {
        const int r = p.tile == TILE_256        ? run_mx_matmul<256, 256, 2, 4, 2>(a, st)
                      : p.tile == TILE_128      ? run_mx_matmul<128, 128, 2, 2, 2>(a, st)
                      : p.tile == TILE_128_DEEP ? run_mx_matmul<128, 128, 2, 2, 4>(a, st)
                      : p.tile == TILE_128_64   ? run_mx_matmul<128, 64, 2, 2, 4>(a, st)
                      : a.K <= MX_SCALES_AHEAD_K ? run_mx_matmul<64, 64, 2, 2, 4, true>(a, st)
                                                 : run_mx_matmul<64, 64, 2, 2, 4>(a, st);
        if (r) return r;
        if (a.splits > 1) {
            if (hipGetLastError() != hipSuccess) return -1;
            return launch_join(a.part, a.splits, a.M, a.N, a.out, a.odt, a.out_stride, st);
        }
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_mx_arrange(const uint8_t* a, int64_t mats, int64_t rows, uint8_t* ao, const uint8_t* b, int64_t rb, uint8_t* bo, int nb,
                      hipStream_t st) {
    const int64_t items = (mats * rows + rb) * ((nb + 7) / 8);
    hipLaunchKernelGGL(mx_arrange_kernel, dim3(grid_for(items)), dim3(256), 0, st, a, mats, rows, reinterpret_cast<uint2*>(ao), b, rb,
                       reinterpret_cast<uint2*>(bo), nb);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int BP, int BQ, int WP, int WQ, int ST>
static int run_mx_gateup(const Mxfp4Args& a, hipStream_t st) {
    using G = MxTile<BP, BQ, WP, WQ, ST>;
    if (!allow_lds<mx_gateup_kernel<BP, BQ, WP, WQ, ST>>(G::LDS)) return -1;
    hipLaunchKernelGGL((mx_gateup_kernel<BP, BQ, WP, WQ, ST>), dim3((a.N + BP / 2 - 1) / (BP / 2), a.S_cap), dim3(G::THREADS), G::LDS, st, a);
    return 0;
}
template <int BP, int BQ, int WP, int WQ, int ST>
static int run_mx_down(const Mxfp4Args& a, hipStream_t st) {
    using G = MxTile<BP, BQ, WP, WQ, ST>;
    if (!allow_lds<mx_down_kernel<BP, BQ, WP, WQ, ST>>(G::LDS)) return -1;
    hipLaunchKernelGGL((mx_down_kernel<BP, BQ, WP, WQ, ST>), dim3((a.K + BP - 1) / BP, a.S_cap), dim3(G::THREADS), G::LDS, st, a);
    return 0;
}

template <int NW>
static void run_mx_gateup_direct(const Mxfp4Args& a, hipStream_t st) {
    const dim3 g(a.N / 32, a.P), d(64 * NW);
    if (a.xdt == DT_F32) hipLaunchKernelGGL((mx_gateup_direct_kernel<DT_F32, NW>), g, d, 0, st, a);
    else if (a.xdt == DT_F16) hipLaunchKernelGGL((mx_gateup_direct_kernel<DT_F16, NW>), g, d, 0, st, a);
    else hipLaunchKernelGGL((mx_gateup_direct_kernel<DT_BF16, NW>), g, d, 0, st, a);
}
int launch_mxfp4_direct(const Mxfp4Args& a, hipStream_t st) {
    run_mx_gateup_direct<4>(a, st);
    hipLaunchKernelGGL(mx_down_direct_kernel, dim3((a.K + 15) / 16, a.T), dim3(512), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_mxfp4(const Mxfp4Args& a, hipStream_t st) {
    if (launch_mx_quant(a.x, a.xdt, a.x_stride, a.T, a.K, a.qx, a.sx, 1, st)) return -1;
    const bool few = a.seg == MX_FEW;
    if (few) hipLaunchKernelGGL(mx_gateup_few_kernel<4>, dim3(a.N / 32, a.S_cap), dim3(256), 0, st, a);
    else if (a.seg == MX_TILE ? run_mx_gateup<128, 64, 2, 2, 3>(a, st) : run_mx_gateup<128, 128, 2, 2, 2>(a, st)) return -1;
    if (few) {
        const int nblk = a.N >> 5;
        auto grid = [&](int cols) { return dim3((a.K + cols - 1) / cols, a.S_cap); };
        if (nblk > 64) hipLaunchKernelGGL((mx_down_few_kernel<2, 8>), grid(32), dim3(512), 0, st, a);
        else if (nblk > 32) hipLaunchKernelGGL((mx_down_few_kernel<2, 4>), grid(64), dim3(512), 0, st, a);
        else if (nblk > 16) hipLaunchKernelGGL((mx_down_few_kernel<2, 2>), grid(128), dim3(512), 0, st, a);
        else hipLaunchKernelGGL((mx_down_few_kernel<2, 1>), grid(256), dim3(512), 0, st, a);
    } else if (a.seg == MX_TILE ? run_mx_down<128, 64, 2, 2, 3>(a, st) : run_mx_down<128, 128, 2, 2, 2>(a, st)) return -1;
    hipLaunchKernelGGL(mx_combine_kernel, dim3(a.T, (a.K + 1023) / 1024), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace mi355moe
