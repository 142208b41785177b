// Workgroup tiles of a matrix product on gfx950's matrix cores, for 16-bit operands and for MXFP4 (e2m1 elements, one
// e8m0 scale per 32 of the contraction).
//
//   out[m][n] = sum over k of P[n][k] Q[m][k]
//
// A workgroup of WP x WQ waves owns BP values of n and BQ of m; a wave owns (BP / WP) x (BQ / WQ) of them as 32 x 32
// MFMA tiles whose D rows are n and D columns m, so a lane holds groups of four consecutive n of one m: the output's
// contiguous dimension, and, over the lane pair l, l ^ 32, whole blocks of 32 n for a quantising epilogue.
//
// A stage is 128 bytes of the contraction: 64 16-bit values or 256 MXFP4 codes, the same bytes and the same fragment
// (16 bytes of one row per lane) for v_mfma_f32_32x32x16 and v_mfma_scale_f32_32x32x64_f8f6f4. Lane half h = lane / 32
// takes 16-byte chunks 4h .. 4h + 3 of a row in the stage's four steps: both operands use the same order, so the sum is
// over the same pairs, and the four scales a lane needs are one aligned dword of its row's scales (one byte a step).
// Stages are filled by asynchronous global-to-LDS loads (16 bytes a lane, 1 KB a wave instruction).
//
// An operand lies in memory in one of two ways:
//   ROW  the contraction is contiguous: LDS holds row R's eight 16-byte chunks, chunk g at slot g ^ ((R >> 1) & 7)
//   COL  the contraction is the row index (16-bit only): LDS holds 64 rows of R values; a fragment is two
//        ds_read_b64_tr_b16, each of which hands lane i of 16 column i of a 4 x 16 block. Consecutive rows are whole
//        bank rounds apart, so the 32-byte segments of row k are rotated (xor) by k's place among the rows that one
//        read touches.
// Both swizzles are applied through the load addresses.
#pragma once
#include "common.cuh"
#include "mi355moe_internal.h"

namespace mi355moe {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

enum MmKind { MM_F16 = 0, MM_BF16 = 1, MM_MX4 = 2 };
enum { LAY_ROW = 0, LAY_COL = 1 };

__device__ __forceinline__ f32x16 mma16(std::integral_constant<int, MM_F16>, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma16(std::integral_constant<int, MM_BF16>, u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
// S: the byte of the scale dwords that this step takes
template <int S>
__device__ __forceinline__ f32x16 mma_mx(u32x4 a, u32x4 b, f32x16 c, int sa, int sb) {
    const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, S, sa, S, sb);
}

__device__ __forceinline__ int row_swz(int R) { return (R >> 1) & 7; }
// the xor of row k's 32-byte segment index (R values a row): distinct over the rows one transposing read touches, as far
// as the row's segments go
template <int R>
__device__ __forceinline__ int col_swz(int k) {
    if constexpr (R >= 256) return ((k & 3) | ((k >> 3) & 4)) << 1;
    else if constexpr (R == 128) return (k & 3) << 1;
    else return ((k >> 1) & 1) << 1;
}

// Staging of one operand of R rows (LAY_COL: R columns) by NW waves.
template <int LAY, int R, int NW>
struct Stager {
    static constexpr int INST = R / 8 / NW;          // 1 KB wave instructions per stage and wave
    static_assert(INST * 8 * NW == R, "rows divide over the waves");
    const unsigned char* base;                       // wave-uniform
    uint32_t off[INST];                              // this lane's source bytes of each instruction
    int lds;                                         // this wave's first byte of the operand's stage

    // ROW: rowoff(R) = byte offset of tile row R from `b`
    template <typename F>
    __device__ __forceinline__ void init_row(const void* b, int wv, int lane, const F& rowoff) {
        static_assert(LAY == LAY_ROW, "");
        base = static_cast<const unsigned char*>(b);
        lds = wv * INST * 1024;
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            const int r = (wv * INST + j) * 8 + (lane >> 3);
            off[j] = rowoff(r) + (((lane & 7) ^ row_swz(r)) << 4);
        }
    }
    // COL: row k at ld * k bytes; `cols` values of the row from `b` on may be read (a multiple of 8)
    __device__ __forceinline__ void init_col(const void* b, int wv, int lane, uint32_t ld, int cols) {
        static_assert(LAY == LAY_COL, "");
        base = static_cast<const unsigned char*>(b);
        lds = wv * INST * 1024;
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            const int p = col_slot(wv, j, lane);
            const int k = p / (R / 8);
            const int c = p % (R / 8);
            const int col = (((c >> 1) ^ col_swz<R>(k)) << 4) + ((c & 1) << 3);
            off[j] = (uint32_t)k * ld + 2u * (uint32_t)min(col, cols - 8);
        }
    }
    __device__ __forceinline__ int col_slot(int wv, int j, int lane) const { return (wv * INST + j) * 64 + lane; }
    __device__ __forceinline__ void issue(unsigned char* st) const {
#pragma unroll
        for (int j = 0; j < INST; ++j) dma16_base(base, off[j], st + lds + j * 1024);
    }
    // the last stage, of which only `valid` chunks (ROW) or rows (COL, of ld bytes) exist: what lies behind them is
    // loaded from the last one that exists (and cleared in LDS by clear_tail)
    __device__ __forceinline__ void issue_tail(unsigned char* st, int wv, int lane, int valid, uint32_t ld) const {
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            uint32_t o = off[j];
            if constexpr (LAY == LAY_ROW) {
                const int g = (lane & 7) ^ row_swz((wv * INST + j) * 8 + (lane >> 3));
                if (g >= valid) o -= (uint32_t)(g - valid + 1) << 4;
            } else {
                const int k = col_slot(wv, j, lane) / (R / 8);
                if (k >= valid) o -= (uint32_t)(k - valid + 1) * ld;
            }
            dma16_base(base, o, st + lds + j * 1024);
        }
    }
    static __device__ __forceinline__ void clear_tail(unsigned char* st, int tid, int valid) {
        const u32x4 z = {0, 0, 0, 0};
        if constexpr (LAY == LAY_ROW) {
            for (int i = tid; i < R * 8; i += NW * 64) {
                const int r = i >> 3, g = i & 7;
                if (g >= valid) *reinterpret_cast<u32x4*>(st + r * 128 + ((g ^ row_swz(r)) << 4)) = z;
            }
        } else {
            for (int i = valid * (R / 8) + tid; i < 64 * (R / 8); i += NW * 64) *reinterpret_cast<u32x4*>(st + i * 16) = z;
        }
    }
};

// The 16 bytes (lane r = lane % 32, half h) of step s of the 32-row tile at row r0.
template <int LAY, int R>
__device__ __forceinline__ u32x4 fragment(const unsigned char* st, int r0, int s, int lane) {
    const int c = 4 * (lane >> 5) + s;
    if constexpr (LAY == LAY_ROW) {
        const int r = r0 + (lane & 31);
        return *reinterpret_cast<const u32x4*>(st + r * 128 + ((c ^ row_swz(r)) << 4));
    } else {
        const int i = lane & 15;
        const int seg = (r0 >> 4) + ((lane >> 4) & 1);
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        union { s16x4 v[2]; u32x4 q; } u;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int k = 8 * c + 4 * t + (i >> 2);
            const unsigned char* a = st + k * (2 * R) + ((seg ^ col_swz<R>(k)) << 5) + ((i & 3) << 3);
            u.v[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(uint32_t)(uintptr_t)a);
        }
        return u.q;
    }
}

// Scale dwords of an MXFP4 operand: a stage holds 8 bytes of each row's scales (the dword of half h at 4h), 256 bytes
// (32 rows) a wave instruction of 4 bytes a lane.
template <int R, int NW>
struct ScaleStager {
    static constexpr int INST = (R / 32 + NW - 1) / NW;
    const unsigned char* base;
    uint32_t off[INST];
    uint32_t last[INST];                             // the row's last dword
    int lds[INST];
    template <typename F>
    __device__ __forceinline__ void init(const void* b, int wv, int lane, int dwords, const F& rowoff) {
        base = static_cast<const unsigned char*>(b);
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            const int blk = min(wv * INST + j, R / 32 - 1);          // (waves past the rows repeat the last block)
            const int r = blk * 32 + (lane >> 1);
            off[j] = rowoff(r) + ((lane & 1) << 2);
            last[j] = rowoff(r) + 4u * (uint32_t)(dwords - 1);
            lds[j] = blk * 256;
        }
    }
    // stage kb; a row with an odd number of dwords ends in the middle of its last stage: that half reads the last dword
    // again (its codes are cleared)
    __device__ __forceinline__ void issue(unsigned char* st, int kb) const {
#pragma unroll
        for (int j = 0; j < INST; ++j) dma4(base + min(off[j] + 8u * (uint32_t)kb, last[j]), st + lds[j]);
    }
    static __device__ __forceinline__ int read(const unsigned char* st, int r0, int lane) {
        return *reinterpret_cast<const int*>(st + (r0 + (lane & 31)) * 8 + ((lane >> 5) << 2));
    }
};

// One workgroup's product. `Cfg`: MM, PL, QL (layouts), BP, BQ, WP, WQ.
template <int MM_, int PL_, int QL_, int BP_, int BQ_, int WP_, int WQ_, int STAGES_>
struct GemmTile {
    static constexpr int MM = MM_, PL = PL_, QL = QL_, BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, STAGES = STAGES_;
    static constexpr int NW = WP * WQ, THREADS = 64 * NW;
    static constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32;      // 32 x 32 tiles of a wave
    static constexpr bool MX = MM == MM_MX4;
    static constexpr int STAGE = (BP + BQ) * (MX ? 136 : 128);      // bytes: P rows, Q rows, P scales, Q scales
    static constexpr int LDS = STAGES * STAGE;
    static constexpr int SCL = (BP + BQ) * 128;
    using SP = Stager<PL, BP, NW>;
    using SQ = Stager<QL, BQ, NW>;
    using XP = ScaleStager<BP, NW>;
    using XQ = ScaleStager<BQ, NW>;
    static constexpr int LOADS = SP::INST + SQ::INST + (MX ? XP::INST + XQ::INST : 0);

    SP p;
    SQ q;
    XP xp;
    XQ xq;
    f32x16 acc[TP][TQ];

    // Stages kb0 .. kb1 - 1 of the contraction (kb0 < kb1; p.base and q.base at stage kb0). tail: what the last one
    // holds (8-value chunks for ROW, rows for COL; 0: it is whole). ldp / ldq: row bytes of COL operands.
    template <int S>
    __device__ __forceinline__ void step(const unsigned char* st, int p0, int q0, int lane, const int (&sp)[TP],
                                         const int (&sq)[TQ]) {
        u32x4 a[TP], b[TQ];
#pragma unroll
        for (int i = 0; i < TP; ++i) a[i] = fragment<PL, BP>(st, p0 + 32 * i, S, lane);
#pragma unroll
        for (int j = 0; j < TQ; ++j) b[j] = fragment<QL, BQ>(st + BP * 128, q0 + 32 * j, S, lane);
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int j = 0; j < TQ; ++j) {
                if constexpr (MX) acc[i][j] = mma_mx<S>(a[i], b[j], acc[i][j], sp[i], sq[j]);
                else acc[i][j] = mma16(std::integral_constant<int, MM>{}, a[i], b[j], acc[i][j]);
            }
    }
    __device__ __forceinline__ void compute(const unsigned char* st, int p0, int q0, int lane) {
        int sp[TP], sq[TQ];
        if constexpr (MX) {
#pragma unroll
            for (int i = 0; i < TP; ++i) sp[i] = XP::read(st + SCL, p0 + 32 * i, lane);
#pragma unroll
            for (int j = 0; j < TQ; ++j) sq[j] = XQ::read(st + SCL + BP * 8, q0 + 32 * j, lane);
        }
        step<0>(st, p0, q0, lane, sp, sq);
        step<1>(st, p0, q0, lane, sp, sq);
        step<2>(st, p0, q0, lane, sp, sq);
        step<3>(st, p0, q0, lane, sp, sq);
    }
    __device__ __forceinline__ void run(unsigned char* lds, int kb0, int kb1, int tail_p, int tail_q, uint32_t ldp,
                                        uint32_t ldq) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int p0 = (wv % WP) * (BP / WP), q0 = (wv / WP) * (BQ / WQ);
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int j = 0; j < TQ; ++j) acc[i][j] = f32x16{};
        const uint64_t advp = PL == LAY_ROW ? 128 : 64 * (uint64_t)ldp, advq = QL == LAY_ROW ? 128 : 64 * (uint64_t)ldq;
        auto issue = [&](int slot, int kb) {
            unsigned char* st = lds + slot * STAGE;
            if (kb == kb1 - 1 && tail_p) {
                p.issue_tail(st, wv, lane, tail_p, ldp);
                q.issue_tail(st + BP * 128, wv, lane, tail_q, ldq);
            } else {
                p.issue(st);
                q.issue(st + BP * 128);
            }
            if constexpr (MX) {
                xp.issue(st + SCL, kb);
                xq.issue(st + SCL + BP * 8, kb);
            }
            p.base += advp;
            q.base += advq;
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s)
            if (kb0 + s < kb1) issue(s, kb0 + s);
        int cur = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (STAGES > 2 && kb + 1 < kb1) WAIT_VM((STAGES - 2) * LOADS);
            else WAIT_VM(0);
            LDS_BARRIER();
            const int nxt = cur == 0 ? STAGES - 1 : cur - 1;         // the slot read in the previous step
            if (kb + STAGES - 1 < kb1) issue(nxt, kb + STAGES - 1);
            unsigned char* st = lds + cur * STAGE;
            if (kb == kb1 - 1 && tail_p) {                           // (uniform)
                SP::clear_tail(st, tid, tail_p);
                SQ::clear_tail(st + BP * 128, tid, tail_q);
                __syncthreads();
            }
            compute(st, p0, q0, lane);
            cur = cur + 1 == STAGES ? 0 : cur + 1;
        }
    }
};

// Row (n) of accumulator register r: 8 (r / 4) + 4 (lane / 32) + r % 4; column (m): lane % 32.

__device__ __forceinline__ float load_value(const void* x, int xdt, size_t i) {
    if (xdt == DT_F32) return reinterpret_cast<const float*>(x)[i];
    if (xdt == DT_BF16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[i]);
    return (float)u16_as_h(reinterpret_cast<const uint16_t*>(x)[i]);
}

__device__ __forceinline__ void store4(void* out, int odt, size_t o, int cols, f32x4 v) {
    // cols: how many of the four exist; o: the first one's index
    if (odt == DT_F32) {
        float* p = static_cast<float*>(out) + o;
        if (cols >= 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) *reinterpret_cast<f32x4*>(p) = v;
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) p[j] = v[j];
    } else {
        uint16_t* p = static_cast<uint16_t*>(out) + o;
        uint32_t d[2];
        if (odt == DT_BF16) d[0] = pack_bf16x2(v[0], v[1]), d[1] = pack_bf16x2(v[2], v[3]);
        else {
            d[0] = h_as_u16((_Float16)v[0]) | (h_as_u16((_Float16)v[1]) << 16);
            d[1] = h_as_u16((_Float16)v[2]) | (h_as_u16((_Float16)v[3]) << 16);
        }
        if (cols >= 4 && (reinterpret_cast<uintptr_t>(p) & 7) == 0) *reinterpret_cast<uint2*>(p) = make_uint2(d[0], d[1]);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) p[j] = (uint16_t)(d[j >> 1] >> (16 * (j & 1)));
    }
}

// The SwiGLU of the experts: g' = min(g, L), u' = clamp(u, -L, L) (iff L != 0), silu(g') u'. NaN operands stay NaN (the
// hardware's min and max drop them).
__device__ __forceinline__ float swiglu(float g, float u, float L) {
    if (L != 0.0f) {
        g = g > L ? L : g;
        u = u > L ? L : u < -L ? -L : u;
    }
    return __fdiv_rn(g, 1.0f + __expf(-g)) * u;
}

// Workgroup order: workgroups go round the 8 XCDs, each with an L2 of its own, so XCD x takes a contiguous run of tiles,
// in bands of `band` tile rows over all columns.
__device__ __forceinline__ int xcd_order(int id, int total) {
    const int x = id & 7, per = total >> 3, rest = total & 7;
    return x * per + min(x, rest) + (id >> 3);
}

// Dynamic LDS beyond 64 KB has to be allowed once per kernel and device.
template <typename F>
static bool allow_lds(F* f, int bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(f), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
}

}  // namespace mi355moe
