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
//   ROW  the contraction is contiguous: LDS holds row R's 16-byte chunks, chunk g at slot g ^ row_swz(R): sixteen
//        consecutive rows' chunk g lie in sixteen different 16-byte columns of the banks
//   COL  the contraction is the row index (16-bit only): LDS holds 64 rows of R values; a fragment is two
//        ds_read_b64_tr_b16, each of which hands lane i of 16 column i of a 4 x 16 block. Consecutive rows are whole
//        bank rounds apart, so the 32-byte segments of row k are rotated (xor) by k's place among the rows that one
//        read touches.
// Both swizzles are applied through the load addresses.
#pragma once
#include <atomic>

#include "common.cuh"
#include "mi355moe_internal.h"

namespace mi355moe {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Keeps the compiler from moving anything across: the loops below are scheduled by hand.
#define SCHED_FENCE() __builtin_amdgcn_sched_barrier(0)

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
// the xor of row k's 32-byte segment index (R values a row): distinct over the rows one transposing read touches (k & 3 in
// both halves of the stage), as far as the row's segments go
template <int R>
__device__ __forceinline__ int col_swz(int k) {
    if constexpr (R >= 256) return ((k & 3) | ((k >> 3) & 4)) << 1;
    else if constexpr (R == 128) return (k & 3) << 1;
    else return ((k >> 1) & 1) << 1;
}
constexpr int SB = 128;                              // bytes of a row in a stage

// Staging of one operand of R rows (LAY_COL: R columns) by NW waves.
template <int LAY, int R, int NW>
struct Stager {
    static constexpr int CH = SB / 16;               // chunks of a row (ROW)
    static constexpr int KR = SB / 2;                // rows of a stage (COL)
    static constexpr int INST = R * SB / 1024 / NW;  // 1 KB wave instructions per stage and wave
    static_assert(INST * 1024 * NW == R * SB, "the stage divides over the waves");
    const unsigned char* base;                       // wave-uniform
    uint32_t off[INST];                              // this lane's source bytes of each instruction
    int lds;                                         // this wave's first byte of the operand's stage

    // the place (in 16 bytes) that instruction j of this lane fills
    static __device__ __forceinline__ int place(int wv, int j, int lane) { return (wv * INST + j) * 64 + lane; }
    // ROW: rowoff(R) = byte offset of tile row R from `b`
    template <typename F>
    __device__ __forceinline__ void init_row(const void* b, int wv, int lane, const F& rowoff) {
        static_assert(LAY == LAY_ROW, "");
        base = static_cast<const unsigned char*>(b);
        lds = wv * INST * 1024;
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            const int r = place(wv, j, lane) / CH;
            off[j] = rowoff(r) + (((lane & (CH - 1)) ^ row_swz(r)) << 4);
        }
    }
    // COL: row k at ld * k bytes; `cols` values of the row from `b` on may be read (a multiple of 8)
    __device__ __forceinline__ void init_col(const void* b, int wv, int lane, uint32_t ld, int cols) {
        static_assert(LAY == LAY_COL, "");
        base = static_cast<const unsigned char*>(b);
        lds = wv * INST * 1024;
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            const int p = place(wv, j, lane), k = p / (R / 8), c = p % (R / 8);
            const int col = (((c >> 1) ^ col_swz<R>(k)) << 4) + ((c & 1) << 3);
            off[j] = (uint32_t)k * ld + 2u * (uint32_t)min(col, cols - 8);
        }
    }
    __device__ __forceinline__ void issue(unsigned char* st, int j) const { dma16_base(base, off[j], st + lds + j * 1024); }
    // from here on the stage being requested is the last one, of which only `valid` chunks (ROW) or rows (COL, of ld bytes)
    // exist: what lies behind them is loaded from the last one that exists (and cleared in LDS by clear_tail)
    __device__ __forceinline__ void to_tail(int wv, int lane, int valid, uint32_t ld) {
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            if constexpr (LAY == LAY_ROW) {
                const int g = (lane & (CH - 1)) ^ row_swz(place(wv, j, lane) / CH);
                if (g >= valid) off[j] -= (uint32_t)(g - valid + 1) << 4;
            } else {
                const int k = place(wv, j, lane) / (R / 8);
                if (k >= valid) off[j] -= (uint32_t)(k - valid + 1) * ld;
            }
        }
    }
    static __device__ __forceinline__ void clear_tail(unsigned char* st, int tid, int valid) {
        const u32x4 z = {0, 0, 0, 0};
        if constexpr (LAY == LAY_ROW) {
            for (int i = tid; i < R * CH; i += NW * 64) {
                const int r = i / CH, g = i % CH;
                if (g >= valid) *reinterpret_cast<u32x4*>(st + r * SB + ((g ^ row_swz(r)) << 4)) = z;
            }
        } else {
            for (int i = valid * (R / 8) + tid; i < KR * (R / 8); i += NW * 64) *reinterpret_cast<u32x4*>(st + i * 16) = z;
        }
    }
};

// The 16 bytes (lane r = lane % 32, half h) of step s of the 32-row tile at row r0.
template <int LAY, int R>
__device__ __forceinline__ u32x4 fragment(const unsigned char* st, int r0, int s, int lane) {
    const int c = SB / 32 * (lane >> 5) + s;
    if constexpr (LAY == LAY_ROW) {
        const int r = r0 + (lane & 31);
        return *reinterpret_cast<const u32x4*>(st + r * SB + ((c ^ row_swz(r)) << 4));
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

// Scale dwords of an MXFP4 operand: a stage holds 8 bytes of each row's scales (the dword of half h at 4h), 256 bytes (32
// rows) a wave instruction of 4 bytes a lane. Row R's scales of stage kb lie at rowoff(R) + kb * step: back to back for the
// rows of a tile where the scales were arranged by steps; in rows of K / 32 bytes they touch as many lines as the stage's
// codes do, for a sixteenth of the bytes.
template <int R, int NW>
struct ScaleStager {
    static constexpr int INST = (R / 32 + NW - 1) / NW;
    const unsigned char* base;
    uint32_t step;
    uint32_t off[INST];
    uint32_t last[INST];                             // the row's last dword (rows of an odd number of them end in mid-stage)
    int lds[INST];
    template <typename F>
    __device__ __forceinline__ void init(const MxScales& s, size_t row0, int dwords, int wv, int lane, const F& row) {
        base = s.p + row0 * s.row;
        step = s.step;
#pragma unroll
        for (int j = 0; j < INST; ++j) {
            const int blk = min(wv * INST + j, R / 32 - 1);          // (waves past the rows repeat the last block)
            const uint32_t r = row(blk * 32 + (lane >> 1)) * s.row;
            off[j] = r + ((lane & 1) << 2);
            last[j] = s.step == 8 ? r + 4u * (uint32_t)(dwords - 1) : 0xFFFFFFFFu;
            lds[j] = blk * 256;
        }
    }
    __device__ __forceinline__ void issue(unsigned char* st, int kb, int j) const {
        dma4(base + min(off[j] + step * (uint32_t)kb, last[j]), st + lds[j]);
    }
    static __device__ __forceinline__ int read(const unsigned char* st, int r0, int lane) {
        return *reinterpret_cast<const int*>(st + (r0 + (lane & 31)) * 8 + ((lane >> 5) << 2));
    }
};

// One workgroup's product. AHEAD (MXFP4): the caller has put the scales of all stages behind the stages, 8 bytes of each P
// and Q row a stage, before run().
template <int MM_, int PL_, int QL_, int BP_, int BQ_, int WP_, int WQ_, int STAGES_, bool AHEAD = false>
struct GemmTile {
    static constexpr int MM = MM_, PL = PL_, QL = QL_, BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, STAGES = STAGES_;
    static constexpr int NW = WP * WQ, THREADS = 64 * NW;
    static constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32;      // 32 x 32 tiles of a wave
    static constexpr bool MX = MM == MM_MX4;
    static constexpr int QOFF = BP * SB, SCL = (BP + BQ) * SB;       // a stage's P rows, Q rows, P scales, Q scales
    static constexpr int XB = MX ? (BP + BQ) * 8 : 0;                // scale bytes of a stage
    static constexpr int STAGE = SCL + (AHEAD ? 0 : XB), LDS = STAGES * STAGE;
    static constexpr int KSTAGE = MX ? 256 : 64;                     // contraction values of a stage
    using SP = Stager<PL, BP, NW>;
    using SQ = Stager<QL, BQ, NW>;
    using XP = ScaleStager<BP, NW>;
    using XQ = ScaleStager<BQ, NW>;
    static constexpr int LOADS = SP::INST + SQ::INST + (MX && !AHEAD ? XP::INST + XQ::INST : 0);   // of a stage and wave

    SP p;
    SQ q;
    XP xp;
    XQ xq;
    f32x16 acc[TP][TQ];

    // What one step of a stage multiplies, held in registers one step ahead.
    struct Frags {
        u32x4 a[TP], b[TQ];
    };
    struct Scales {
        int p[TP], q[TQ];
    };
    template <int S>
    __device__ __forceinline__ void fetch(const unsigned char* st, int p0, int q0, int lane, Frags& f) const {
#pragma unroll
        for (int i = 0; i < TP; ++i) f.a[i] = fragment<PL, BP>(st, p0 + 32 * i, S, lane);
#pragma unroll
        for (int j = 0; j < TQ; ++j) f.b[j] = fragment<QL, BQ>(st + QOFF, q0 + 32 * j, S, lane);
    }
    // (st: the stage, the rel-th of those this workgroup multiplies, whose first lies at lds)
    __device__ __forceinline__ void fetch_scales(const unsigned char* lds, const unsigned char* st, int rel, int p0, int q0,
                                                 int lane, Scales& x) const {
        if constexpr (MX) {
            const unsigned char* sc = AHEAD ? lds + LDS + rel * XB : st + SCL;
#pragma unroll
            for (int i = 0; i < TP; ++i) x.p[i] = XP::read(sc, p0 + 32 * i, lane);
#pragma unroll
            for (int j = 0; j < TQ; ++j) x.q[j] = XQ::read(sc + BP * 8, q0 + 32 * j, lane);
        }
    }
    // after(i): called behind the i-th of the step's TP TQ multiplications, in this order
    template <int S, typename After>
    __device__ __forceinline__ void multiply(const Frags& f, const Scales& x, const After& after) {
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int j = 0; j < TQ; ++j) {
                if constexpr (MX) acc[i][j] = mma_mx<S>(f.a[i], f.b[j], acc[i][j], x.p[i], x.q[j]);
                else acc[i][j] = mma16(std::integral_constant<int, MM>{}, f.a[i], f.b[j], acc[i][j]);
                // the sums pass through here: otherwise the compiler is free to gather several steps' multiplications
                asm volatile("" : "+v"(acc[i][j]));
                after(i * TQ + j);
            }
    }
    // Load i of the LOADS that stage kb takes (the scales', then P's, then Q's), to `st`.
    __device__ __forceinline__ void load(unsigned char* st, int kb, int i) const {
        constexpr int NX = MX && !AHEAD ? XP::INST : 0, NY = MX && !AHEAD ? NX + XQ::INST : 0;
        if (i < NX) xp.issue(st + SCL, kb, i);
        else if (i < NY) xq.issue(st + SCL + BP * 8, kb, i - NX);
        else if (i < NY + SP::INST) p.issue(st, i - NY);
        else q.issue(st + QOFF, i - NY - SP::INST);
    }
    // Stages kb0 .. kb1 - 1 of the contraction (kb0 < kb1; p.base and q.base at stage kb0). tail_p / tail_q: what the
    // last one holds of each operand (8-value chunks or MXFP4 blocks for ROW, rows for COL; 0: it is whole). ldp / ldq:
    // row bytes of COL operands. One barrier a stage, before its last step: by then every wave has read the stage's last
    // fragments, so its buffer can be refilled, and the next stage has landed, so its first fragments are read while the
    // last step multiplies. The refill's loads are spread over the multiplications of the next stage's first
    // two steps: issued together they hold the waves up at the address pipeline while the matrix cores idle.
    __device__ __forceinline__ void run(unsigned char* lds, int kb0, int kb1, int tail_p, int tail_q, uint32_t ldp,
                                        uint32_t ldq) {
        const int tid = threadIdx.x, lane = tid & 63;
        const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int p0 = (wv % WP) * (BP / WP), q0 = (wv / WP) * (BQ / WQ);
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int j = 0; j < TQ; ++j) acc[i][j] = f32x16{};
        const uint64_t advp = PL == LAY_ROW ? SB : SB / 2 * (uint64_t)ldp, advq = QL == LAY_ROW ? SB : SB / 2 * (uint64_t)ldq;
        int next = kb0;                                              // the stage that is being requested
        auto start = [&]() {                                         // before its first load
            if (next == kb1 - 1 && tail_p) {                         // (uniform)
                p.to_tail(wv, lane, tail_p, ldp);
                q.to_tail(wv, lane, tail_q, ldq);
            }
        };
        auto done = [&]() {                                          // behind its last one
            p.base += advp;
            q.base += advq;
            ++next;
        };
        // stage kb has landed for every wave, and nobody reads the stage before it any more
        auto arrive = [&](unsigned char* st, int kb) {
            if (STAGES > 2 && kb + STAGES - 2 < kb1) WAIT_VM((STAGES - 2) * LOADS);   // (the stages after it are on their way)
            else WAIT_VM(0);
            LDS_BARRIER();
            if (kb == kb1 - 1 && tail_p) {                           // (uniform)
                SP::clear_tail(st, tid, tail_p);
                SQ::clear_tail(st + QOFF, tid, tail_q);
                __syncthreads();
            }
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s)
            if (next < kb1) {
                start();
#pragma unroll
                for (int i = 0; i < LOADS; ++i) load(lds + s * STAGE, next, i);
                done();
            }
        Frags f0, f1;
        Scales x0, x1;
        int cur = 0;
        unsigned char* fill = lds + (STAGES - 1) * STAGE;            // where the requested stage goes
        arrive(lds, kb0);
        fetch_scales(lds, lds, 0, p0, q0, lane, x0);
        fetch<0>(lds, p0, q0, lane, f0);
        auto nothing = [](int) {};
        // a stage's steps, the next one's fragments read while each multiplies; REQ: with the loads of stage `next`
        auto stage = [&](auto REQ, auto LAST, int kb) {
            constexpr bool req = decltype(REQ)::value, last_stage = decltype(LAST)::value;
            constexpr int M = TP * TQ;
            const unsigned char* st = lds + cur * STAGE;
            // loads [LOADS at / (2 M), LOADS (at + 1) / (2 M)) behind multiplication `at` of the window's 2 M
            auto loads = [&](int at) {
                if constexpr (req) {
#pragma unroll
                    for (int i = LOADS * at / (2 * M); i < LOADS * (at + 1) / (2 * M); ++i) load(fill, next, i);
                    SCHED_FENCE();
                }
            };
            if constexpr (req) start();
            fetch<1>(st, p0, q0, lane, f1);
            SCHED_FENCE();
            multiply<0>(f0, x0, [&](int i) { loads(i); });
            SCHED_FENCE();
            fetch<2>(st, p0, q0, lane, f0);
            SCHED_FENCE();
            multiply<1>(f1, x0, [&](int i) { loads(M + i); });
            if constexpr (req) done();
            SCHED_FENCE();
            fetch<3>(st, p0, q0, lane, f1);
            SCHED_FENCE();
            multiply<2>(f0, x0, nothing);
            SCHED_FENCE();
            if constexpr (!last_stage) {
                fill = lds + cur * STAGE;
                cur = cur + 1 == STAGES ? 0 : cur + 1;
                unsigned char* nx = lds + cur * STAGE;
                arrive(nx, kb + 1);
                fetch_scales(lds, nx, kb + 1 - kb0, p0, q0, lane, x1);
                fetch<0>(nx, p0, q0, lane, f0);
                SCHED_FENCE();
            }
            multiply<3>(f1, x0, nothing);
            SCHED_FENCE();
            if constexpr (MX && !last_stage) x0 = x1;
        };
        int kb = kb0;
        for (; next < kb1; ++kb) stage(std::true_type{}, std::false_type{}, kb);
        for (; kb + 1 < kb1; ++kb) stage(std::false_type{}, std::false_type{}, kb);
        stage(std::false_type{}, std::true_type{}, kb);
    }

    // Stores TN x 32 columns of 16-bit (V gives a uint2) or fp32 values (V gives a f32x4) in whole rows: value(i, j, r) =
    // columns 8 r + 4 h .. + 3 of column tile i and row tile j. Through LDS, 32 rows of the wave at a time, 16 bytes a lane
    // and whole lines a row. `out` at the wave's first row and column, at 16-byte addresses; cols (a multiple of 8): the
    // columns that exist from there on; exists(row): whether the wave's row does. Called by all waves after run(). (8192 x
    // 4096 bf16: 17 us of 8-byte stores straight from the accumulators.)
    template <int TN, typename T, typename E, typename V>
    __device__ __forceinline__ void store_rows(unsigned char* lds, T* out, int64_t stride, int cols, const E& exists,
                                               const V& value) const {
        constexpr int ES = sizeof(T), UNITS = TN * 2 * ES;           // 16-byte units of a row
        static_assert(ES == 2 || ES == 4, "");
        const int lane = threadIdx.x & 63, h = lane >> 5;
        const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        unsigned char* mine = lds + wv * (32 * 16 * UNITS);
        static_assert(NW * 32 * 16 * UNITS <= LDS, "the stages hold the waves' rows");
        __syncthreads();                                             // no wave reads a stage any more
#pragma unroll
        for (int j = 0; j < TQ; ++j) {
            const int m = lane & 31;
            unsigned char* row = mine + m * (16 * UNITS);
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (ES == 2)
                        *reinterpret_cast<uint2*>(row + (((4 * i + r) ^ (m & (UNITS - 1))) << 4) + 8 * h) = value(i, j, r);
                    else *reinterpret_cast<f32x4*>(row + (((8 * i + 2 * r + h) ^ (m & (UNITS - 1))) << 4)) = value(i, j, r);
                }
            asm volatile("" ::: "memory");                           // (a wave's LDS accesses are performed in order)
#pragma unroll
            for (int t = 0; t < UNITS / 2; ++t) {
                const int at = t * 64 + lane, rr = at / UNITS, u = at % UNITS;
                const u32x4 v = *reinterpret_cast<const u32x4*>(mine + rr * (16 * UNITS) + ((u ^ (rr & (UNITS - 1))) << 4));
                if (exists(32 * j + rr) && 16 / ES * u < cols)
                    *reinterpret_cast<u32x4*>(out + (32 * j + rr) * stride + 16 / ES * u) = v;
            }
            asm volatile("" ::: "memory");
        }
    }
};

// Row (n) of accumulator register r: 8 (r / 4) + 4 (lane / 32) + r % 4; column (m): lane % 32.

__device__ __forceinline__ float load_value(const void* x, int xdt, size_t i) {
    if (xdt == DT_F32) return reinterpret_cast<const float*>(x)[i];
    if (xdt == DT_BF16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(x)[i]);
    return (float)u16_as_h(reinterpret_cast<const uint16_t*>(x)[i]);
}

__device__ __forceinline__ uint2 pack4(int odt, float a, float b, float c, float d) {
    if (odt == DT_BF16) return make_uint2(pack_bf16x2(a, b), pack_bf16x2(c, d));
    return make_uint2(h_as_u16((_Float16)a) | (h_as_u16((_Float16)b) << 16), h_as_u16((_Float16)c) | (h_as_u16((_Float16)d) << 16));
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

// The tile (column n, row m) of a workgroup among nt x mt. Workgroups go round the 8 XCDs, each with an L2 of its own: XCD
// x takes a contiguous run of tiles, in bands of four tile rows, down each column of a band first, so that what it has in
// flight is about square and reads the fewest different rows of both operands.
__device__ __forceinline__ int2 tile_order(int id, int nt, int mt) {
    const int total = nt * mt, x = id & 7, per = total >> 3, rest = total & 7;
    const int pos = x * per + min(x, rest) + (id >> 3);
    const int band = pos / (4 * nt), in = pos - band * 4 * nt, rows = min(4, mt - 4 * band);
    return make_int2(in / rows, 4 * band + in % rows);
}

// Dynamic LDS beyond 64 KB has to be allowed once per kernel and device (more than 64 devices: every time).
template <auto Kernel>
static bool allow_lds(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return true;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
        return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

}  // namespace mi355moe
