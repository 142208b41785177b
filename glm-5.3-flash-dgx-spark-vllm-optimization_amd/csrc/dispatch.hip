// Tokens sorted by expert, and back.
//
//   sort          the P = T topk pairs of a router's ids in the order (local expert, pair): row[pair] = the pair's place,
//                 pair[place] the inverse, offsets[e] the first place of expert e. What no local expert takes comes behind
//                 offsets[n], in pair order, and carries its place as ~place (negative): every row has one owner
//   to experts    rows[row[t, j]] = x[t]; rows behind offsets[n] are zero
//   from experts  out[t] = shared[t] + sum over j of w[t, j] rows[row[t, j]], j ascending, fp32, one rounding
//   gradients     of to experts: from experts without weights; of from experts: drows[row[t, j]] = w[t, j] dout[t],
//                 dw[t, j] = <dout[t], rows[row[t, j]]>
//
// Without atomics on values: two calls give the same bits.
#include <algorithm>
#include <climits>

#include "gemm_tile.cuh"
#include "rows.cuh"

namespace mi355moe {

// ------------------------------------------------------------------------------------------------ sort

constexpr int SORT_ONE = 4096;          // pairs that one workgroup sorts alone

template <typename IT>
__device__ __forceinline__ int sort_local(const SortArgs& a, int64_t i) {
    const int64_t id = (int64_t)static_cast<const IT*>(a.ids)[i];
    if (!a.emap) return id >= 0 && id < a.n ? (int)id : a.n;
    if (id < 0 || id >= a.n_global) return a.n;
    const int64_t l = a.emap[id];
    return l >= 0 && l < a.n ? (int)l : a.n;
}

// How many pairs of each workgroup's share (a.chunk of them) every expert takes: counts in LDS, whose atomics on whole numbers give the
// same sums in any order. Bound: latency (65536 pairs, 288 experts: 3 us; the ids are 0.25 MB).
template <typename IT>
__global__ __launch_bounds__(1024) void sort_count_kernel(SortArgs a) {
    extern __shared__ __align__(16) int cnt[];                       // [n + 1]
    const int n1 = a.n + 1;
    for (int e = threadIdx.x; e < n1; e += 1024) cnt[e] = 0;
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * a.chunk, p1 = min(a.P, p0 + a.chunk);
    for (int64_t p = p0 + threadIdx.x; p < p1; p += 1024) atomicAdd(&cnt[sort_local<IT>(a, p)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < n1; e += 1024) a.counts[(size_t)blockIdx.x * n1 + e] = cnt[e];
}

// The places of a workgroup's share. Its waves take runs of it one after the other; each counts its run's pairs by expert, the
// counts of the share and of the shares before it (all of them are read again by every workgroup: 128 x 289 words, from cache)
// give every wave the place of its first pair of each expert, and 64 pairs at a time the lanes of one expert find each
// other by ballots over the bits of its number, in pair order. The counts are taken twice (here and in the kernel before) rather than
// kept: that costs the ids' second read, from cache, where a wave's counts would cost sixteen times the workgroup's. Bound: the
// chain of loads, three barriers and the waves' steps, not the bytes: 8 pairs 4.2 us, 65536 pairs with 288 experts 8.6 us (0.8 MB).
template <typename IT>
__global__ __launch_bounds__(1024) void sort_place_kernel(SortArgs a, int blocks) {
    extern __shared__ __align__(16) int lds[];
    __shared__ int carry[16];
    const int n1 = a.n + 1, waves = blockDim.x >> 6;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int* start = lds;                                                // [n + 1]: pairs of each expert, then its first place
    int* at = lds + n1 + wv * n1;                                    // this wave's [n + 1]
    for (int e = threadIdx.x; e < waves * n1; e += blockDim.x) lds[n1 + e] = 0;
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * a.chunk, run = a.chunk / waves;      // (a multiple of 64)
    const int64_t w0 = p0 + wv * run, w1 = min(a.P, w0 + run);
    for (int64_t p = w0 + lane; p < w1; p += 64) atomicAdd(&at[sort_local<IT>(a, p)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < n1; e += blockDim.x) {
        int before = 0, all = 0;
        if (blocks > 1) {
#pragma unroll 8
            for (int b = 0; b < blocks; ++b) {
                const int c = a.counts[(size_t)b * n1 + e];
                before += b < (int)blockIdx.x ? c : 0;
                all += c;
            }
        }
        int sum = before;
        for (int w = 0; w < waves; ++w) {
            int& c = lds[n1 + w * n1 + e];
            const int v = c;
            c = sum;
            sum += v;
        }
        start[e] = blocks > 1 ? all : sum;
    }
    __syncthreads();
    // exclusive sums of start: the waves scan 64 entries each, workgroup by workgroup of them
    int base = 0;
    for (int e0 = 0; e0 < n1; e0 += blockDim.x) {
        const int e = e0 + threadIdx.x;
        const int v = e < n1 ? start[e] : 0;
        int s = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o, 64);
            s += lane >= o ? u : 0;
        }
        if (lane == 63) carry[wv] = s;
        __syncthreads();
        int before = base, total = 0;
        for (int w = 0; w < waves; ++w) {
            before += w < wv ? carry[w] : 0;
            total += carry[w];
        }
        if (e < n1) {
            start[e] = before + s - v;
            if (blockIdx.x == 0) a.offsets[e] = before + s - v;
        }
        base += total;
        __syncthreads();
    }
    const int bits = 32 - __builtin_clz((unsigned)a.n);              // (n >= 1: ids 0 .. n)
    for (int64_t q = w0; q < w1; q += 64) {                          // (uniform)
        const int64_t p = q + lane;
        const bool here = p < w1;
        const int l = here ? sort_local<IT>(a, p) : 0;
        uint64_t same = __ballot(here);
        for (int b = 0; b < bits; ++b) {
            const bool bit = (l >> b) & 1;
            const uint64_t m = __ballot(bit);
            same &= bit ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (here) {
            const int first = at[l], place = start[l] + first + rank;
            asm volatile("" ::: "memory");                           // (a wave's LDS accesses are performed in order: all lanes
            if (rank == 0) at[l] = first + __popcll(same);           // have read at[l] when the first one moves it on)
            const bool live = l < a.n;
            a.row[p] = live ? place : ~place;
            a.pair[place] = live ? (int)p : ~(int)p;
        }
        asm volatile("" ::: "memory");
    }
}

// Pairs of a workgroup: up to SORT_ONE one sorts alone (us alone / by eight: 4096 pairs 7.9 / -, 8192 12.0 / 7.9); else 1024, and in at
// most 128 workgroups, with many experts, whose counts each of them reads, in 32 (us by 128 / 64 / 32 workgroups, 288 experts: 65536
// pairs - / 10.9 / 10.5, 2^20 23.7 / 29 / 47; 4096 experts: 65536 - / 37.7 / 28.6, 2^18 62 / 46 / 44).
static int64_t sort_chunk(int64_t P, int64_t n) {
    if (P <= SORT_ONE) return std::max<int64_t>(1024, (P + 1023) / 1024 * 1024);
    const int64_t most = n <= 1024 ? 128 : 32;
    return ((P + most - 1) / most + 1023) / 1024 * 1024;
}
static int sort_blocks(int64_t P, int64_t n) { return P <= SORT_ONE ? 1 : (int)((P + sort_chunk(P, n) - 1) / sort_chunk(P, n)); }
int64_t sort_count_words(int64_t P, int64_t n) { return sort_blocks(P, n) > 1 ? sort_blocks(P, n) * (n + 1) : 0; }

template <typename IT>
static int run_sort(SortArgs a, hipStream_t st) {
    const int blocks = sort_blocks(a.P, a.n), n1 = a.n + 1;
    a.chunk = sort_chunk(a.P, a.n);
    if (blocks > 1) {
        hipLaunchKernelGGL(sort_count_kernel<IT>, dim3(blocks), dim3(1024), n1 * 4, st, a);
        if (hipGetLastError() != hipSuccess) return -1;
    }
    const int threads = n1 <= 2048 ? 1024 : 512;                     // a word per expert and wave in LDS, 160 KB at most
    const int bytes = (threads / 64 + 1) * n1 * 4;
    if (!allow_lds<sort_place_kernel<IT>>(160 * 1024 - 256)) return -1;
    hipLaunchKernelGGL(sort_place_kernel<IT>, dim3(blocks), dim3(threads), bytes, st, a, blocks);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_sort(const SortArgs& a, hipStream_t st) { return a.ids64 ? run_sort<int64_t>(a, st) : run_sort<int>(a, st); }

// ------------------------------------------------------------------------------------------------ rows

// The threads of a workgroup lie over 256 / lanes tokens and `lanes` = 2^shift of the 16-byte units of a row; the workgroups of a
// token's `segs` pieces follow one another. UNI: a wave has one token (lanes >= 64), whose table entries are then scalar.
struct RowsPlace {
    int64_t t;
    int unit;
};
template <bool UNI>
__device__ __forceinline__ RowsPlace rows_place(int shift, int segs) {
    const uint32_t i = wide_block(), g = i / (uint32_t)segs, seg = i - g * segs;
    const int64_t t = ((int64_t)g << (8 - shift)) + (threadIdx.x >> shift);
    return {UNI ? (int64_t)__builtin_amdgcn_readfirstlane((int)t) : t, (int)(seg << shift) + (int)(threadIdx.x & ((1 << shift) - 1))};
}

// rows[row] = x[t] (live) or zero, 16 bytes a thread and store; ES: bytes of a value. x is read once, whatever topk: a thread keeps
// its 16 bytes and stores them to each row. Bound: HBM, its writes above all (bf16 rows of 4096, top 8: 4096 tokens 302 MB in 50 to
// 59 us, 8192 in 106 to 116, 5.3 TB/s; 4096 in fp32 604 MB in 106 to 117).
template <int ES, bool UNI>
__global__ __launch_bounds__(256) void rows_scatter_kernel(RowsArgs a, int shift, int segs) {
    const auto [t, u] = rows_place<UNI>(shift, segs);
    const int RB = a.H * ES, b = u * 16;                             // bytes of a row, and this thread's first
    if (t >= a.T || b >= RB) return;
    const int left = min(16, RB - b);
    const unsigned char* src = static_cast<const unsigned char*>(a.x) + (size_t)t * a.x_stride * ES + b;
    u32x4 v = {0, 0, 0, 0};
    if (left == 16) v = *reinterpret_cast<const rows_u32x4*>(src);
    else
        for (int i = 0; i < left; i += 2) v[i >> 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + i) << (8 * (i & 2));
    const int* row = a.row + t * a.topk;
    for (int j = 0; j < a.topk; ++j) {
        const int r = row[j];
        const int64_t to = r < 0 ? ~r : r;
        if (to >= a.P) continue;                                     // (a table that the sort did not make)
        unsigned char* dst = static_cast<unsigned char*>(a.rows) + (size_t)to * RB + b;
        const u32x4 o = r < 0 ? u32x4{0, 0, 0, 0} : v;
        if (left == 16) *reinterpret_cast<rows_u32x4*>(dst) = o;
        else
            for (int i = 0; i < left; i += 2) *reinterpret_cast<uint16_t*>(dst + i) = (uint16_t)(o[i >> 2] >> (8 * (i & 2)));
    }
}

// The next N live slots' rows, requested together, then added in order.
template <int DT, bool ONCE, int N>
__device__ __forceinline__ void add_rows(const RowsArgs& a, uint64_t& live, int rv, float wv, int c, int n, float (&acc)[8]) {
    Raw8<DT> v[N];
    float w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int j = __builtin_ctzll(live);
        live &= live - 1;
        v[k].template load<ONCE>(a.rows, (size_t)__builtin_amdgcn_readlane(rv, j) * a.H + c, n);
        w[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wv), j));
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        float x[8];
        v[k].get(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(w[k], x[i], acc[i]);
    }
}

// out[t] = shared[t] + the weighted rows of t, eight values a thread. A wave's lanes read the table entries of its token's slots
// (at most 32), and the rows of up to eight slots are on their way at once; rows of fewer than 64 pieces share a wave, and each
// thread reads the table itself. Bound: HBM (bf16 rows of 4096, top 8, 4096 tokens with shared: 336 MB in 58 to 70 us, 5.2 TB/s; in
// fp32 671 MB in 128 to 145); a few hundred tokens: latency (517 tokens of 2051, top 6, fp16: 5.3 us).
template <int DT, bool UNI, bool ONCE>
__global__ __launch_bounds__(256) void rows_gather_kernel(RowsArgs a, int shift, int segs) {
    const auto [t, u] = rows_place<UNI>(shift, segs);
    const int c = u * 8, n = min(8, a.H - c);
    if (t >= a.T || (!UNI && n <= 0)) return;
    float acc[8] = {};
    Raw8<DT> sh;
    if (a.shared) sh.load(a.shared, (size_t)t * a.shared_stride + c, n);
    if constexpr (UNI) {
        const int lane = threadIdx.x & 63;
        const int64_t p = t * a.topk + min(lane, a.topk - 1);
        const int rv = lane < a.topk ? a.row[p] : -1;
        const float wv = a.w ? any_value(a.w, a.wdt, p) : 1.0f;
        uint64_t live = __ballot(rv >= 0 && rv < a.P);
        if (a.shared) sh.get(acc);
        int left = __popcll(live);
        for (; left >= 8; left -= 8) add_rows<DT, ONCE, 8>(a, live, rv, wv, c, n, acc);
        if (left & 4) add_rows<DT, ONCE, 4>(a, live, rv, wv, c, n, acc);
        if (left & 2) add_rows<DT, ONCE, 2>(a, live, rv, wv, c, n, acc);
        if (left & 1) add_rows<DT, ONCE, 1>(a, live, rv, wv, c, n, acc);
    } else {
        if (a.shared) sh.get(acc);
        for (int j = 0; j < a.topk; ++j) {
            const int64_t p = t * a.topk + j;
            const int r = a.row[p];
            if (r < 0 || r >= a.P) continue;
            const float w = a.w ? any_value(a.w, a.wdt, p) : 1.0f;
            float v[8];
            load8<DT>(a.rows, (size_t)r * a.H + c, n, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(w, v[i], acc[i]);
        }
    }
    store8<DT>(a.out, (size_t)t * a.out_stride + c, n, acc);
}

// drows and dw of the next N live slots of token t.
template <int DT, bool ONCE, int N>
__device__ __forceinline__ void grad_rows(const RowsArgs& a, int64_t t, uint64_t& live, int rv, float wv, float (*red)[4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int slot[N];
    size_t row[N];
    float w[N], dot[N] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) {
        slot[k] = __builtin_ctzll(live);
        live &= live - 1;
        row[k] = (size_t)__builtin_amdgcn_readlane(rv, slot[k]) * a.H;
        w[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wv), slot[k]));
    }
    for (int c = threadIdx.x * 8; c < a.H; c += blockDim.x * 8) {
        const int n = a.H - c;
        Raw8<DT> d8, y8[N];
        d8.load(a.x, (size_t)t * a.x_stride + c, n);
        if (a.dw)                                                    // (uniform)
#pragma unroll
            for (int k = 0; k < N; ++k) y8[k].template load<ONCE>(a.y, row[k] + c, n);
        float d[8];
        d8.get(d);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float v[8];
            if (a.dw) {
                y8[k].get(v);
#pragma unroll
                for (int i = 0; i < 8; ++i) dot[k] = __builtin_fmaf(d[i], v[i], dot[k]);
            }
            if (a.rows) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = w[k] * d[i];
                store8<DT>(a.rows, row[k] + c, n, v);
            }
        }
    }
    if (!a.dw) return;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        dot[k] = wave_sum(dot[k]);
        if (lane == 0) red[k][wave] = dot[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
        if ((int)threadIdx.x == k) {
            float s = 0.0f;
            for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[k][i];
            store_any(a.dw, a.wdt, t * a.topk + slot[k], s);
        }
    __syncthreads();                                                 // (the sums have been read: the next slots write them)
}

// A workgroup a token: dout[t] is read once for eight slots, whose rows are on their way at once; at most four waves. The dots are
// sums of a thread, a wave (by lane exchanges) and the waves in order. Bound: HBM (bf16 rows of 4096, top 8, 4096 tokens: 571 MB in
// 113 to 118 us, 4.9 TB/s; in fp32 1142 MB in 234 to 240).
template <int DT, bool ONCE>
__global__ __launch_bounds__(256) void rows_grad_kernel(RowsArgs a) {
    __shared__ float red[8][4];
    const int64_t t = wide_block();
    if (t >= a.T) return;                                            // (uniform)
    const int lane = threadIdx.x & 63;
    const int64_t p = t * a.topk + min(lane, a.topk - 1);
    const int rv = lane < a.topk ? a.row[p] : INT_MAX;
    const float wv = any_value(a.w, a.wdt, p);
    uint64_t live = __ballot(rv >= 0 && rv < a.P), dead = __ballot(rv < 0 && ~rv < a.P);      // (the same in every wave)
    if (a.dw && threadIdx.x < 64 && (dead >> lane & 1)) store_any(a.dw, a.wdt, p, 0.0f);
    if (a.rows)
        for (; dead; dead &= dead - 1) {
            const size_t row = (size_t)~__builtin_amdgcn_readlane(rv, __builtin_ctzll(dead)) * a.H;
            const float zero[8] = {};
            for (int c = threadIdx.x * 8; c < a.H; c += blockDim.x * 8) store8<DT>(a.rows, row + c, a.H - c, zero);
        }
    int left = __popcll(live);
    for (; left >= 8; left -= 8) grad_rows<DT, ONCE, 8>(a, t, live, rv, wv, red);
    if (left & 4) grad_rows<DT, ONCE, 4>(a, t, live, rv, wv, red);
    if (left & 2) grad_rows<DT, ONCE, 2>(a, t, live, rv, wv, red);
    if (left & 1) grad_rows<DT, ONCE, 1>(a, t, live, rv, wv, red);
}

// log2 of the threads on a row of `units` pieces: all of them, 8 to 256.
static int row_shift(int64_t units) {
    int s = 3;
    while (s < 8 && (1 << s) < units) ++s;
    return s;
}
// (at most 64 pieces of 2^24 tokens)
static dim3 rows_grid(int64_t T, int shift, int segs) { return wide_grid((T + (256 >> shift) - 1) / (256 >> shift) * segs); }

template <int ES>
static int run_scatter(const RowsArgs& a, hipStream_t st) {
    const int units = (a.H * ES + 15) / 16, s = row_shift(units), segs = (units + (1 << s) - 1) >> s;
    const dim3 g = rows_grid(a.T, s, segs);
    if (s >= 6) hipLaunchKernelGGL((rows_scatter_kernel<ES, true>), g, dim3(256), 0, st, a, s, segs);
    else hipLaunchKernelGGL((rows_scatter_kernel<ES, false>), g, dim3(256), 0, st, a, s, segs);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_rows_scatter(const RowsArgs& a, hipStream_t st) { return a.dt == DT_F32 ? run_scatter<4>(a, st) : run_scatter<2>(a, st); }

// Rows of 64 MB and more are marked as read once. us plain / marked, bf16 rows of 4096, top 8: gather, 512 tokens (34 MB) 8.7 / 8.7, 1024
// 21 / 15.6, 4096 79 / 59, 8192 130 / 106; gradient, 512 17.8 / 18.6, and after a gather that left nothing of them in the caches,
// as in a training step, 2048 75 / 60, 4096 136 / 116.
static bool rows_once(const RowsArgs& a) { return a.P * a.H * (a.dt == DT_F32 ? 4 : 2) >= (64 << 20); }

template <int DT>
static int run_gather(const RowsArgs& a, hipStream_t st) {
    const int units = (a.H + 7) / 8, s = row_shift(units), segs = (units + (1 << s) - 1) >> s;
    const dim3 g = rows_grid(a.T, s, segs);
    if (s >= 6 && rows_once(a)) hipLaunchKernelGGL((rows_gather_kernel<DT, true, true>), g, dim3(256), 0, st, a, s, segs);
    else if (s >= 6) hipLaunchKernelGGL((rows_gather_kernel<DT, true, false>), g, dim3(256), 0, st, a, s, segs);
    else hipLaunchKernelGGL((rows_gather_kernel<DT, false, false>), g, dim3(256), 0, st, a, s, segs);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_rows_gather(const RowsArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_gather<DT_F32>(a, st) : a.dt == DT_BF16 ? run_gather<DT_BF16>(a, st) : run_gather<DT_F16>(a, st);
}

template <int DT>
static int run_rows_grad(const RowsArgs& a, hipStream_t st) {
    const dim3 g = wide_grid(a.T), b(std::min(256, (a.H + 511) / 512 * 64));
    if (rows_once(a)) hipLaunchKernelGGL((rows_grad_kernel<DT, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((rows_grad_kernel<DT, false>), g, b, 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_rows_grad(const RowsArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_rows_grad<DT_F32>(a, st) : a.dt == DT_BF16 ? run_rows_grad<DT_BF16>(a, st) : run_rows_grad<DT_F16>(a, st);
}

}  // namespace mi355moe
