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

#include "gemm_tile.cuh"
#include "rows.cuh"

namespace mi355moe {

// ------------------------------------------------------------------------------------------------ sort

constexpr int SORT_ONE = 4096;          // pairs that one workgroup sorts alone
constexpr int SORT_BLOCKS = 128;        // most workgroups of a call

template <typename IT>
__device__ __forceinline__ int sort_local(const SortArgs& a, int64_t i) {
    const int64_t id = (int64_t)static_cast<const IT*>(a.ids)[i];
    if (!a.emap) return id >= 0 && id < a.n ? (int)id : a.n;
    if (id < 0 || id >= a.n_global) return a.n;
    const int64_t l = a.emap[id];
    return l >= 0 && l < a.n ? (int)l : a.n;
}

// How many pairs of each workgroup's share (a.chunk of them) every expert takes.
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
// other by ballots over the bits of its number, in pair order. Bound: latency, ...
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

static int64_t sort_chunk(int64_t P) {
    if (P <= SORT_ONE) return std::max<int64_t>(1024, (P + 1023) / 1024 * 1024);
    return std::max<int64_t>(1024, ((P + SORT_BLOCKS - 1) / SORT_BLOCKS + 1023) / 1024 * 1024);
}
static int sort_blocks(int64_t P) { return P <= SORT_ONE ? 1 : (int)((P + sort_chunk(P) - 1) / sort_chunk(P)); }
int64_t sort_count_words(int64_t P, int64_t n) { return sort_blocks(P) > 1 ? sort_blocks(P) * (n + 1) : 0; }

template <typename IT>
static int run_sort(SortArgs a, hipStream_t st) {
    const int blocks = sort_blocks(a.P), n1 = a.n + 1;
    a.chunk = sort_chunk(a.P);
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

// The threads of a workgroup lie over 256 / lanes tokens, `lanes` (a power of two) over the 16-byte units of a row; UNI: a wave
// has one token (lanes >= 64), whose table entries are then scalar.
template <bool UNI>
__device__ __forceinline__ int64_t token_of(int shift) {
    const int64_t t = ((int64_t)blockIdx.x << (8 - shift)) + (threadIdx.x >> shift);
    if constexpr (UNI) return __builtin_amdgcn_readfirstlane((int)t);
    else return t;
}

// rows[row] = x[t] (live) or zero, 16 bytes a thread and store; ES: bytes of a value.
template <int ES, bool UNI>
__global__ __launch_bounds__(256) void rows_scatter_kernel(RowsArgs a, int shift) {
    const int64_t t = token_of<UNI>(shift);
    const int64_t u = ((int64_t)blockIdx.y << shift) + (threadIdx.x & ((1 << shift) - 1));
    const int64_t RB = (int64_t)a.H * ES;                            // bytes of a row
    const int64_t b = u * 16;
    if (t >= a.T || b >= RB) return;
    const int left = (int)min((int64_t)16, RB - b);
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

// out[t] = shared[t] + the weighted rows of t, eight values a thread.
template <int DT, bool UNI>
__global__ __launch_bounds__(256) void rows_gather_kernel(RowsArgs a, int shift) {
    const int64_t t = token_of<UNI>(shift);
    const int64_t c = (((int64_t)blockIdx.y << shift) + (threadIdx.x & ((1 << shift) - 1))) * 8;
    const int n = (int)min((int64_t)8, a.H - c);
    if (t >= a.T || n <= 0) return;
    float acc[8] = {};
    if (a.shared) load8<DT>(a.shared, (size_t)t * a.shared_stride + c, n, acc);
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
    store8<DT>(a.out, (size_t)t * a.out_stride + c, n, acc);
}

// drows and dw of one pair a wave: the waves of a workgroup are neighbours, mostly slots of one token.
template <int DT>
__global__ __launch_bounds__(256) void rows_grad_kernel(RowsArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t p = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (p >= a.P) return;
    const int r = a.row[p];
    const int64_t to = r < 0 ? ~r : r, t = p / a.topk;
    if (to >= a.P) return;
    const float w = r < 0 ? 0.0f : any_value(a.w, a.wdt, p);
    float dot = 0.0f;
    for (int c = lane * 8; c < a.H; c += 512) {
        const int n = a.H - c;
        float d[8] = {}, y[8];
        if (r >= 0) {                                                // (uniform)
            load8<DT>(a.x, (size_t)t * a.x_stride + c, n, d);
            if (a.dw) {
                load8<DT>(a.y, (size_t)to * a.H + c, n, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(d[i], y[i], dot);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] *= w;
        }
        if (a.rows) store8<DT>(a.rows, (size_t)to * a.H + c, n, d);
    }
    if (a.dw) {
        dot = wave_sum(dot);
        if (lane == 0) store_any(a.dw, a.wdt, p, dot);
    }
}

// log2 of the threads on a row of `units` pieces: all of them, 8 to 256.
static int row_shift(int64_t units) {
    int s = 3;
    while (s < 8 && (1 << s) < units) ++s;
    return s;
}

template <int ES>
static int run_scatter(const RowsArgs& a, hipStream_t st) {
    const int64_t units = ((int64_t)a.H * ES + 15) / 16;
    const int s = row_shift(units), per = 256 >> s;
    const dim3 g((unsigned)((a.T + per - 1) / per), (unsigned)((units + (1 << s) - 1) >> s));
    if (s >= 6) hipLaunchKernelGGL((rows_scatter_kernel<ES, true>), g, dim3(256), 0, st, a, s);
    else hipLaunchKernelGGL((rows_scatter_kernel<ES, false>), g, dim3(256), 0, st, a, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_rows_scatter(const RowsArgs& a, hipStream_t st) { return a.dt == DT_F32 ? run_scatter<4>(a, st) : run_scatter<2>(a, st); }

template <int DT>
static int run_gather(const RowsArgs& a, hipStream_t st) {
    const int64_t units = (a.H + 7) / 8;
    const int s = row_shift(units), per = 256 >> s;
    const dim3 g((unsigned)((a.T + per - 1) / per), (unsigned)((units + (1 << s) - 1) >> s));
    if (s >= 6) hipLaunchKernelGGL((rows_gather_kernel<DT, true>), g, dim3(256), 0, st, a, s);
    else hipLaunchKernelGGL((rows_gather_kernel<DT, false>), g, dim3(256), 0, st, a, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_rows_gather(const RowsArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_gather<DT_F32>(a, st) : a.dt == DT_BF16 ? run_gather<DT_BF16>(a, st) : run_gather<DT_F16>(a, st);
}

template <int DT>
static int run_rows_grad(const RowsArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(rows_grad_kernel<DT>, dim3((unsigned)((a.P + 3) / 4)), dim3(256), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_rows_grad(const RowsArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_rows_grad<DT_F32>(a, st) : a.dt == DT_BF16 ? run_rows_grad<DT_BF16>(a, st) : run_rows_grad<DT_F16>(a, st);
}

}  // namespace mi355moe
