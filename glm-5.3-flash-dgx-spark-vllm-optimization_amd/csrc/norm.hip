// The norms around a block, with its gate and the scaled residual sum, in one pass over the rows.
//
//   u = b r(b) post  (or b);   s = alpha res + beta gate u;   y = s r(s) pre;   r(v) = 1 / sqrt(mean v^2 + eps)
//
// in fp32 from the loads to one rounding of s and of y (r(s) and y go by the unrounded s). With n_b = b r(b), n_s = s r(s),
// dn = dy pre the gradients are
//
//   gs = ds + r(s) (dn - n_s mean(n_s dn));   dres = alpha gs;   dgate = beta gs u;   du = beta gate gs
//   db = r(b) (du post - n_b mean(n_b du post))  (or du);   dpre = sum over rows dy n_s;   dpost = sum over rows du n_b
//
// s is formed again from b, res and gate, which have to be read anyway, in fp32: the rounded s would put its rounding into
// dpre, whose weights may be fp32. Only the two r of a row are kept from the forward pass.
#include <algorithm>

#include "gemm_tile.cuh"
#include "rows.cuh"

namespace mi355moe {

// Sums of N values over a row's threads: a wave (WG false), or a workgroup of up to sixteen waves; `red` has 16 N floats of this
// call's own.
template <bool WG, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
    if constexpr (WG) {
        const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) red[16 * k + (threadIdx.x >> 6)] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float s = (lane & 15) < waves ? red[16 * k + (lane & 15)] : 0.0f;
            s += xor_lane<1>(s, lane);
            s += xor_lane<2>(s, lane);
            s += xor_lane<4>(s, lane);
            v[k] = s + xor_lane<8>(s, lane);
        }
    }
}

__device__ __forceinline__ float inv_rms(float sum, int H, float eps) { return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sum, (float)H) + eps)); }

// A row of up to 8 NV values a thread: by a wave, four rows a workgroup (WG false), or by a workgroup of as many threads as the row
// needs. Everything that the row reads is requested before the first sum.
template <int DT, bool WG, int NV, bool ONCE>
__global__ __launch_bounds__(WG ? 1024 : 256) void norm_kernel(NormArgs a) {
    __shared__ float red[2][16];
    const int tpr = WG ? blockDim.x : 64, tid = WG ? threadIdx.x : threadIdx.x & 63;
    const int64_t r = WG ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= a.rows) return;                                         // (whole waves, which share no barrier)
    Raw8<DT> rb8[NV], rr8[NV];
    RawAny8 post8[NV], pre8[NV], gate8[NV];
    float token = 1.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * tpr + tid) * 8, n = a.H - c;
        rb8[v].template load<ONCE>(a.branch, (size_t)r * a.branch_stride + c, n);
        if (a.res) rr8[v].template load<ONCE>(a.res, (size_t)r * a.res_stride + c, n);
        if (a.post) post8[v].load(a.post, a.wdt, c, n);
        if (a.gate_kind == GATE_CHANNEL) gate8[v].load(a.gate, a.gdt, c, n);
        if (a.gate_kind == GATE_FULL) gate8[v].load(a.gate, a.gdt, (size_t)r * a.H + c, n);
        if (a.pre) pre8[v].load(a.pre, a.wdt, c, n);
    }
    if (a.gate_kind == GATE_TOKEN) token = any_value(a.gate, a.gdt, r);
    float t[NV][8];
    float q[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        rb8[v].get(t[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[0] = __builtin_fmaf(t[v][j], t[v][j], q[0]);
    }
    float rb = 1.0f;
    if (a.post) {                                                    // (uniform)
        row_sums<WG>(q, red[0]);
        rb = inv_rms(q[0], a.H, a.eps);
    }
    const float beta = a.gate_kind == GATE_TOKEN ? a.beta * token : a.beta;
    q[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * tpr + tid) * 8, n = a.H - c;
        float w[8];
        if (a.post) {
            post8[v].get(a.wdt, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] = t[v][j] * rb * w[j];
        }
        if (a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_FULL) {
            gate8[v].get(a.gdt, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] *= w[j];
        }
        if (a.res) {
            rr8[v].get(w);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] = __builtin_fmaf(beta, t[v][j], a.alpha * w[j]);
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] *= beta;
        if (a.s) store8<DT>(a.s, (size_t)r * a.H + c, n, t[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[0] = j < n ? __builtin_fmaf(t[v][j], t[v][j], q[0]) : q[0];   // (0 times infinity is not 0)
    }
    float rs = 1.0f;
    if (a.pre) {                                                     // (uniform)
        row_sums<WG>(q, red[1]);
        rs = inv_rms(q[0], a.H, a.eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + tid) * 8;
            float w[8];
            pre8[v].get(a.wdt, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = t[v][j] * rs * w[j];
            store8<DT>(a.y, (size_t)r * a.H + c, a.H - c, w);
        }
    }
    if (a.stats && tid == 0) {
        a.stats[2 * r] = rb;
        a.stats[2 * r + 1] = rs;
    }
}

// A thread's own values of the weights and of a channel's gate, which it reads again for every row: in LDS as fp32, where they take
// neither registers nor the caches' bandwidth (a row of 4096 with fp32 weights would read 40 KB of them for 32 KB of its own).
// CACHED false (rows of more than 8192 values): from memory each time.
template <bool CACHED>
struct RowConstants {
    f32x4* lds;                                                      // [3][2][threads]
    __device__ __forceinline__ f32x4* at(int k, int half) const { return lds + (2 * k + half) * blockDim.x + threadIdx.x; }
    __device__ __forceinline__ void keep(int k, const void* p, int dt, int n) const {
        if constexpr (CACHED) {
            float v[8];
            load8_any(p, dt, threadIdx.x * 8, n, v);
            *at(k, 0) = f32x4{v[0], v[1], v[2], v[3]};
            *at(k, 1) = f32x4{v[4], v[5], v[6], v[7]};
        }
    }
    __device__ __forceinline__ void get(int k, const void* p, int dt, int c, int n, float (&v)[8]) const {
        if constexpr (CACHED) {
            const f32x4 lo = *at(k, 0), hi = *at(k, 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
        } else load8_any(p, dt, c, n, v);
    }
};

// Gradients of rows blockIdx, blockIdx + gridDim, ...: those of the weights and of a channel's gate stay in registers and go to
// this workgroup's part [2][H] at the end (norm_join_kernel adds the parts in order): the sums of dy n_s, and of du n_b; a
// channel's gate takes its factors out of the second, sum of gs n_b, which then gives dpost (times beta gate) and dgate (times
// beta post) both. A row's loads are requested while the row before it is worked on.
template <int DT, int NV>
__global__ __launch_bounds__(1024) void norm_grad_kernel(NormArgs a) {
    extern __shared__ __align__(16) f32x4 lds[];
    __shared__ float red[2][2 * 16];
    const RowConstants<NV == 1> kept{lds};
    const int tid = threadIdx.x, tpr = blockDim.x;
    float dpre[NV][8] = {}, sum[NV][8] = {};
    const bool channel = a.gate_kind == GATE_CHANNEL;
    if constexpr (NV == 1) {
        const int n = a.H - tid * 8;
        if (a.post) kept.keep(0, a.post, a.wdt, n);
        if (a.dy) kept.keep(1, a.pre, a.wdt, n);
        if (a.gate_kind == GATE_CHANNEL) kept.keep(2, a.gate, a.gdt, n);
    }
    Raw8<DT> b8[NV], r8[NV], s8[NV], y8[NV];
    auto request = [&](int64_t r) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + tid) * 8, n = a.H - c;
            b8[v].load(a.branch, (size_t)r * a.branch_stride + c, n);
            if (a.dy) {
                y8[v].load(a.dy, (size_t)r * a.dy_stride + c, n);
                if (a.res) r8[v].load(a.res, (size_t)r * a.res_stride + c, n);
            }
            if (a.ds) s8[v].load(a.ds, (size_t)r * a.ds_stride + c, n);
        }
    };
    request(blockIdx.x);                                             // (gridDim <= rows)
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float rb = a.post ? a.stats[2 * r] : 1.0f, rs = a.stats[2 * r + 1];
        const float beta = a.gate_kind == GATE_TOKEN ? a.beta * any_value(a.gate, a.gdt, r) : a.beta;
        float nb[NV][8], t[NV][8], gs[NV][8], dn[NV][8];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            b8[v].get(nb[v]);
            if (a.dy) y8[v].get(dn[v]);
            if (a.dy && a.res) r8[v].get(t[v]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) t[v][j] = 0.0f;
            if (a.ds) s8[v].get(gs[v]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[v][j] = 0.0f;
        }
        if (r + gridDim.x < a.rows) request(r + gridDim.x);
        // what the branch's value passes on its way to s: post and the gate, whose product also takes gs back
        auto gate = [&](int c, int n, float (&g)[8]) {
            if (a.gate_kind == GATE_CHANNEL) kept.get(2, a.gate, a.gdt, c, n, g);
            else if (a.gate_kind == GATE_FULL) load8_any(a.gate, a.gdt, (size_t)r * a.H + c, n, g);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = 1.0f;
        };
        float q[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + tid) * 8, n = a.H - c;
            if (a.post)
#pragma unroll
                for (int j = 0; j < 8; ++j) nb[v][j] *= rb;
            if (a.dy) {
                float u[8], w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = nb[v][j];
                if (a.post) {
                    kept.get(0, a.post, a.wdt, c, n, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] *= w[j];
                }
                if (a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_FULL) {
                    gate(c, n, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] *= w[j];
                }
                kept.get(1, a.pre, a.wdt, c, n, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    t[v][j] = __builtin_fmaf(beta, u[j], a.alpha * t[v][j]) * rs;        // n_s
                    dpre[v][j] = __builtin_fmaf(dn[v][j], t[v][j], dpre[v][j]);          // (columns behind the row's end: never read)
                    dn[v][j] *= w[j];
                    q[0] = j < n ? __builtin_fmaf(t[v][j], dn[v][j], q[0]) : q[0];
                }
            }
        }
        if (a.dy) {                                                  // (uniform)
            row_sums<true>(q, red[0]);
            const float m = __fdiv_rn(q[0], (float)a.H);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[v][j] = __builtin_fmaf(rs, dn[v][j] - t[v][j] * m, gs[v][j]);
        }
        float p[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + tid) * 8, n = a.H - c;
            float g[8], w[8];
            if (a.dres) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = a.alpha * gs[v][j];
                store8<DT>(a.dres, (size_t)r * a.H + c, n, w);
            }
            gate(c, n, g);
            if (a.post) kept.get(0, a.post, a.wdt, c, n, w);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = 1.0f;
            if (a.dgate && !channel) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = a.beta * gs[v][j] * (nb[v][j] * w[j]);
                if (a.gate_kind == GATE_TOKEN) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[1] += j < n ? d[j] : 0.0f;
                } else if (a.gdt == DT_F32) store8<DT_F32>(a.dgate, (size_t)r * a.H + c, n, d);
                else if (a.gdt == DT_BF16) store8<DT_BF16>(a.dgate, (size_t)r * a.H + c, n, d);
                else store8<DT_F16>(a.dgate, (size_t)r * a.H + c, n, d);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float du = beta * g[j] * gs[v][j];
                sum[v][j] = __builtin_fmaf(channel ? gs[v][j] : du, nb[v][j], sum[v][j]);
                gs[v][j] = du * w[j];
                p[0] = j < n ? __builtin_fmaf(nb[v][j], gs[v][j], p[0]) : p[0];
            }
        }
        const bool token = a.dgate && a.gate_kind == GATE_TOKEN;
        if (a.post || token) {                                       // (uniform)
            row_sums<true>(p, red[1]);
            if (token && tid == 0) store_any(a.dgate, a.gdt, r, p[1]);
        }
        if (a.dbranch) {
            const float m = a.post ? __fdiv_rn(p[0], (float)a.H) : 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * tpr + tid) * 8;
                if (a.post)
#pragma unroll
                    for (int j = 0; j < 8; ++j) gs[v][j] = rb * (gs[v][j] - nb[v][j] * m);
                store8<DT>(a.dbranch, (size_t)r * a.H + c, a.H - c, gs[v]);
            }
        }
        __syncthreads();                                             // (the sums have been read: the next row writes them)
    }
    if (!a.part) return;
    float* part = a.part + (size_t)blockIdx.x * 2 * a.H;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * tpr + tid) * 8, n = a.H - c;
        if (a.dpre) store8<DT_F32>(part, c, n, dpre[v]);
        if (a.dpost || (a.dgate && channel)) store8<DT_F32>(part + a.H, c, n, sum[v]);
    }
}

// dpre (grid y 0), and dpost and a channel's dgate (1), from the sums over the parts of part[.][y][c], in order: 64 columns a
// workgroup, the parts cut over its sixteen waves.
__global__ __launch_bounds__(1024) void norm_join_kernel(NormArgs a, int parts) {
    __shared__ float red[16][64];
    const int k = blockIdx.y;
    void* dgate = a.gate_kind == GATE_CHANNEL ? a.dgate : nullptr;
    if (k == 0 ? !a.dpre : !a.dpost && !dgate) return;               // (uniform)
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const int per = (parts + 15) / 16, g0 = wv * per, g1 = min(parts, g0 + per);
    float v = 0.0f;
    if (c < a.H) {
#pragma unroll 8
        for (int g = g0; g < g1; ++g) v += a.part[((size_t)g * 2 + k) * a.H + c];
    }
    red[wv][lane] = v;
    __syncthreads();
    if (wv || c >= a.H) return;
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += red[w][lane];
    if (k == 0) {
        store_any(a.dpre, a.wdt, c, v);
        return;
    }
    if (a.dpost) store_any(a.dpost, a.wdt, c, a.gate_kind == GATE_CHANNEL ? v * a.beta * any_value(a.gate, a.gdt, c) : v);
    if (dgate) store_any(dgate, a.gdt, c, v * a.beta * (a.post ? any_value(a.post, a.wdt, c) : 1.0f));
}

// Threads of a row: eight values each up to 8192, sixteen beyond; whole waves.
static int norm_threads(int H) { return H <= 8192 ? (H + 511) / 512 * 64 : 1024; }

// Tensors of 64 MB and more are marked as read once (us plain / marked, bf16 rows of 4096: 1237 rows 11.2 / 11.7, 8192 47.5 / 46.0,
// 16384 94.6 / 86.5; the gradient, which reads and writes more besides: no difference).
static bool norm_once(const NormArgs& a) { return a.rows * a.H * (a.dt == DT_F32 ? 4 : 2) >= (64 << 20); }

template <int DT>
static int run_norm(const NormArgs& a, hipStream_t st) {
    const int t = norm_threads(a.H);
    if (t == 64) hipLaunchKernelGGL((norm_kernel<DT, false, 1, false>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
    else if (a.H <= 8192 && norm_once(a)) hipLaunchKernelGGL((norm_kernel<DT, true, 1, true>), dim3((unsigned)a.rows), dim3(t), 0, st, a);
    else if (a.H <= 8192) hipLaunchKernelGGL((norm_kernel<DT, true, 1, false>), dim3((unsigned)a.rows), dim3(t), 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<DT, true, 2, false>), dim3((unsigned)a.rows), dim3(t), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_norm(const NormArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_norm<DT_F32>(a, st) : a.dt == DT_BF16 ? run_norm<DT_BF16>(a, st) : run_norm<DT_F16>(a, st);
}

// Workgroups of the gradient: 1024 threads a CU, what its registers hold.
static int norm_parts(int64_t rows, int H) { return (int)std::min<int64_t>(rows, 256 * std::min(8, 1024 / norm_threads(H))); }
int64_t norm_part_floats(int64_t rows, int H) { return (int64_t)norm_parts(rows, H) * 2 * H; }

template <int DT>
static int run_norm_grad(const NormArgs& a, hipStream_t st) {
    const int parts = norm_parts(a.rows, a.H), t = norm_threads(a.H);
    if (a.H <= 8192) {
        if (!allow_lds<norm_grad_kernel<DT, 1>>(96 * 1024)) return -1;
        hipLaunchKernelGGL((norm_grad_kernel<DT, 1>), dim3(parts), dim3(t), 96 * t, st, a);
    } else hipLaunchKernelGGL((norm_grad_kernel<DT, 2>), dim3(parts), dim3(t), 0, st, a);
    if (hipGetLastError() != hipSuccess) return -1;
    if (a.part) {
        hipLaunchKernelGGL(norm_join_kernel, dim3((a.H + 63) / 64, 2), dim3(1024), 0, st, a, parts);
        if (hipGetLastError() != hipSuccess) return -1;
    }
    return 0;
}
int launch_norm_grad(const NormArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_norm_grad<DT_F32>(a, st) : a.dt == DT_BF16 ? run_norm_grad<DT_BF16>(a, st) : run_norm_grad<DT_F16>(a, st);
}

}  // namespace mi355moe
