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

#include "rows.cuh"

namespace mi355moe {

// Sums over the TPR threads of a row of N values at once; `red` has N x TPR / 64 floats of this call's own.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = wave_sum(v[k]);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wv = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) red[k * W + wv] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += red[k * W + w];
            v[k] = s;
        }
    }
}

__device__ __forceinline__ float inv_rms(float sum, int H, float eps) { return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sum, (float)H) + eps)); }

// The row's gate values of columns c ..; token gates: one value.
__device__ __forceinline__ void gate8(const NormArgs& a, int64_t r, int c, int n, float (&g)[8]) {
    if (a.gate_kind == GATE_CHANNEL) load8_any(a.gate, a.gdt, c, n, g);
    else if (a.gate_kind == GATE_FULL) load8_any(a.gate, a.gdt, (size_t)r * a.H + c, n, g);
    else {
        const float v = a.gate_kind == GATE_TOKEN ? any_value(a.gate, a.gdt, r) : 1.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = v;
    }
}

// A row by TPR threads, 8 NV values each: 64 threads (four rows a workgroup) or a workgroup.
template <int DT, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormArgs a) {
    constexpr int PER = TPR < 256 ? 256 / TPR : 1;
    constexpr int W = TPR / 64;
    static_assert(TPR == 64 || PER == 1, "rows that share a workgroup have a wave each");
    __shared__ float red[2 * W];
    const int tid = threadIdx.x % TPR;
    const int64_t r = (int64_t)blockIdx.x * PER + threadIdx.x / TPR;
    if (r >= a.rows) return;                                         // (whole waves; PER > 1 has no barrier)
    float t[NV][8];
    float q[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + tid) * 8;
        load8<DT>(a.branch, (size_t)r * a.branch_stride + c, a.H - c, t[v]);
        if (a.post)
#pragma unroll
            for (int j = 0; j < 8; ++j) q[0] = __builtin_fmaf(t[v][j], t[v][j], q[0]);
    }
    float rb = 1.0f;
    if (a.post) {                                                    // (uniform)
        row_sums<TPR>(q, red);
        rb = inv_rms(q[0], a.H, a.eps);
    }
    q[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + tid) * 8, n = a.H - c;
        float w[8];
        if (a.post) {
            load8_any(a.post, a.wdt, c, n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] = t[v][j] * rb * w[j];
        }
        if (a.gate_kind != GATE_NONE) {
            gate8(a, r, c, n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] *= w[j];
        }
        if (a.res) {
            load8<DT>(a.res, (size_t)r * a.res_stride + c, n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] = __builtin_fmaf(a.beta, t[v][j], a.alpha * w[j]);
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j) t[v][j] *= a.beta;
        if (a.s) store8<DT>(a.s, (size_t)r * a.H + c, n, t[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) q[0] = __builtin_fmaf(t[v][j], t[v][j], q[0]);   // (a token's gate times nothing is not always zero)
    }
    float rs = 1.0f;
    if (a.pre) {                                                     // (uniform)
        row_sums<TPR>(q, red + W);
        rs = inv_rms(q[0], a.H, a.eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * TPR + tid) * 8, n = a.H - c;
            float w[8];
            load8_any(a.pre, a.wdt, c, n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = t[v][j] * rs * w[j];
            store8<DT>(a.y, (size_t)r * a.H + c, n, w);
        }
    }
    if (a.stats && tid == 0) {
        a.stats[2 * r] = rb;
        a.stats[2 * r + 1] = rs;
    }
}

// Gradients of rows blockIdx, blockIdx + gridDim, ...: those of the weights and of a channel's gate stay in registers and go to
// this workgroup's part [3][H] at the end (dpre, dpost, dgate; norm_join_kernel adds the parts in order).
template <int DT, int TPR, int NV>
__global__ __launch_bounds__(TPR) void norm_grad_kernel(NormArgs a) {
    constexpr int W = TPR / 64;
    __shared__ float red[2][2 * W];
    const int tid = threadIdx.x;
    float dpre[NV][8] = {}, dpost[NV][8] = {}, dgate[NV][8] = {};
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float rb = a.post ? a.stats[2 * r] : 1.0f, rs = a.stats[2 * r + 1];
        float nb[NV][8], t[NV][8], gs[NV][8], dn[NV][8];
        float q[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * TPR + tid) * 8, n = a.H - c;
            float w[8];
            load8<DT>(a.branch, (size_t)r * a.branch_stride + c, n, nb[v]);
            if (a.ds) load8<DT>(a.ds, (size_t)r * a.ds_stride + c, n, gs[v]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[v][j] = 0.0f;
            if (a.dy) {
                load8<DT>(a.dy, (size_t)r * a.dy_stride + c, n, dn[v]);
                if (a.res) load8<DT>(a.res, (size_t)r * a.res_stride + c, n, t[v]);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[v][j] = 0.0f;
            }
            if (a.post)
#pragma unroll
                for (int j = 0; j < 8; ++j) nb[v][j] *= rb;
            if (a.dy) {
                float u[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] = nb[v][j];
                if (a.post) {
                    load8_any(a.post, a.wdt, c, n, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] *= w[j];
                }
                if (a.gate_kind != GATE_NONE) {
                    gate8(a, r, c, n, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] *= w[j];
                }
                load8_any(a.pre, a.wdt, c, n, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    t[v][j] = __builtin_fmaf(a.beta, u[j], a.alpha * t[v][j]) * rs;      // n_s
                    dpre[v][j] = j < n ? __builtin_fmaf(dn[v][j], t[v][j], dpre[v][j]) : 0.0f;
                    dn[v][j] *= w[j];
                    q[0] += j < n ? t[v][j] * dn[v][j] : 0.0f;
                }
            }
        }
        if (a.dy) {                                                  // (uniform)
            row_sums<TPR>(q, red[0]);
            const float m = __fdiv_rn(q[0], (float)a.H);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[v][j] = __builtin_fmaf(rs, dn[v][j] - t[v][j] * m, gs[v][j]);
        }
        float p[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * TPR + tid) * 8, n = a.H - c;
            float g[8], w[8];
            if (a.dres) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = a.alpha * gs[v][j];
                store8<DT>(a.dres, (size_t)r * a.H + c, n, w);
            }
            gate8(a, r, c, n, g);
            if (a.post) load8_any(a.post, a.wdt, c, n, w);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = 1.0f;
            if (a.dgate) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = a.beta * gs[v][j] * (nb[v][j] * w[j]);
                if (a.gate_kind == GATE_FULL) {
                    if (a.gdt == DT_F32) store8<DT_F32>(a.dgate, (size_t)r * a.H + c, n, d);
                    else if (a.gdt == DT_BF16) store8<DT_BF16>(a.dgate, (size_t)r * a.H + c, n, d);
                    else store8<DT_F16>(a.dgate, (size_t)r * a.H + c, n, d);
                } else if (a.gate_kind == GATE_CHANNEL) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) dgate[v][j] += d[j];
                } else
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[1] += j < n ? d[j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float du = a.beta * g[j] * gs[v][j];
                if (a.post) dpost[v][j] = __builtin_fmaf(du, nb[v][j], dpost[v][j]);
                gs[v][j] = du * w[j];
                p[0] += j < n ? nb[v][j] * gs[v][j] : 0.0f;
            }
        }
        const bool token = a.dgate && a.gate_kind == GATE_TOKEN;
        if (a.post || token) {                                       // (uniform)
            row_sums<TPR>(p, red[1]);
            if (token && tid == 0) store_any(a.dgate, a.gdt, r, p[1]);
        }
        if (a.dbranch) {
            const float m = a.post ? __fdiv_rn(p[0], (float)a.H) : 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * TPR + tid) * 8;
                if (a.post)
#pragma unroll
                    for (int j = 0; j < 8; ++j) gs[v][j] = rb * (gs[v][j] - nb[v][j] * m);
                store8<DT>(a.dbranch, (size_t)r * a.H + c, a.H - c, gs[v]);
            }
        }
        if (TPR > 64) __syncthreads();                               // (the sums have been read: the next row writes them)
    }
    if (!a.part) return;
    float* part = a.part + (size_t)blockIdx.x * 3 * a.H;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + tid) * 8, n = a.H - c;
        if (a.dpre) store8<DT_F32>(part, c, n, dpre[v]);
        if (a.dpost) store8<DT_F32>(part + a.H, c, n, dpost[v]);
        if (a.dgate && a.gate_kind == GATE_CHANNEL) store8<DT_F32>(part + 2 * (size_t)a.H, c, n, dgate[v]);
    }
}

// out[k][c] = the sum over the parts of part[.][k][c], in order: 64 columns a workgroup, the parts cut over its sixteen waves.
__global__ __launch_bounds__(1024) void norm_join_kernel(NormArgs a, int parts) {
    __shared__ float red[16][64];
    const int k = blockIdx.y;
    void* out = k == 0 ? a.dpre : k == 1 ? a.dpost : a.gate_kind == GATE_CHANNEL ? a.dgate : nullptr;
    if (!out) return;                                                // (uniform)
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const int per = (parts + 15) / 16, g0 = wv * per, g1 = min(parts, g0 + per);
    float v = 0.0f;
    if (c < a.H) {
#pragma unroll 8
        for (int g = g0; g < g1; ++g) v += a.part[((size_t)g * 3 + k) * a.H + c];
    }
    red[wv][lane] = v;
    __syncthreads();
    if (wv || c >= a.H) return;
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += red[w][lane];
    store_any(out, k == 2 ? a.gdt : a.wdt, c, v);
}

template <int DT>
static int run_norm(const NormArgs& a, hipStream_t st) {
    const auto g = [&](int per) { return dim3((unsigned)((a.rows + per - 1) / per)); };
    if (a.H <= 512) hipLaunchKernelGGL((norm_kernel<DT, 64, 1>), g(4), dim3(256), 0, st, a);
    else if (a.H <= 2048) hipLaunchKernelGGL((norm_kernel<DT, 256, 1>), g(1), dim3(256), 0, st, a);
    else if (a.H <= 4096) hipLaunchKernelGGL((norm_kernel<DT, 512, 1>), g(1), dim3(512), 0, st, a);
    else if (a.H <= 8192) hipLaunchKernelGGL((norm_kernel<DT, 1024, 1>), g(1), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<DT, 1024, 2>), g(1), dim3(1024), 0, st, a);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_norm(const NormArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_norm<DT_F32>(a, st) : a.dt == DT_BF16 ? run_norm<DT_BF16>(a, st) : run_norm<DT_F16>(a, st);
}

// Workgroups of the gradient: what the card holds at once (1024 threads a CU at the registers that these kernels take).
static int norm_threads(int H) { return H <= 512 ? 64 : H <= 2048 ? 256 : H <= 4096 ? 512 : 1024; }
static int norm_parts(int64_t rows, int H) { return (int)std::min<int64_t>(rows, 256 * 1024 / norm_threads(H)); }
int64_t norm_part_floats(int64_t rows, int H) { return (int64_t)norm_parts(rows, H) * 3 * H; }

template <int DT>
static int run_norm_grad(const NormArgs& a, hipStream_t st) {
    const int parts = norm_parts(a.rows, a.H);
    const dim3 g(parts), b(norm_threads(a.H));
    if (a.H <= 512) hipLaunchKernelGGL((norm_grad_kernel<DT, 64, 1>), g, b, 0, st, a);
    else if (a.H <= 2048) hipLaunchKernelGGL((norm_grad_kernel<DT, 256, 1>), g, b, 0, st, a);
    else if (a.H <= 4096) hipLaunchKernelGGL((norm_grad_kernel<DT, 512, 1>), g, b, 0, st, a);
    else if (a.H <= 8192) hipLaunchKernelGGL((norm_grad_kernel<DT, 1024, 1>), g, b, 0, st, a);
    else hipLaunchKernelGGL((norm_grad_kernel<DT, 1024, 2>), g, b, 0, st, a);
    if (hipGetLastError() != hipSuccess) return -1;
    if (a.part) {
        hipLaunchKernelGGL(norm_join_kernel, dim3((a.H + 63) / 64, 3), dim3(1024), 0, st, a, parts);
        if (hipGetLastError() != hipSuccess) return -1;
    }
    return 0;
}
int launch_norm_grad(const NormArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_norm_grad<DT_F32>(a, st) : a.dt == DT_BF16 ? run_norm_grad<DT_BF16>(a, st) : run_norm_grad<DT_F16>(a, st);
}

}  // namespace mi355moe
