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

// Sums of N values over a row's threads: 2^shift lanes of a wave (WG false), or a workgroup of up to sixteen waves; `red` has 16 N
// floats of this call's own.
template <bool WG, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int shift) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        float s = v[k];
        s += xor_lane<1>(s, lane);
        s += xor_lane<2>(s, lane);
        s += xor_lane<4>(s, lane);
        if (WG || shift > 3) s += xor_lane<8>(s, lane);              // (uniform)
        if (WG || shift > 4) s += xor_lane<16>(s, lane);
        if (WG || shift > 5) s += xor_lane<32>(s, lane);
        v[k] = s;
    }
    if constexpr (WG) {
        const int waves = blockDim.x >> 6;
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

// A row of up to 8 NV values a thread: by 2^shift lanes, as many rows a workgroup as fit (WG false), or by a workgroup of as many
// threads as the row needs. Everything that the row reads is requested before the first sum, and stays in registers to the end: one
// pass. Bound: HBM for many rows (16384 of 4096, bf16 with post, pre and residual: 537 MB in 80 to 86 us, 6.4 TB/s, what the caches
// still hold among it; 32768 of 64: 7 us; 8192 fp32 rows of 4096: 537 MB in 107 to 113 us, 4.9 TB/s; 2048 rows of 16384: bf16 268
// MB in 75 us, fp32 537 MB in 120), latency for few (1 row 3.0 us, 1237 odd fp16 rows of 4099 15 us: their rows begin at any 2-byte
// address, which costs 4 us over 1237 of 4096).
template <int DT, bool WG, int NV, bool ONCE>
__global__ __launch_bounds__(WG ? 1024 : 256) void norm_kernel(NormArgs a, int shift) {
    __shared__ float red[2][16];
    const int tpr = WG ? blockDim.x : 1 << shift, tid = WG ? threadIdx.x : threadIdx.x & ((1 << shift) - 1);
    const int64_t first = WG ? (int64_t)wide_block() : (int64_t)wide_block() << (8 - shift);
    if (first >= a.rows) return;                                     // (uniform)
    const int64_t at = WG ? first : first + (threadIdx.x >> shift);
    const int64_t r = min(at, a.rows - 1);                           // (lanes without a row repeat the last one's values)
    const bool mine = WG || at < a.rows;
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
        row_sums<WG>(q, red[0], shift);
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
        if (a.s && mine) store8<DT>(a.s, (size_t)r * a.H + c, n, t[v]);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[0] = j < n ? __builtin_fmaf(t[v][j], t[v][j], q[0]) : q[0];   // (0 times infinity is not 0)
    }
    float rs = 1.0f;
    if (a.pre) {                                                     // (uniform)
        row_sums<WG>(q, red[1], shift);
        rs = inv_rms(q[0], a.H, a.eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * tpr + tid) * 8;
            float w[8];
            pre8[v].get(a.wdt, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = t[v][j] * rs * w[j];
            if (mine) store8<DT>(a.y, (size_t)r * a.H + c, a.H - c, w);
        }
    }
    if (a.stats && tid == 0 && mine) {
        a.stats[2 * r] = rb;
        a.stats[2 * r + 1] = rs;
    }
}

// A thread's own values of the weights and of a channel's gate, which it reads again for every row: in LDS as fp32, where they take
// neither registers nor the caches' bandwidth (a row of 4096 with fp32 weights would read 40 KB of them for 32 KB of its own).
struct RowConstants {
    f32x4* lds;                                                      // [3][2][threads]
    __device__ __forceinline__ f32x4* at(int k, int half) const { return lds + (2 * k + half) * blockDim.x + threadIdx.x; }
    __device__ __forceinline__ void keep(int k, const void* p, int dt, int c, int n) const {
        float v[8];
        load8_any(p, dt, c, n, v);
        *at(k, 0) = f32x4{v[0], v[1], v[2], v[3]};
        *at(k, 1) = f32x4{v[4], v[5], v[6], v[7]};
    }
    __device__ __forceinline__ void get(int k, float (&v)[8]) const {
        const f32x4 lo = *at(k, 0), hi = *at(k, 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
    }
};

template <int DT>
struct RowInputs {
    Raw8<DT> b, r, s, y;                                             // branch, residual, ds, dy
    __device__ __forceinline__ void load(const NormArgs& a, int64_t row, int c) {
        const int n = a.H - c;
        b.load(a.branch, (size_t)row * a.branch_stride + c, n);
        if (a.dy) {
            y.load(a.dy, (size_t)row * a.dy_stride + c, n);
            if (a.res) r.load(a.res, (size_t)row * a.res_stride + c, n);
        }
        if (a.ds) s.load(a.ds, (size_t)row * a.ds_stride + c, n);
    }
};

__device__ __forceinline__ void store_gate(const NormArgs& a, size_t at, int n, const float (&d)[8]) {
    if (a.gdt == DT_F32) store8<DT_F32>(a.dgate, at, n, d);
    else if (a.gdt == DT_BF16) store8<DT_BF16>(a.dgate, at, n, d);
    else store8<DT_F16>(a.dgate, at, n, d);
}

// Gradients of rows blockIdx, blockIdx + gridDim, ... (WG false: of as many rows at once as 2^shift lanes each leave room for):
// those of the weights and of a channel's gate stay in registers and go to this workgroup's part [2][H] at the end
// (norm_join_kernel adds the parts in order): the sums of dy n_s, and of du n_b; a channel's gate takes its factors out of the
// second, sum of gs n_b, which then gives dpost (times beta gate) and dgate (times beta post) both. A row's loads are requested
// while the row before it is worked on. Bound: HBM with the two barriers of a row in its way (8192 rows of 4096, bf16, a channel's
// gate: 403 MB in 90 to 96 us, 4.3 TB/s; in fp32 805 MB in 164 to 168, 4.8; 32768 rows of 64 11 us, of 512 43 us).
template <int DT, bool WG>
__global__ __launch_bounds__(WG ? 1024 : 256, WG ? 1 : DT == DT_F32 ? 3 : 4) void norm_grad_kernel(NormArgs a, int shift) {
    extern __shared__ __align__(16) f32x4 lds[];
    __shared__ float red[2][2 * 16];
    const RowConstants kept{lds};
    const int tid = WG ? threadIdx.x : threadIdx.x & ((1 << shift) - 1);
    const int per = WG ? 1 : 256 >> shift, sub = WG ? 0 : threadIdx.x >> shift;      // rows at once, and this thread's of them
    const int c = tid * 8, n = a.H - c;
    float dpre[8] = {}, sum[8] = {};
    const bool channel = a.gate_kind == GATE_CHANNEL, gated = channel || a.gate_kind == GATE_FULL;
    if (a.post) kept.keep(0, a.post, a.wdt, c, n);
    if (a.dy) kept.keep(1, a.pre, a.wdt, c, n);
    if (channel) kept.keep(2, a.gate, a.gdt, c, n);
    RowInputs<DT> next;
    const int64_t step = (int64_t)gridDim.x * per;
    int64_t r0 = (int64_t)blockIdx.x * per;
    if (r0 < a.rows) next.load(a, WG ? r0 : min(r0 + sub, a.rows - 1), c);
    for (; r0 < a.rows; r0 += step) {                                // (uniform)
        const int64_t r = WG ? r0 : min(r0 + sub, a.rows - 1);
        const bool mine = WG || r0 + sub < a.rows;                   // (lanes without a row repeat the last one and add nothing)
        const float rb = a.post ? a.stats[2 * r] : 1.0f, rs = a.stats[2 * r + 1];
        const float beta = a.gate_kind == GATE_TOKEN ? a.beta * any_value(a.gate, a.gdt, r) : a.beta;
        float nb[8], t[8], gs[8], dn[8];
        next.b.get(nb);
        if (a.dy) next.y.get(dn);
        if (a.dy && a.res) next.r.get(t);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = 0.0f;
        if (a.ds) next.s.get(gs);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) gs[j] = 0.0f;
        if (r0 + step < a.rows) next.load(a, WG ? r0 + step : min(r0 + step + sub, a.rows - 1), c);
        // what the branch's value passes on its way to s: post and the gate, whose product also takes gs back
        auto gate = [&](float (&g)[8]) {
            if (channel) kept.get(2, g);
            else if (gated) load8_any(a.gate, a.gdt, (size_t)r * a.H + c, n, g);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = 1.0f;
        };
        if (a.post)
#pragma unroll
            for (int j = 0; j < 8; ++j) nb[j] *= rb;
        if (a.dy) {                                                  // (uniform)
            float q[1] = {0.0f};
            float u[8], w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = nb[j];
            if (a.post) {
                kept.get(0, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] *= w[j];
            }
            if (gated) {
                gate(w);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] *= w[j];
            }
            kept.get(1, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                t[j] = __builtin_fmaf(beta, u[j], a.alpha * t[j]) * rs;                  // n_s
                dpre[j] = mine ? __builtin_fmaf(dn[j], t[j], dpre[j]) : dpre[j];         // (columns behind the row's end: never read)
                dn[j] *= w[j];
                q[0] = j < n ? __builtin_fmaf(t[j], dn[j], q[0]) : q[0];
            }
            row_sums<WG>(q, red[0], shift);
            const float m = __fdiv_rn(q[0], (float)a.H);
#pragma unroll
            for (int j = 0; j < 8; ++j) gs[j] = __builtin_fmaf(rs, dn[j] - t[j] * m, gs[j]);
        }
        float p[2] = {0.0f, 0.0f};
        float g[8], w[8];
        if (a.dres && mine) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = a.alpha * gs[j];
            store8<DT>(a.dres, (size_t)r * a.H + c, n, w);
        }
        gate(g);
        if (a.post) kept.get(0, w);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = 1.0f;
        if (a.dgate && !channel) {
            float d[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = a.beta * gs[j] * (nb[j] * w[j]);
            if (a.gate_kind == GATE_TOKEN) {
#pragma unroll
                for (int j = 0; j < 8; ++j) p[1] += j < n ? d[j] : 0.0f;
            } else if (mine) store_gate(a, (size_t)r * a.H + c, n, d);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float du = beta * g[j] * gs[j];
            sum[j] = mine ? __builtin_fmaf(channel ? gs[j] : du, nb[j], sum[j]) : sum[j];
            gs[j] = du * w[j];
            p[0] = j < n ? __builtin_fmaf(nb[j], gs[j], p[0]) : p[0];
        }
        const bool token = a.dgate && a.gate_kind == GATE_TOKEN;
        if (a.post || token) {                                       // (uniform)
            row_sums<WG>(p, red[1], shift);
            if (token && tid == 0 && mine) store_any(a.dgate, a.gdt, r, p[1]);
        }
        if (a.dbranch && mine) {
            const float m = a.post ? __fdiv_rn(p[0], (float)a.H) : 0.0f;
            if (a.post)
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[j] = rb * (gs[j] - nb[j] * m);
            store8<DT>(a.dbranch, (size_t)r * a.H + c, n, gs);
        }
        if (WG) __syncthreads();                                     // (the sums have been read: the next row writes them)
    }
    if (!a.part) return;
    if constexpr (!WG) {
        // the sums of the workgroup's rows: of a wave's groups, which hold the same columns, then of the waves, in order
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        float* const all = (float*)lds;                              // [4][2][8 << shift]
        __syncthreads();                                             // (the weights in it have been read)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (shift < 4) dpre[j] += xor_lane<8>(dpre[j], lane), sum[j] += xor_lane<8>(sum[j], lane);
            if (shift < 5) dpre[j] += xor_lane<16>(dpre[j], lane), sum[j] += xor_lane<16>(sum[j], lane);
            if (shift < 6) dpre[j] += xor_lane<32>(dpre[j], lane), sum[j] += xor_lane<32>(sum[j], lane);
            if (!(lane >> shift)) {
                all[((2 * wave * 8 + j) << shift) + lane] = dpre[j];
                all[(((2 * wave + 1) * 8 + j) << shift) + lane] = sum[j];
            }
        }
        __syncthreads();
        if (threadIdx.x >> shift) return;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int w = 1; w < 4; ++w) {
                dpre[j] += all[((2 * w * 8 + j) << shift) + lane];
                sum[j] += all[(((2 * w + 1) * 8 + j) << shift) + lane];
            }
    }
    float* part = a.part + (size_t)blockIdx.x * 2 * a.H;
    if (a.dpre) store8<DT_F32>(part, c, n, dpre);
    if (a.dpost || (a.dgate && channel)) store8<DT_F32>(part + a.H, c, n, sum);
}

// The same for rows of 8193 to 16384 values, sixteen a thread: held as floats they would not fit the registers of 1024 threads (the
// kernel above with twice its values, which kept 360 to 500 bytes a lane in scratch: 2048 rows of 16384 284 us). So a row's values
// stay as they were loaded and each pass makes them floats again, and the sums over the rows stay in LDS. Four tensors' values over
// two barriers pass 128 registers even so: 112 bytes a lane are in scratch for bf16 and fp16, 228 for fp32. Bound: that, and the
// one workgroup that a CU holds, which waits at each row's barriers (2048 rows of 16384, a channel's gate: bf16 403 MB in 166 us,
// 2.4 TB/s, fp16 177; fp32 805 MB in 325).
template <int DT>
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(NormArgs a) {
    extern __shared__ __align__(16) f32x4 lds[];
    __shared__ float red[2][2 * 16];
    constexpr int NV = 2;
    const int tid = threadIdx.x;
    const bool channel = a.gate_kind == GATE_CHANNEL, gated = channel || a.gate_kind == GATE_FULL;
    f32x4* const mem = lds + tid;                                    // [2][NV][2][1024]: this thread's own
    for (int k = 0; k < 4 * NV; ++k) mem[k * 1024] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](int k, int v, const float (&x)[8], const float (&y)[8]) {     // += x y
        f32x4* const at = mem + 2 * (NV * k + v) * 1024;
        f32x4 lo = at[0], hi = at[1024];
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = __builtin_fmaf(x[j], y[j], lo[j]), hi[j] = __builtin_fmaf(x[4 + j], y[4 + j], hi[j]);
        at[0] = lo;
        at[1024] = hi;
    };
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        RowInputs<DT> in[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) in[v].load(a, r, (v * 1024 + tid) * 8);
        const float rb = a.post ? a.stats[2 * r] : 1.0f, rs = a.stats[2 * r + 1];
        const float beta = a.gate_kind == GATE_TOKEN ? a.beta * any_value(a.gate, a.gdt, r) : a.beta;
        auto times = [&](const void* p, int dt, size_t at, int n, float (&x)[8]) {
            float w[8];
            load8_any(p, dt, at, n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= w[j];
        };
        auto times_gate = [&](int c, int n, float (&x)[8]) {
            if (gated) times(a.gate, a.gdt, channel ? c : (size_t)r * a.H + c, n, x);
        };
        // n_s and dn of eight values
        auto after = [&](const RowInputs<DT>& x, int c, int n, float (&t)[8], float (&dn)[8]) {
            float u[8];
            x.b.get(u);
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] *= rb;
            if (a.post) times(a.post, a.wdt, c, n, u);
            times_gate(c, n, u);
            if (a.res) x.r.get(t);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = 0.0f;
            x.y.get(dn);
            times(a.pre, a.wdt, c, n, dn);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = __builtin_fmaf(beta, u[j], a.alpha * t[j]) * rs;
        };
        float m = 0.0f;
        if (a.dy) {                                                  // (uniform)
            float q[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * 1024 + tid) * 8, n = a.H - c;
                float t[8], dn[8], dy[8];
                after(in[v], c, n, t, dn);
                in[v].y.get(dy);
                add(0, v, dy, t);                                    // (behind the row's end: never read)
#pragma unroll
                for (int j = 0; j < 8; ++j) q[0] = j < n ? __builtin_fmaf(t[j], dn[j], q[0]) : q[0];
            }
            row_sums<true>(q, red[0], 0);
            m = __fdiv_rn(q[0], (float)a.H);
        }
        float p[2] = {0.0f, 0.0f};
        float back[NV][8];                                           // du post
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int c = (v * 1024 + tid) * 8, n = a.H - c;
            float gs[8], nb[8], w[8];
            if (a.ds) in[v].s.get(gs);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[j] = 0.0f;
            if (a.dy) {
                float t[8], dn[8];
                after(in[v], c, n, t, dn);
#pragma unroll
                for (int j = 0; j < 8; ++j) gs[j] = __builtin_fmaf(rs, dn[j] - t[j] * m, gs[j]);
            }
            if (a.dres) {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = a.alpha * gs[j];
                store8<DT>(a.dres, (size_t)r * a.H + c, n, w);
            }
            in[v].b.get(nb);
#pragma unroll
            for (int j = 0; j < 8; ++j) nb[j] *= rb, w[j] = 1.0f;
            if (a.post) load8_any(a.post, a.wdt, c, n, w);
            if (a.dgate && !channel) {
                float d[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) d[j] = a.beta * gs[j] * (nb[j] * w[j]);
                if (a.gate_kind == GATE_TOKEN) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[1] += j < n ? d[j] : 0.0f;
                } else store_gate(a, (size_t)r * a.H + c, n, d);
            }
            if (channel) add(1, v, gs, nb);
#pragma unroll
            for (int j = 0; j < 8; ++j) gs[j] *= beta;
            times_gate(c, n, gs);
            if (!channel) add(1, v, gs, nb);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                back[v][j] = gs[j] * w[j];
                p[0] = j < n ? __builtin_fmaf(nb[j], back[v][j], p[0]) : p[0];
            }
        }
        const bool token = a.dgate && a.gate_kind == GATE_TOKEN;
        if (a.post || token) {                                       // (uniform)
            row_sums<true>(p, red[1], 0);
            if (token && tid == 0) store_any(a.dgate, a.gdt, r, p[1]);
        }
        if (a.dbranch) {
            const float k = a.post ? __fdiv_rn(p[0], (float)a.H) : 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int c = (v * 1024 + tid) * 8;
                if (a.post) {
                    float nb[8];
                    in[v].b.get(nb);
#pragma unroll
                    for (int j = 0; j < 8; ++j) back[v][j] = rb * (back[v][j] - nb[j] * rb * k);
                }
                store8<DT>(a.dbranch, (size_t)r * a.H + c, a.H - c, back[v]);
            }
        }
        __syncthreads();                                             // (the sums have been read: the next row writes them)
    }
    if (!a.part) return;
    float* part = a.part + (size_t)blockIdx.x * 2 * a.H;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * 1024 + tid) * 8, n = a.H - c;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const f32x4 lo = mem[2 * (NV * k + v) * 1024], hi = mem[(2 * (NV * k + v) + 1) * 1024];
            const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (k ? a.dpost || (a.dgate && channel) : a.dpre != nullptr) store8<DT_F32>(part + (k ? a.H : 0), c, n, x);
        }
    }
}

// dpre (grid y 0), and dpost and a channel's dgate (1), from the sums over the parts of part[.][y][c], in order: 64 columns a
// workgroup, the parts cut over its sixteen waves. Bound: latency (512 parts of 4096 columns, 17 MB: 5.4 us; 2048 of 640 10 us).
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
#pragma unroll 16
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

// Threads of a row: eight values each up to 8192, sixteen beyond; up to 512 a power of two of a wave's lanes, else whole waves.
static int norm_threads(int H) { return H <= 8192 ? (H + 511) / 512 * 64 : 1024; }
static int norm_shift(int H) { return H <= 64 ? 3 : H <= 128 ? 4 : H <= 256 ? 5 : 6; }

// Tensors of 64 MB and more are marked as read once (us plain / marked, bf16 rows of 4096: 1237 rows 11.2 / 11.7, 8192 47.5 / 46.0,
// 16384 94.6 / 86.5; the gradient, which reads and writes more besides: no difference).
static bool norm_once(const NormArgs& a) { return a.rows * a.H * (a.dt == DT_F32 ? 4 : 2) >= (64 << 20); }

template <int DT>
static int run_norm(const NormArgs& a, hipStream_t st) {
    const int t = norm_threads(a.H), shift = norm_shift(a.H);
    const dim3 g = wide_grid(a.H <= 512 ? (a.rows + (256 >> shift) - 1) >> (8 - shift) : a.rows);
    if (a.H <= 512) hipLaunchKernelGGL((norm_kernel<DT, false, 1, false>), g, dim3(256), 0, st, a, shift);
    else if (a.H <= 8192 && norm_once(a)) hipLaunchKernelGGL((norm_kernel<DT, true, 1, true>), g, dim3(t), 0, st, a, 0);
    else if (a.H <= 8192) hipLaunchKernelGGL((norm_kernel<DT, true, 1, false>), g, dim3(t), 0, st, a, 0);
    else hipLaunchKernelGGL((norm_kernel<DT, true, 2, false>), g, dim3(t), 0, st, a, 0);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
int launch_norm(const NormArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_norm<DT_F32>(a, st) : a.dt == DT_BF16 ? run_norm<DT_BF16>(a, st) : run_norm<DT_F16>(a, st);
}

// Workgroups of the gradient, each with a part of the sums: what the card holds at once.
constexpr int NORM_WAVES = 16;                                       // a CU's
static int norm_parts(int64_t rows, int H) {
    if (H <= 512) return (int)std::min<int64_t>((rows + (256 >> norm_shift(H)) - 1) >> (8 - norm_shift(H)), 256 * NORM_WAVES / 4);
    return (int)std::min<int64_t>(rows, 256 * std::max(1, NORM_WAVES * 64 / norm_threads(H)));
}
int64_t norm_part_floats(int64_t rows, int H) { return (int64_t)norm_parts(rows, H) * 2 * H; }

template <int DT>
static int run_norm_grad(const NormArgs& a, hipStream_t st) {
    const dim3 g(norm_parts(a.rows, a.H));
    const int t = norm_threads(a.H);
    if (a.H <= 512) hipLaunchKernelGGL((norm_grad_kernel<DT, false>), g, dim3(256), 96 * 256, st, a, norm_shift(a.H));
    else if (a.H <= 8192) {
        if (!allow_lds<norm_grad_kernel<DT, true>>(96 * 1024)) return -1;
        hipLaunchKernelGGL((norm_grad_kernel<DT, true>), g, dim3(t), 96 * t, st, a, 0);
    } else {
        if (!allow_lds<norm_grad_long_kernel<DT>>(128 * 1024)) return -1;
        hipLaunchKernelGGL((norm_grad_long_kernel<DT>), g, dim3(t), 128 * t, st, a);
    }
    if (hipGetLastError() != hipSuccess) return -1;
    if (a.part) {
        hipLaunchKernelGGL(norm_join_kernel, dim3((a.H + 63) / 64, 2), dim3(1024), 0, st, a, norm_parts(a.rows, a.H));
        if (hipGetLastError() != hipSuccess) return -1;
    }
    return 0;
}
int launch_norm_grad(const NormArgs& a, hipStream_t st) {
    return a.dt == DT_F32 ? run_norm_grad<DT_F32>(a, st) : a.dt == DT_BF16 ? run_norm_grad<DT_BF16>(a, st) : run_norm_grad<DT_F16>(a, st);
}

}  // namespace mi355moe
