// Reading and writing rows of fp32, fp16 or bf16 values eight at a time, at any address of their type and any row length.
#pragma once
#include "common.cuh"
#include "mi355moe_internal.h"

namespace mi355moe {

// Vectors at any address of their element (the hardware takes global accesses at any byte address).
typedef uint32_t rows_u32x4 __attribute__((ext_vector_type(4), aligned(2)));

template <int DT>
__device__ __forceinline__ float row_value(const void* p, size_t i) {
    if constexpr (DT == DT_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == DT_BF16) return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
    else return (float)u16_as_h(static_cast<const uint16_t*>(p)[i]);
}
// One value of a type known at run time only.
__device__ __forceinline__ float any_value(const void* p, int dt, size_t i) {
    return dt == DT_F32 ? row_value<DT_F32>(p, i) : dt == DT_BF16 ? row_value<DT_BF16>(p, i) : row_value<DT_F16>(p, i);
}

__device__ __forceinline__ void unpack8_f32(u32x4 lo, u32x4 hi, float (&v)[8]) {
    const f32x4 a = __builtin_bit_cast(f32x4, lo), b = __builtin_bit_cast(f32x4, hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
}
__device__ __forceinline__ void unpack8_bf16(u32x4 w, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __builtin_bit_cast(float, w[j] << 16);
        v[2 * j + 1] = __builtin_bit_cast(float, w[j] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void unpack8_f16(u32x4 w, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = (float)u16_as_h(w[j] & 0xFFFFu);
        v[2 * j + 1] = (float)u16_as_h(w[j] >> 16);
    }
}

// v = values i .. i + 7 of p, of which the first n exist (n <= 0: none; what does not exist reads as zero).
template <int DT>
__device__ __forceinline__ void load8(const void* p, size_t i, int n, float (&v)[8]) {
    if (n >= 8) {
        if constexpr (DT == DT_F32) {
            const rows_u32x4* q = reinterpret_cast<const rows_u32x4*>(static_cast<const float*>(p) + i);
            unpack8_f32(q[0], q[1], v);
        } else {
            const u32x4 w = *reinterpret_cast<const rows_u32x4*>(static_cast<const uint16_t*>(p) + i);
            if constexpr (DT == DT_BF16) unpack8_bf16(w, v);
            else unpack8_f16(w, v);
        }
    } else
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? row_value<DT>(p, i + j) : 0.0f;
}
__device__ __forceinline__ void load8_any(const void* p, int dt, size_t i, int n, float (&v)[8]) {
    if (dt == DT_F32) load8<DT_F32>(p, i, n, v);
    else if (dt == DT_BF16) load8<DT_BF16>(p, i, n, v);
    else load8<DT_F16>(p, i, n, v);
}

// Two values rounded to a 16-bit type, packed lo | hi << 16.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (DT == DT_BF16) return pack_bf16x2(lo, hi);
    else return h_as_u16((_Float16)lo) | (h_as_u16((_Float16)hi) << 16);
}
// The first n of v to values i .. of p, rounded once.
template <int DT>
__device__ __forceinline__ void store8(void* p, size_t i, int n, const float (&v)[8]) {
    if constexpr (DT == DT_F32) {
        float* o = static_cast<float*>(p) + i;
        if (n >= 8) {
            reinterpret_cast<rows_u32x4*>(o)[0] = __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
            reinterpret_cast<rows_u32x4*>(o)[1] = __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]});
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) o[j] = v[j];
    } else {
        uint16_t* o = static_cast<uint16_t*>(p) + i;
        const u32x4 w = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
        if (n >= 8) *reinterpret_cast<rows_u32x4*>(o) = w;
        else
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) o[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
}
__device__ __forceinline__ void store_any(void* p, int dt, size_t i, float v) {
    if (dt == DT_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = (uint16_t)(dt == DT_BF16 ? pack2<DT_BF16>(v, 0.0f) : pack2<DT_F16>(v, 0.0f));
}

// A launch of n < 2^30 workgroups in a row. The runtime takes fewer than 2^32 threads a dimension, which 2^24 tokens of 256 threads
// pass: beyond 2^20 workgroups a second dimension counts on, and the last ones of a launch can lie behind n.
static inline dim3 wide_grid(int64_t n) {
    return n <= 1 << 20 ? dim3((unsigned)n) : dim3(1 << 20, (unsigned)((n + (1 << 20) - 1) >> 20));
}
__device__ __forceinline__ uint32_t wide_block() { return blockIdx.y * gridDim.x + blockIdx.x; }

// Eight values as they lie in memory: loaded first, made floats where they are used, so that a kernel's loads are all on their
// way before the first is waited for.
template <int DT>
struct Raw8 {
    u32x4 w[DT == DT_F32 ? 2 : 1];
    // ONCE: marked as read once, so that a stream larger than the caches does not push other lines out of them
    template <bool ONCE = false>
    __device__ __forceinline__ void load(const void* p, size_t i, int n) {
        if (n >= 8) {
            const rows_u32x4* q = reinterpret_cast<const rows_u32x4*>(static_cast<const unsigned char*>(p) + i * (DT == DT_F32 ? 4 : 2));
            w[0] = ONCE ? __builtin_nontemporal_load(q) : q[0];
            if constexpr (DT == DT_F32) w[1] = ONCE ? __builtin_nontemporal_load(q + 1) : q[1];
        } else {
            w[0] = u32x4{0, 0, 0, 0};
            if constexpr (DT == DT_F32) w[1] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (j < n) {
                    if constexpr (DT == DT_F32) w[j >> 2][j & 3] = static_cast<const uint32_t*>(p)[i + j];
                    else w[0][j >> 1] |= (uint32_t)static_cast<const uint16_t*>(p)[i + j] << (16 * (j & 1));
                }
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (DT == DT_F32) unpack8_f32(w[0], w[1], v);
        else if constexpr (DT == DT_BF16) unpack8_bf16(w[0], v);
        else unpack8_f16(w[0], v);
    }
};
// The same for a type known at run time only.
struct RawAny8 {
    u32x4 w[2];
    __device__ __forceinline__ void load(const void* p, int dt, size_t i, int n) {
        if (dt == DT_F32) {
            Raw8<DT_F32> r;
            r.load(p, i, n);
            w[0] = r.w[0], w[1] = r.w[1];
        } else {
            Raw8<DT_BF16> r;
            r.load(p, i, n);
            w[0] = r.w[0];
        }
    }
    __device__ __forceinline__ void get(int dt, float (&v)[8]) const {
        if (dt == DT_F32) unpack8_f32(w[0], w[1], v);
        else if (dt == DT_BF16) unpack8_bf16(w[0], v);
        else unpack8_f16(w[0], v);
    }
};

// The sum over a wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
    const int lane = threadIdx.x & 63;
    v += xor_lane<1>(v, lane);
    v += xor_lane<2>(v, lane);
    v += xor_lane<4>(v, lane);
    v += xor_lane<8>(v, lane);
    v += xor_lane<16>(v, lane);
    return v + xor_lane<32>(v, lane);
}

}  // namespace mi355moe
