// row_io.cuh -- typed row access and warp reductions shared by the row
// kernels around the expert GEMMs (norm, routing, balance loss): bf16, fp16
// and fp32 elements are read into and written from fp32 registers.
#pragma once

#include <cuda_fp16.h>

#include "capi_internal.h"

namespace ferret {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// 16-byte load that leaves no line in L1 (data read once).  Not the read-only
// path: an output may be the same memory as an input.
__device__ __forceinline__ uint4 ld16_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// Eight consecutive elements <-> raw 16-byte words (one for 16-bit types, two
// for fp32).
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float v[8]) {
    T e[8];
    memcpy(e, r.w, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float v[8]) {
    T e[8];
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    memcpy(r.w, e, sizeof(e));
    return r;
}

// Four consecutive elements of a row, VEC: as one aligned load; else element by
// element with indices clamped into the row of n (the caller discards what lies
// behind it).
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* row, int at, int n, T v[4]) {
    if (VEC) {
        if (sizeof(T) == 4) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + min(at, n - 4)));
            memcpy(v, &w, 16);
        } else {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + min(at, n - 4)));
            memcpy(v, &w, 8);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = row[min(at + i, n - 1)];
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int at, int n, const float v[4]) {
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f32<T>(v[i]);
    if (VEC) {
        if (at >= n) return;
        if (sizeof(T) == 4) {
            uint4 w;
            memcpy(&w, e, 16);
            *reinterpret_cast<uint4*>(row + at) = w;
        } else {
            uint2 w;
            memcpy(&w, e, 8);
            *reinterpret_cast<uint2*>(row + at) = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n) row[at + i] = e[i];
    }
}

// Logits as the row kernels see them: NaN closes an expert like -inf, +inf is
// the largest finite value (so that differences stay defined).
__device__ __forceinline__ float clean_logit(float z) {
    return z > -INFINITY ? fminf(z, 3.402823466e38f) : -INFINITY;
}

// Reductions over the lanes of aligned groups of N lanes.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int N>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float warp_sum(float v) { return lanes_sum<32>(v); }
__device__ __forceinline__ float warp_max(float v) { return lanes_max<32>(v); }

}  // namespace

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline int dtype_size(int dtype) {
    return dtype == FERRET_FP32 ? 4 : dtype == FERRET_BF16 || dtype == FERRET_FP16 ? 2 : 0;
}

}  // namespace ferret
