// fp8_quant.cuh -- the 1x128 block scale and the e4m3 rounding of DeepGEMM's
// per_token_cast_to_fp8 (as called at
// baselines/fp8-group-gemm/baseline_dsv3_decode.py:42), one definition for
// every kernel that produces FP8 rows.  Every step is IEEE round-to-nearest.
#pragma once

#include "ferret_common.cuh"

namespace ferret {
namespace {

struct Fp8Scale {
    float mul;     // what the elements are multiplied with
    float scale;   // what dequantization multiplies with
};

// amax: the block's largest magnitude, clamped here at 1e-4.  ue8m0: the scale
// is the smallest power of two >= fl(amax / 448), taken from the fp32 bits
// (exact; no log2), and mul is its exact inverse.
__device__ __forceinline__ Fp8Scale fp8_block_scale(float amax, bool ue8m0) {
    amax = fmaxf(amax, 1e-4f);
    Fp8Scale r;
    if (ue8m0) {
        const uint32_t bits = __float_as_uint(__fdiv_rn(amax, 448.0f));
        const uint32_t ex = (bits >> 23) + ((bits & 0x7FFFFFu) ? 1u : 0u);
        r.scale = __uint_as_float(ex >= 255u ? 0x7F800000u : ex << 23);
        r.mul = ex >= 255u ? 0.0f : __uint_as_float(ex == 254u ? 0x00400000u : (254u - ex) << 23);
    } else {
        // `448.0 / amax` in the published torch code is reciprocal-then-multiply
        r.mul = __fmul_rn(__frcp_rn(amax), 448.0f);
        r.scale = __fdiv_rn(amax, 448.0f);
    }
    return r;
}

// Eight elements -> eight e4m3 bytes (round-to-nearest-even, saturating).
__device__ __forceinline__ uint2 fp8_pack8(const float v[8], float mul) {
    uint32_t packed[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(
            make_float2(__fmul_rn(v[4 * j], mul), __fmul_rn(v[4 * j + 1], mul)), __NV_SATFINITE,
            __NV_E4M3);
        const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(
            make_float2(__fmul_rn(v[4 * j + 2], mul), __fmul_rn(v[4 * j + 3], mul)),
            __NV_SATFINITE, __NV_E4M3);
        packed[j] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    return make_uint2(packed[0], packed[1]);
}

}  // namespace
}  // namespace ferret
