// rms_norm.cu -- residual addition, root-mean-square norm and the FP8 rows of
// the expert GEMMs in one pass:
//
//   s = x + residual                    (fp32, never rounded on the way)
//   y = s * (mean(s^2) + eps)^(-1/2) * weight
//   residual_out = round(s), y_out = round(y)
//   per 128 columns: amax = max(max |y|, 1e-4), q = e4m3(y * f), scale = amax / 448
//
// with f and scale computed as the activation quantizer (quant_act.cu) does.
// Every output is rounded once, from the fp32 value: q comes from y itself,
// not from the rounded y_out.
//
// HBM-bound: a row's x and residual are read once, kept in registers across
// the reduction, and every output is written once (9 bytes per element with
// bf16 and all outputs).  One CTA (or one warp, for short rows) owns a row; a
// thread owns NV chunks of 8 consecutive columns, so a half-warp holds exactly
// one 128-column block and its amax takes four shuffles.
#include <algorithm>

#include "fp8_quant.cuh"
#include "row_io.cuh"

namespace ferret {
namespace {

constexpr int kNormMaxThreads = 1024;
constexpr int kNormMaxNV = 4;

struct NormArgs {
    const void* x;
    long long ldx;
    const void* residual;
    long long ldr;
    const void* weight;
    bool weight_f32;
    int T, K;
    float eps;
    void* y;
    void* residual_out;
    uint8_t* q;
    float* scale;
    bool ue8m0;
    int tpr;   // threads per row: 16, 32 or a multiple of 32 (then one row per CTA)
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float v[8]) {
    if (VEC) {
        Raw8<T> r;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
            r.w[i] = ld16_stream(reinterpret_cast<const uint4*>(p) + i);
        unpack8<T>(r, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float v[8]) {
    if (VEC) {
        const Raw8<T> r = pack8<T>(v);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_weight8(const NormArgs& a, int c, int n, float w[8]) {
    if (a.weight_f32 && sizeof(T) != 4) {
        const float* p = static_cast<const float*>(a.weight) + c * 8;
        if (VEC) {
            const float4 lo = __ldg(reinterpret_cast<const float4*>(p));
            const float4 hi = __ldg(reinterpret_cast<const float4*>(p) + 1);
            w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w;
            w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i < n ? p[i] : 0.0f;
        }
        return;
    }
    const T* p = static_cast<const T*>(a.weight) + c * 8;
    if (VEC) {
        Raw8<T> r;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
            r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        unpack8<T>(r, w);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
}

// VEC: K is a multiple of 8 and every row of x, residual, weight, y and
// residual_out starts on a 16-byte boundary; otherwise elements move one by one.
template <typename T, int NV, bool VEC>
__global__ void __launch_bounds__(kNormMaxThreads) add_rms_norm_kernel(const NormArgs a) {
    pdl_begin();
    __shared__ float warp_sums[kNormMaxThreads / 32];
    const int tpr = a.tpr, K = a.K;
    const int sub = tpr <= 32 ? threadIdx.x / tpr : 0;
    const int tid = tpr <= 32 ? threadIdx.x % tpr : threadIdx.x;
    const int per_cta = tpr <= 32 ? blockDim.x / tpr : 1;
    const long long row = (long long)blockIdx.x * per_cta + sub;
    const bool live = row < a.T;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* res = static_cast<const T*>(a.residual) + row * a.ldr;

    float v[NV][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = i * tpr + tid, n = live ? K - c * 8 : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (n <= 0) continue;
        load8<T, VEC>(x + c * 8, n, v[i]);
        if (a.residual) {
            float r[8];
            load8<T, VEC>(res + c * 8, n, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] += r[j];
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
    for (int o = min(tpr, 32) >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (tpr > 32) {
        if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = ss;
        __syncthreads();
        ss = (threadIdx.x & 31) < (tpr >> 5) ? warp_sums[threadIdx.x & 31] : 0.0f;
        ss = warp_sum(ss);
    }
    const float inv = 1.0f / sqrtf(ss / (float)K + a.eps);

    const int nk = K >> 7;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = i * tpr + tid, n = live ? K - c * 8 : 0;
        float y[8];
        float amax = 0.0f;
        if (n > 0) {
            if (a.residual_out)
                store8<T, VEC>(static_cast<T*>(a.residual_out) + row * K + c * 8, n, v[i]);
            float w[8];
            load_weight8<T, VEC>(a, c, n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = v[i][j] * inv * w[j];
            if (a.y) store8<T, VEC>(static_cast<T*>(a.y) + row * K + c * 8, n, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
        }
        if (!a.q) continue;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)          // within the 16 lanes of a 128-column block
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (n <= 0) continue;
        const Fp8Scale f = fp8_block_scale(amax, a.ue8m0);
        *reinterpret_cast<uint2*>(a.q + row * K + c * 8) = fp8_pack8(y, f.mul);
        if ((tid & 15) == 0) a.scale[row * nk + (c >> 4)] = f.scale;
    }
}

template <typename T, int NV>
int launch_norm(const NormArgs& a, bool vec, int threads, cudaStream_t s) {
    const int per_cta = a.tpr <= 32 ? threads / a.tpr : 1;
    const dim3 grid((unsigned)(((long long)a.T + per_cta - 1) / per_cta));
    return vec ? launch_kernel(add_rms_norm_kernel<T, NV, true>, grid, dim3(threads), 0, s, a)
               : launch_kernel(add_rms_norm_kernel<T, NV, false>, grid, dim3(threads), 0, s, a);
}

template <typename T>
int run_norm(NormArgs& a, bool vec, int sms, cudaStream_t s) {
    const int chunks = (a.K + 7) / 8;
    if (chunks <= 32 * kNormMaxNV && a.T > sms * 8) {
        // short rows, many of them: a warp (or half of one) per row, 8 warps per CTA
        const int nv = chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4;
        a.tpr = chunks <= 16 ? 16 : 32;
        return nv == 1   ? launch_norm<T, 1>(a, vec, 256, s)
               : nv == 2 ? launch_norm<T, 2>(a, vec, 256, s)
                         : launch_norm<T, 4>(a, vec, 256, s);
    }
    // few rows: one chunk per thread (shortest path through a row); many: more
    // chunks per thread, so that more rows are in flight on an SM
    int nv = a.T <= sms * 2 ? 1 : 2;
    while ((chunks + nv - 1) / nv > kNormMaxThreads) nv *= 2;
    a.tpr = std::max(64, ((chunks + nv - 1) / nv + 31) / 32 * 32);
    return nv == 1   ? launch_norm<T, 1>(a, vec, a.tpr, s)
           : nv == 2 ? launch_norm<T, 2>(a, vec, a.tpr, s)
                     : launch_norm<T, 4>(a, vec, a.tpr, s);
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" int ferret_add_rms_norm(const void* x, long long ldx, const void* residual,
                                   long long ldr, const void* weight, int weight_dtype, int dtype,
                                   int T, int K, float eps, void* y, void* residual_out,
                                   void* q_fp8, float* q_scale, int flags, void* stream) {
    const int size = dtype_size(dtype);
    if (!size || (weight_dtype != dtype && weight_dtype != FERRET_FP32)) return FERRET_ERR_SHAPE;
    if (T < 0 || K <= 0 || K > 8 * kNormMaxNV * kNormMaxThreads) return FERRET_ERR_SHAPE;
    if (q_fp8 && K % 128) return FERRET_ERR_SHAPE;
    if (ldx < K || (residual && ldr < K) || !(eps >= 0.0f)) return FERRET_ERR_SHAPE;
    if (T == 0) return FERRET_OK;
    if (!x || !weight || (!y && !q_fp8) || (q_fp8 && !q_scale) || (residual_out && !residual))
        return FERRET_ERR_NULL;
    if (!aligned_to(x, size) || !aligned_to(residual, size) || !aligned_to(y, size) ||
        !aligned_to(residual_out, size) || !aligned_to(weight, dtype_size(weight_dtype)) ||
        !aligned_to(q_fp8, 8) || !aligned_to(q_scale, 4))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    // 16-byte accesses need every row of every tensor on a 16-byte boundary
    const bool vec = K % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(y) &&
                     aligned16(residual_out) && aligned16(weight) && (ldx * size) % 16 == 0 &&
                     (!residual || (ldr * size) % 16 == 0);
    NormArgs a{x, ldx, residual, ldr, weight, weight_dtype == FERRET_FP32, T, K, eps, y,
               residual_out, static_cast<uint8_t*>(q_fp8), q_scale,
               (flags & FERRET_UE8M0_SCALES) != 0, 0};
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_norm<__nv_bfloat16>(a, vec, info->num_sms, s);
        case FERRET_FP16: return run_norm<__half>(a, vec, info->num_sms, s);
        default: return run_norm<float>(a, vec, info->num_sms, s);
    }
}
