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
// bf16 and all outputs).  A thread owns NV chunks of 8 consecutive columns, so a
// half-warp holds exactly one 128-column block and its amax takes four shuffles.
//
// Two forms.  Few rows, short rows and rows off the 16-byte grid: one CTA (or
// one warp, for short rows) per row, loads straight to registers.  Many long
// rows: a persistent grid whose CTAs copy their next rows into a shared-memory
// ring with bulk copies while they work on the current one; between a row's
// loads and its stores lies a reduction, and without the ring the memory idles
// there.  B200, 32768 x 7168 bf16 with all outputs, on several boxes: 353-378 us, 5.6-6.0
// TB/s (0.86-0.92 of the measured copy rate), against 574 us without the ring; one row 6 us
// with the host's share, 1021 x 1001 fp16 5.1-5.9 us (10 us element by element).
//
// The sum of the squares is an fp32 sum: rows whose elements stay below 1e17 keep it finite.
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

// How a row's chunks of 8 columns are reached.
enum Rows {
    kElements,   // one by one
    kVectors,    // every row of every tensor starts on a 16-byte boundary
    kShifted,    // the rows of x, residual, y and residual_out share their distance from
                 // one: chunks start there, `shift` columns before the row, and only
                 // the row's two ends move one by one (and the weight, which stays in L1)
};

// Columns [at + lo, at + hi) of a chunk; hi <= lo: none.
struct Piece {
    int at, lo, hi;
    __device__ __forceinline__ Piece(int c, int shift, int K) {
        at = 8 * c - shift;
        lo = max(0, -at);
        hi = min(8, K - at);
    }
};

template <typename T, int ROWS>
__device__ __forceinline__ void load8(const T* row, const Piece& p, float v[8]) {
    if (ROWS != kElements && (ROWS == kVectors || p.hi - p.lo == 8)) {
        Raw8<T> r;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
            r.w[i] = ld16_stream(reinterpret_cast<const uint4*>(row + p.at) + i);
        unpack8<T>(r, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i >= p.lo && i < p.hi ? to_f32(row[p.at + i]) : 0.0f;
    }
}

template <typename T, int ROWS>
__device__ __forceinline__ void store8(T* row, const Piece& p, const float v[8]) {
    if (ROWS != kElements && (ROWS == kVectors || p.hi - p.lo == 8)) {
        const Raw8<T> r = pack8<T>(v);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
            reinterpret_cast<uint4*>(row + p.at)[i] = r.w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i >= p.lo && i < p.hi) row[p.at + i] = from_f32<T>(v[i]);
    }
}

template <typename W, bool VEC>
__device__ __forceinline__ void load_weight8(const W* w, const Piece& p, float v[8]) {
    if (VEC) {
        Raw8<W> r;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(W) / 2); ++i)
            r.w[i] = __ldg(reinterpret_cast<const uint4*>(w + p.at) + i);
        unpack8<W>(r, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i >= p.lo && i < p.hi ? to_f32(w[p.at + i]) : 0.0f;
    }
}

// The outputs of a row from its s (v) and the sum of its squares (ss).  All lanes
// of the warp take part; those without a live row or column store nothing.
template <typename T, int NV, int ROWS>
__device__ __forceinline__ void finish_row(const NormArgs& a, long long row, int tid, int shift,
                                           bool live, const float (&v)[NV][8], float ss) {
    const int tpr = a.tpr, K = a.K;
    const float inv = 1.0f / sqrtf(ss / (float)K + a.eps);
    const int nk = K >> 7;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = i * tpr + tid;
        const Piece p(c, shift, K);
        const bool some = live && p.hi > p.lo;
        float y[8];
        float amax = 0.0f;
        if (some) {
            if (a.residual_out)
                store8<T, ROWS>(static_cast<T*>(a.residual_out) + row * K, p, v[i]);
            float w[8];
            if (sizeof(T) != 4 && a.weight_f32)
                load_weight8<float, ROWS == kVectors>(static_cast<const float*>(a.weight), p, w);
            else
                load_weight8<T, ROWS == kVectors>(static_cast<const T*>(a.weight), p, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = v[i][j] * inv * w[j];
            if (a.y) store8<T, ROWS>(static_cast<T*>(a.y) + row * K, p, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
        }
        if (!a.q) continue;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)          // within the 16 lanes of a 128-column block
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (!some) continue;
        const Fp8Scale f = fp8_block_scale(amax, a.ue8m0);
        *reinterpret_cast<uint2*>(a.q + row * K + c * 8) = fp8_pack8(y, f.mul);
        if ((tid & 15) == 0) a.scale[row * nk + (c >> 4)] = f.scale;
    }
}

template <typename T, int NV, int ROWS>
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
    const int shift =
        ROWS == kShifted ? (int)(reinterpret_cast<uintptr_t>(x) & 15u) / (int)sizeof(T) : 0;

    float v[NV][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const Piece p(i * tpr + tid, shift, K);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (!live || p.hi <= p.lo) continue;
        load8<T, ROWS>(x, p, v[i]);
        if (a.residual) {
            float r[8];
            load8<T, ROWS>(res, p, r);
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
    finish_row<T, NV, ROWS>(a, row, tid, shift, live, v, ss);
}

// --------------------------------------------------------- the persistent form

constexpr int kRingMax = 4;

// Stage layout: x row, then the residual row (K elements each, 16-byte multiple).
template <typename T, int NV>
__global__ void __launch_bounds__(512) add_rms_norm_ring_kernel(const NormArgs a, int stages,
                                                                const DevCtl ctl) {
    pdl_begin();
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float warp_sums[2][16];
    __shared__ uint64_t full[kRingMax];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, tpr = a.tpr, K = a.K, lane = tid & 31;
    const uint32_t row_bytes = (uint32_t)K * sizeof(T);
    const uint32_t stage_bytes = a.residual ? 2 * row_bytes : row_bytes;
    if (tid == 0) {
        for (int i = 0; i < stages; ++i) mbar_init(smem_addr(&full[i]), 1);
        abort_flag = 0;
        mbar_init_fence();
    }
    __syncthreads();
    auto fetch = [&](int slot, long long row) {            // thread 0
        const uint32_t bar = smem_addr(&full[slot]), dst = smem_addr(ring) + slot * stage_bytes;
        mbar_expect_tx(bar, stage_bytes);
        const uint64_t policy = policy_evict_first();
        bulk_load_hint(dst, static_cast<const T*>(a.x) + row * a.ldx, row_bytes, bar, policy);
        if (a.residual)
            bulk_load_hint(dst + row_bytes, static_cast<const T*>(a.residual) + row * a.ldr,
                           row_bytes, bar, policy);
    };
    const long long step = gridDim.x;
    if (tid == 0)
        for (int i = 0; i < stages && blockIdx.x + i * step < a.T; ++i)
            fetch(i, blockIdx.x + i * step);

    RingPos pos;
    int odd = 0;
    for (long long row = blockIdx.x; row < a.T; row += step, odd ^= 1) {
        const bool ok = mbar_wait(smem_addr(&full[pos.slot]), pos.phase, &abort_flag, ctl, 22);
        const uint8_t* stage = ring + pos.slot * stage_bytes;
        float v[NV][8];
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = i * tpr + tid;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            if (c * 8 >= K) continue;
            Raw8<T> raw;
            const uint4* p = reinterpret_cast<const uint4*>(stage + (size_t)c * 8 * sizeof(T));
#pragma unroll
            for (int j = 0; j < (int)(sizeof(T) / 2); ++j) raw.w[j] = p[j];
            unpack8<T>(raw, v[i]);
            if (a.residual) {
                float r[8];
                p = reinterpret_cast<const uint4*>(stage + row_bytes + (size_t)c * 8 * sizeof(T));
#pragma unroll
                for (int j = 0; j < (int)(sizeof(T) / 2); ++j) raw.w[j] = p[j];
                unpack8<T>(raw, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] += r[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
        }
        ss = warp_sum(ss);
        if (lane == 0) warp_sums[odd][tid >> 5] = ss;
        // every thread has the row in registers: the stage is free again
        if (__syncthreads_or(!ok)) break;
        if (tid == 0 && row + stages * step < a.T) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            fetch(pos.slot, row + stages * step);
        }
        pos.advance(stages);
        ss = warp_sum(lane < (tpr >> 5) ? warp_sums[odd][lane] : 0.0f);
        finish_row<T, NV, kVectors>(a, row, tid, 0, true, v, ss);
    }
    // a wait ran out: the copies in flight land before the CTA leaves (slots
    // that hold no further row end this wait by its time limit)
    if (abort_flag && tid == 0)
        for (int i = 0; i < stages; ++i, pos.advance(stages))
            mbar_wait(smem_addr(&full[pos.slot]), pos.phase, &abort_flag, ctl, 22, false);
}

template <typename T, int NV>
int launch_norm(const NormArgs& a, Rows rows, int threads, cudaStream_t s) {
    const int per_cta = a.tpr <= 32 ? threads / a.tpr : 1;
    const dim3 grid((unsigned)(((long long)a.T + per_cta - 1) / per_cta)), block(threads);
    switch (rows) {
        case kVectors: return launch_kernel(add_rms_norm_kernel<T, NV, kVectors>, grid, block, 0, s, a);
        case kShifted: return launch_kernel(add_rms_norm_kernel<T, NV, kShifted>, grid, block, 0, s, a);
        default: return launch_kernel(add_rms_norm_kernel<T, NV, kElements>, grid, block, 0, s, a);
    }
}

template <typename T, int NV>
int launch_ring(const NormArgs& a, int ctas_per_sm, int stages, size_t smem, const DeviceInfo* info,
                cudaStream_t s) {
    auto kern = add_rms_norm_ring_kernel<T, NV>;
    if (smem > 40 * 1024 &&           // 48 KB less the static arrays need no opt-in
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
            cudaSuccess) {
        cudaGetLastError();
        return FERRET_ERR_CUDA;
    }
    const dim3 grid((unsigned)std::min<long long>(a.T, (long long)info->num_sms * ctas_per_sm));
    return launch_kernel(kern, grid, dim3(a.tpr), smem, s, a, stages, make_ctl(info));
}

template <typename T>
int run_norm(NormArgs& a, Rows rows, const DeviceInfo* info, cudaStream_t s) {
    // a shifted row may start late in its first chunk
    int chunks = (a.K + 7 + (rows == kShifted ? 16 / (int)sizeof(T) - 1 : 0)) / 8;
    if (chunks > kNormMaxNV * kNormMaxThreads) {
        rows = kElements;
        chunks = (a.K + 7) / 8;
    }
    const int sms = info->num_sms;
    if (chunks <= 32 * kNormMaxNV && a.T > sms * 8) {
        // short rows, many of them: a warp (or half of one) per row, 8 warps per CTA
        const int nv = chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4;
        a.tpr = chunks <= 16 ? 16 : 32;
        return nv == 1   ? launch_norm<T, 1>(a, rows, 256, s)
               : nv == 2 ? launch_norm<T, 2>(a, rows, 256, s)
                         : launch_norm<T, 4>(a, rows, 256, s);
    }
    // Many long rows: the ring, with at least three rows in it.  An SM has 1 KB of
    // shared memory more than a CTA may use; a CTA takes 1 KB besides its own.
    const size_t stage = (size_t)a.K * sizeof(T) * (a.residual ? 2 : 1);
    const int room = info->max_smem_optin + 1024, own = 1024 + 512;
    if (rows == kVectors && a.T > sms * 8 && chunks <= 2 * 512 && 3 * stage + own <= (size_t)room) {
        const int nv = chunks <= 256 ? 1 : 2;
        a.tpr = ((chunks + nv - 1) / nv + 31) / 32 * 32;
        const int ctas = std::min(2048 / a.tpr / 2, (int)(room / (3 * stage + own)));
        const int stages = std::min<int>(kRingMax, (int)((room / ctas - own) / stage));
        return nv == 1 ? launch_ring<T, 1>(a, ctas, stages, stage * stages, info, s)
                       : launch_ring<T, 2>(a, ctas, stages, stage * stages, info, s);
    }
    // few rows: one chunk per thread (shortest path through a row); many: more
    // chunks per thread, so that more rows are in flight on an SM
    int nv = a.T <= sms * 2 ? 1 : 2;
    while ((chunks + nv - 1) / nv > kNormMaxThreads) nv *= 2;
    a.tpr = std::max(64, ((chunks + nv - 1) / nv + 31) / 32 * 32);
    return nv == 1   ? launch_norm<T, 1>(a, rows, a.tpr, s)
           : nv == 2 ? launch_norm<T, 2>(a, rows, a.tpr, s)
                     : launch_norm<T, 4>(a, rows, a.tpr, s);
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
    auto off = [&](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16; };
    const bool together = (!residual || off(residual) == off(x)) && (!y || off(y) == off(x)) &&
                          (!residual_out || off(residual_out) == off(x));
    const size_t step = (size_t)K * size % 16;          // of the outputs' rows
    const bool same_step = (T == 1 || (size_t)ldx * size % 16 == step) &&
                           (!residual || T == 1 || (size_t)ldr * size % 16 == step);
    const Rows rows = together && same_step && off(x) == 0 && off(weight) == 0 && K % 8 == 0
                          ? kVectors
                      : together && same_step && !q_fp8 ? kShifted
                                                        : kElements;
    NormArgs a{x, ldx, residual, ldr, weight, weight_dtype == FERRET_FP32, T, K, eps, y,
               residual_out, static_cast<uint8_t*>(q_fp8), q_scale,
               (flags & FERRET_UE8M0_SCALES) != 0, 0};
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_norm<__nv_bfloat16>(a, rows, info, s);
        case FERRET_FP16: return run_norm<__half>(a, rows, info, s);
        default: return run_norm<float>(a, rows, info, s);
    }
}
