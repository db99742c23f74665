// moe_balance.cu -- per-expert counts, probability sums and the balance loss
// of a routed batch, and the gradient of the logits.
//
// Over the V live tokens (token_mask, default all), with p_t the softmax of a
// token's logits (or its sigmoids divided by their sum), c_e the number of
// (token, slot) pairs routed to expert e and P_e = sum_t p_te:
//
//   loss   = coef * E / (topk * V^2) * sum_e c_e P_e
//   dz_te  = grad * coef * E / (topk * V^2) * p_te (c_e - sum_j c_j p_tj)   softmax
//            the same times (1 - sigmoid(z_te))                             sigmoid
//
// (counts are constants of the gradient).  A perfectly even batch has loss
// coef.  Ids outside [0, E) count for nothing; a masked token contributes to
// no output and gets a zero gradient row, whatever its logits hold.  Logits of
// -inf or NaN have p = 0.
//
// HBM-bound: forward reads the logits once; backward reads them once and writes
// the gradient once.  A warp takes a token at a time with its row in registers
// and sums probabilities for its 32 x VPL columns in registers over all its
// tokens, so the only reduction across CTAs is one [CTAs, E] table of partial
// sums and counts in the workspace.  A second launch adds its rows in CTA
// order: no floating-point atomics, the same bits every time.
#include <algorithm>

#include "row_io.cuh"

namespace ferret {
namespace {

constexpr int kBalWarps = 8;
constexpr int kBalThreads = kBalWarps * 32;
constexpr int kBalMaxE = 1024;
constexpr int kBalTokensPerWarp = 2;   // below this many a further CTA costs more than it saves

struct BalanceArgs {
    const void* logits;
    long long ld;
    const int32_t* ids;
    const uint8_t* mask;
    int T, E, topk;
    bool sigmoid;
    float* part_sums;     // [ctas, E]
    int32_t* part_counts; // [ctas, E]
    int32_t* part_live;   // [ctas]
};

// A token's probabilities in registers, column 32 k + lane (all zero for a row
// of closed logits), and the factor of the gradient that the scoring adds:
// 1 - sigmoid(z), or 1 for the softmax.
template <typename LT, int VPL>
__device__ __forceinline__ void row_probs(const LT* row, int E, bool sigmoid, float (&p)[VPL],
                                          float (&rest)[VPL]) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const int e = 32 * k + lane;
        const float z = e < E ? to_f32(row[e]) : -INFINITY;
        p[k] = z > -INFINITY ? fminf(z, 3.402823466e38f) : -INFINITY;
        m = fmaxf(m, p[k]);
    }
    float sum = 0.0f;
    if (sigmoid) {
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const float e = expf(-fabsf(p[k])), r = 1.0f / (1.0f + e);
            rest[k] = p[k] >= 0.0f ? e * r : r;
            p[k] = p[k] >= 0.0f ? r : e * r;      // -inf: e = 0
            sum += p[k];
        }
    } else {
        m = warp_max(m);
        const float shift = m > -INFINITY ? m : 0.0f;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            p[k] = expf(p[k] - shift);
            rest[k] = 1.0f;
            sum += p[k];
        }
    }
    sum = warp_sum(sum);
    if (sum < 0x1p-100f) {                        // sigmoids of far negative logits alone
#pragma unroll
        for (int k = 0; k < VPL; ++k) p[k] *= 0x1p100f;
        sum *= 0x1p100f;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) p[k] *= inv;
}

template <typename LT, int VPL>
__global__ void __launch_bounds__(kBalThreads) moe_balance_kernel(const BalanceArgs a) {
    pdl_begin();
    __shared__ float sums[kBalWarps][32 * VPL];
    __shared__ int counts[32 * VPL];
    __shared__ int live;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < 32 * VPL; e += kBalThreads) counts[e] = 0;
    if (threadIdx.x == 0) live = 0;
    __syncthreads();

    float acc[VPL];
#pragma unroll
    for (int k = 0; k < VPL; ++k) acc[k] = 0.0f;
    int mine = 0;
    for (long long t = (long long)blockIdx.x * kBalWarps + warp; t < a.T;
         t += (long long)gridDim.x * kBalWarps) {
        if (a.mask && !a.mask[t]) continue;
        ++mine;
        float p[VPL], rest[VPL];
        row_probs<LT, VPL>(static_cast<const LT*>(a.logits) + t * a.ld, a.E, a.sigmoid, p, rest);
#pragma unroll
        for (int k = 0; k < VPL; ++k) acc[k] += p[k];
        for (int j = lane; j < a.topk; j += 32) {
            const int e = a.ids[t * a.topk + j];
            if (e >= 0 && e < a.E) atomicAdd(&counts[e], 1);
        }
    }
#pragma unroll
    for (int k = 0; k < VPL; ++k) sums[warp][32 * k + lane] = acc[k];
    if (lane == 0 && mine) atomicAdd(&live, mine);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kBalThreads) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kBalWarps; ++w) s += sums[w][e];
        a.part_sums[(long long)blockIdx.x * a.E + e] = s;
        a.part_counts[(long long)blockIdx.x * a.E + e] = counts[e];
    }
    if (threadIdx.x == 0) a.part_live[blockIdx.x] = live;
}

// Adds the partial tables' rows in order and forms the loss.  One CTA: its
// threads split into groups of consecutive experts times slices of the rows.
__global__ void __launch_bounds__(1024)
    moe_balance_join_kernel(const float* __restrict__ part_sums,
                            const int32_t* __restrict__ part_counts,
                            const int32_t* __restrict__ part_live, int ctas, int E, int topk,
                            float coef, float* __restrict__ loss, int32_t* __restrict__ counts,
                            float* __restrict__ prob_sums, int32_t* __restrict__ n_tokens) {
    pdl_begin();
    __shared__ float s_sum[1024];
    __shared__ int s_cnt[1024];
    __shared__ double s_loss[32];
    __shared__ int s_live;
    const int tid = threadIdx.x;
    const int width = min(1024, (E + 31) / 32 * 32), slices = 1024 / width;
    const int e = tid % width, slice = tid / width;
    float s = 0.0f;
    int c = 0;
    if (tid == 0) s_live = 0;
    if (e < E && slice < slices) {
        const int lo = (int)((long long)ctas * slice / slices),
                  hi = (int)((long long)ctas * (slice + 1) / slices);
#pragma unroll 8
        for (int i = lo; i < hi; ++i) {
            s += part_sums[(long long)i * E + e];
            c += part_counts[(long long)i * E + e];
        }
    }
    s_sum[tid] = s;
    s_cnt[tid] = c;
    __syncthreads();
    int v = 0;
    for (int i = tid; i < ctas; i += 1024) v += part_live[i];
    if (v) atomicAdd(&s_live, v);
    double part = 0.0;
    if (tid < E) {
        s = 0.0f;
        c = 0;
        for (int i = 0; i < slices; ++i) {
            s += s_sum[i * width + tid];
            c += s_cnt[i * width + tid];
        }
        prob_sums[tid] = s;
        counts[tid] = c;
        part = (double)c * (double)s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if ((tid & 31) == 0) s_loss[tid >> 5] = part;
    __syncthreads();
    if (tid == 0) {
        double total = 0.0;
        for (int i = 0; i < 32; ++i) total += s_loss[i];
        const double n = s_live;
        *n_tokens = s_live;
        *loss = s_live ? (float)((double)coef * E / (topk * n * n) * total) : 0.0f;
    }
}

struct BalanceBwdArgs {
    const float* grad_loss;
    const void* logits;
    long long ld;
    const int32_t* counts;
    const int32_t* n_tokens;
    const uint8_t* mask;
    int T, E, topk;
    float coef;
    bool sigmoid;
    void* dlogits;
};

template <typename LT, int VPL>
__global__ void __launch_bounds__(kBalThreads) moe_balance_bwd_kernel(const BalanceBwdArgs a) {
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // Since sum_e p_e = 1, c may be taken relative to any constant; relative
    // to its mean the difference below loses no digits to the common part.
    float c[VPL];
    double mean = 0.0;
#pragma unroll
    for (int k = 0; k < VPL; ++k)
        if (32 * k + lane < a.E) mean += a.counts[32 * k + lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    mean /= a.E;
#pragma unroll
    for (int k = 0; k < VPL; ++k)
        c[k] = 32 * k + lane < a.E ? (float)(a.counts[32 * k + lane] - mean) : 0.0f;
    const double n = *a.n_tokens;
    const float factor =
        n > 0 ? (float)((double)*a.grad_loss * a.coef * a.E / (a.topk * n * n)) : 0.0f;

    for (long long t = (long long)blockIdx.x * kBalWarps + warp; t < a.T;
         t += (long long)gridDim.x * kBalWarps) {
        LT* out = static_cast<LT*>(a.dlogits) + t * a.E;
        if (a.mask && !a.mask[t]) {
            for (int e = lane; e < a.E; e += 32) out[e] = from_f32<LT>(0.0f);
            continue;
        }
        float p[VPL], rest[VPL];
        row_probs<LT, VPL>(static_cast<const LT*>(a.logits) + t * a.ld, a.E, a.sigmoid, p, rest);
        float inner = 0.0f;
#pragma unroll
        for (int k = 0; k < VPL; ++k) inner = fmaf(p[k], c[k], inner);
        inner = warp_sum(inner);
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if (32 * k + lane < a.E)
                out[32 * k + lane] = from_f32<LT>(p[k] * rest[k] * (c[k] - inner) * factor);
    }
}

int balance_ctas(int T, int sms) {
    const int want = (int)(((long long)T + kBalWarps * kBalTokensPerWarp - 1) /
                           (kBalWarps * kBalTokensPerWarp));
    return std::max(1, std::min(want, sms * 2));
}

// The workspace is sized for the largest device this library runs on, so that
// the size needs no device: sums and counts [ctas, E], live tokens [ctas].
constexpr int kBalMaxCtas = 2 * 256;

template <typename LT>
int run_balance(const BalanceArgs& a, int ctas, cudaStream_t s) {
    const dim3 grid(ctas), block(kBalThreads);
    const int vpl = (a.E + 31) / 32;
    if (vpl <= 2) return launch_kernel(moe_balance_kernel<LT, 2>, grid, block, 0, s, a);
    if (vpl <= 4) return launch_kernel(moe_balance_kernel<LT, 4>, grid, block, 0, s, a);
    if (vpl <= 8) return launch_kernel(moe_balance_kernel<LT, 8>, grid, block, 0, s, a);
    if (vpl <= 16) return launch_kernel(moe_balance_kernel<LT, 16>, grid, block, 0, s, a);
    return launch_kernel(moe_balance_kernel<LT, 32>, grid, block, 0, s, a);
}

template <typename LT>
int run_balance_bwd(const BalanceBwdArgs& a, int ctas, cudaStream_t s) {
    const dim3 grid(ctas), block(kBalThreads);
    const int vpl = (a.E + 31) / 32;
    if (vpl <= 2) return launch_kernel(moe_balance_bwd_kernel<LT, 2>, grid, block, 0, s, a);
    if (vpl <= 4) return launch_kernel(moe_balance_bwd_kernel<LT, 4>, grid, block, 0, s, a);
    if (vpl <= 8) return launch_kernel(moe_balance_bwd_kernel<LT, 8>, grid, block, 0, s, a);
    if (vpl <= 16) return launch_kernel(moe_balance_bwd_kernel<LT, 16>, grid, block, 0, s, a);
    return launch_kernel(moe_balance_bwd_kernel<LT, 32>, grid, block, 0, s, a);
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" size_t ferret_moe_balance_loss_workspace_size(int T, int E) {
    if (T <= 0 || E <= 0 || E > kBalMaxE) return 0;
    return (size_t)balance_ctas(T, kBalMaxCtas / 2) * (2 * (size_t)E + 1) * 4;
}

extern "C" int ferret_moe_balance_loss(const void* logits, long long ld, int dtype,
                                       const int32_t* topk_ids, const uint8_t* token_mask, int T,
                                       int E, int topk, float coef, int flags, float* loss,
                                       int32_t* counts, float* prob_sums, int32_t* n_tokens,
                                       void* workspace, size_t ws_bytes, void* stream) {
    const int size = dtype_size(dtype);
    if (!size || T < 0 || E <= 0 || E > kBalMaxE || topk <= 0 || ld < E ||
        (long long)T * topk >= (1ll << 31))
        return FERRET_ERR_SHAPE;
    if (!loss || !counts || !prob_sums || !n_tokens || (T > 0 && (!logits || !topk_ids)))
        return FERRET_ERR_NULL;
    if (!aligned_to(logits, size) || !aligned_to(topk_ids, 4) || !aligned_to(loss, 4) ||
        !aligned_to(counts, 4) || !aligned_to(prob_sums, 4) || !aligned_to(n_tokens, 4) ||
        !aligned_to(workspace, 4))
        return FERRET_ERR_ALIGN;
    if (T > 0 && (!workspace || ws_bytes < ferret_moe_balance_loss_workspace_size(T, E)))
        return FERRET_ERR_WORKSPACE;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    const cudaStream_t s = as_stream(stream);
    const int ctas = T ? balance_ctas(T, std::min(info->num_sms, kBalMaxCtas / 2)) : 0;
    float* sums = static_cast<float*>(workspace);
    int32_t* cnts = reinterpret_cast<int32_t*>(sums + (size_t)ctas * E);
    int32_t* live = cnts + (size_t)ctas * E;
    if (T) {
        const BalanceArgs a{logits, ld, topk_ids, token_mask, T, E, topk,
                            (flags & FERRET_ROUTE_SIGMOID) != 0, sums, cnts, live};
        rc = dtype == FERRET_BF16   ? run_balance<__nv_bfloat16>(a, ctas, s)
             : dtype == FERRET_FP16 ? run_balance<__half>(a, ctas, s)
                                    : run_balance<float>(a, ctas, s);
        if (rc != FERRET_OK) return rc;
    }
    return launch_kernel(moe_balance_join_kernel, dim3(1), dim3(1024), 0, s, sums, cnts, live, ctas,
                         E, topk, coef, loss, counts, prob_sums, n_tokens);
}

extern "C" int ferret_moe_balance_loss_backward(const float* grad_loss, const void* logits,
                                                long long ld, int dtype, const int32_t* counts,
                                                const int32_t* n_tokens, const uint8_t* token_mask,
                                                int T, int E, int topk, float coef, int flags,
                                                void* grad_logits, void* stream) {
    const int size = dtype_size(dtype);
    if (!size || T < 0 || E <= 0 || E > kBalMaxE || topk <= 0 || ld < E) return FERRET_ERR_SHAPE;
    if (T == 0) return FERRET_OK;
    if (!grad_loss || !logits || !counts || !n_tokens || !grad_logits) return FERRET_ERR_NULL;
    if (!aligned_to(grad_loss, 4) || !aligned_to(logits, size) || !aligned_to(counts, 4) ||
        !aligned_to(n_tokens, 4) || !aligned_to(grad_logits, size))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    const BalanceBwdArgs a{grad_loss, logits, ld, counts, n_tokens, token_mask, T, E, topk, coef,
                           (flags & FERRET_ROUTE_SIGMOID) != 0, grad_logits};
    const int ctas = (int)std::min<long long>(((long long)T + kBalWarps - 1) / kBalWarps,
                                              (long long)info->num_sms * 8);
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_balance_bwd<__nv_bfloat16>(a, ctas, s);
        case FERRET_FP16: return run_balance_bwd<__half>(a, ctas, s);
        default: return run_balance_bwd<float>(a, ctas, s);
    }
}
