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
// the gradient once.  LPT lanes share a token's row, NV vectors of 4 columns
// each, and the next token's row is loaded before the current one is used.  The
// forward kernel sums probabilities for its columns in registers over all its
// tokens, so the only reduction across CTAs is one [CTAs, E] table of partial
// sums and counts in the workspace.  A second launch (128 columns per CTA, one
// cluster) adds its rows in a fixed order: no floating-point atomics, the same
// bits every time.
#include <algorithm>
#include <cooperative_groups.h>

#include "row_io.cuh"

namespace ferret {
namespace {

namespace cg = cooperative_groups;

constexpr int kBalWarps = 8;
constexpr int kBalThreads = kBalWarps * 32;
constexpr int kBalMaxE = 1024;
constexpr int kBalMaxCtas = 256 * 4;   // partial rows, on the largest device

struct BalanceArgs {
    const void* logits;
    long long ld;
    const int32_t* ids;
    const uint8_t* mask;
    int T, E, topk;
    bool sigmoid;
    float* part_sums;     // [ctas, stride]: stride is E, rounded up to whole vectors
    int32_t* part_counts; // [ctas, stride]
    int32_t* part_live;   // [ctas]
    int stride;
};

// A row's pieces as loaded: vector i of a lane holds columns 4 (LPT i + lane) ..+3.
template <typename LT, int NV>
struct RowRaw {
    LT e[NV][4];
};

template <typename LT, int LPT, int NV, bool VEC>
__device__ __forceinline__ RowRaw<LT, NV> load_row(const LT* row, int E) {
    RowRaw<LT, NV> r;
    const int sub = threadIdx.x % LPT;
#pragma unroll
    for (int i = 0; i < NV; ++i) load4<LT, VEC>(row, 4 * (LPT * i + sub), E, r.e[i]);
    return r;
}

// Its probabilities (all zero for a row of closed logits), and the factor that
// the scoring adds to the gradient: 1 - sigmoid(z), or 1 for the softmax.
template <typename LT, int LPT, int NV>
__device__ __forceinline__ void row_probs(const RowRaw<LT, NV>& r, int E, bool sigmoid,
                                          float (&p)[NV][4], float (&rest)[NV][4]) {
    const int sub = threadIdx.x % LPT;
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float z = clean_logit(to_f32(r.e[i][k]));
            p[i][k] = 4 * (LPT * i + sub) + k < E ? z : -INFINITY;
            m = fmaxf(m, p[i][k]);
        }
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = p[i][k], e = expf(-fabsf(z)), inv = 1.0f / (1.0f + e);
                rest[i][k] = z >= 0.0f ? e * inv : inv;
                p[i][k] = z >= 0.0f ? inv : e * inv;      // -inf: e = 0
                sum += p[i][k];
            }
    } else {
        m = lanes_max<LPT>(m);
        const float shift = m > -INFINITY ? m : 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                p[i][k] = expf(p[i][k] - shift);
                rest[i][k] = 1.0f;
                sum += p[i][k];
            }
    }
    sum = lanes_sum<LPT>(sum);
    float scale = 1.0f;
    if (sum < 0x1p-100f) scale = 0x1p100f;        // sigmoids of far negative logits alone
    sum *= scale;
    scale = sum > 0.0f ? scale / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) p[i][k] *= scale;
}

template <typename LT, int LPT, int NV, bool VEC>
__global__ void __launch_bounds__(kBalThreads) moe_balance_kernel(const BalanceArgs a) {
    pdl_begin();
    constexpr int kCols = LPT * NV * 4, kSubs = kBalThreads / LPT;
    __shared__ float sums[kBalWarps][kCols];
    __shared__ int counts[kCols];
    __shared__ int live;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = threadIdx.x / LPT;
    // this CTA's tokens, a contiguous run
    const int t0 = (int)((long long)a.T * blockIdx.x / gridDim.x);
    const int t1 = (int)((long long)a.T * (blockIdx.x + 1) / gridDim.x);
    const LT* logits = static_cast<const LT*>(a.logits);
    auto row_of = [&](int t) { return logits + (long long)min(t, t1 - 1) * a.ld; };
    RowRaw<LT, NV> next = load_row<LT, LPT, NV, VEC>(row_of(t0 + sub), a.E);

    for (int e = threadIdx.x; e < kCols; e += kBalThreads) counts[e] = 0;
    if (threadIdx.x == 0) live = 0;
    __syncthreads();
    const long long first = (long long)t0 * a.topk, pairs = (long long)(t1 - t0) * a.topk;
    for (long long i = threadIdx.x; i < pairs; i += kBalThreads) {
        const int e = a.ids[first + i];
        if (e >= 0 && e < a.E && (!a.mask || a.mask[t0 + (int)(i / a.topk)]))
            atomicAdd(&counts[e], 1);
    }

    float acc[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[i][k] = 0.0f;
    int mine = 0;
    const int rounds = (t1 - t0 + kSubs - 1) / kSubs;
    for (int n = 0; n < rounds; ++n) {
        const int t = t0 + n * kSubs + sub;
        const RowRaw<LT, NV> row = next;
        if (n + 1 < rounds) next = load_row<LT, LPT, NV, VEC>(row_of(t + kSubs), a.E);
        const bool counted = t < t1 && (!a.mask || a.mask[t]);
        mine += counted;
        float p[NV][4], rest[NV][4];
        row_probs<LT, LPT, NV>(row, a.E, a.sigmoid, p, rest);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][k] += counted ? p[i][k] : 0.0f;
    }
#pragma unroll
    for (int o = LPT; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][k] += __shfl_xor_sync(0xffffffffu, acc[i][k], o);
    if (lane < LPT)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) sums[warp][4 * (LPT * i + lane) + k] = acc[i][k];
    if (threadIdx.x % LPT == 0 && mine) atomicAdd(&live, mine);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kBalThreads) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kBalWarps; ++w) s += sums[w][e];
        a.part_sums[(long long)blockIdx.x * a.stride + e] = s;
        a.part_counts[(long long)blockIdx.x * a.stride + e] = counts[e];
    }
    if (threadIdx.x == 0) a.part_live[blockIdx.x] = live;
}

// Adds the partial tables' rows in a fixed order and forms the loss.  A CTA
// takes 128 columns, 4 adjacent ones per lane; warp w adds rows w, w + 32, ..., four of
// them in flight at a time.
constexpr int kJoinThreads = 1024;
constexpr int kJoinCols = 128;
constexpr int kJoinAhead = 4;

__global__ void __launch_bounds__(kJoinThreads)
    moe_balance_join_kernel(const float* part_sums, const int32_t* part_counts,
                            const int32_t* part_live, int ctas, int stride, int E, int topk,
                            float coef, float* loss, int32_t* counts, float* prob_sums,
                            int32_t* n_tokens) {
    pdl_begin();
    __shared__ __align__(16) float s_sum[32][kJoinCols];
    __shared__ __align__(16) int s_cnt[32][kJoinCols];
    __shared__ int s_live[32];
    __shared__ double s_loss[kJoinCols / 32];
    __shared__ double cta_loss;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int e0 = blockIdx.x * kJoinCols;
    const int at = min(e0 + 4 * lane, stride - 4);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int c[4] = {0, 0, 0, 0};
    for (int i = warp; i < ctas; i += 32 * kJoinAhead) {
        float4 f[kJoinAhead];
        int4 n[kJoinAhead];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const long long row = (long long)min(i + 32 * j, ctas - 1) * stride + at;
            f[j] = *reinterpret_cast<const float4*>(part_sums + row);
            n[j] = *reinterpret_cast<const int4*>(part_counts + row);
        }
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            if (i + 32 * j >= ctas) break;
            s[0] += f[j].x, s[1] += f[j].y, s[2] += f[j].z, s[3] += f[j].w;
            c[0] += n[j].x, c[1] += n[j].y, c[2] += n[j].z, c[3] += n[j].w;
        }
    }
    *reinterpret_cast<float4*>(&s_sum[warp][4 * lane]) = make_float4(s[0], s[1], s[2], s[3]);
    *reinterpret_cast<int4*>(&s_cnt[warp][4 * lane]) = make_int4(c[0], c[1], c[2], c[3]);
    int v = 0;
    for (int i = tid; i < ctas; i += kJoinThreads) v += part_live[i];
    v = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) s_live[warp] = v;
    __syncthreads();
    double part = 0.0;
    if (tid < kJoinCols) {
        float sum = 0.0f;
        int cnt = 0;
#pragma unroll
        for (int w = 0; w < 32; ++w) {
            sum += s_sum[w][tid];
            cnt += s_cnt[w][tid];
        }
        if (e0 + tid < E) {
            prob_sums[e0 + tid] = sum;
            counts[e0 + tid] = cnt;
            part = (double)cnt * (double)sum;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
        if (lane == 0) s_loss[warp] = part;
    }
    __syncthreads();
    if (tid == 0) {
        cta_loss = 0.0;
        for (int i = 0; i < kJoinCols / 32; ++i) cta_loss += s_loss[i];
    }
    const int ranks = (int)cluster.num_blocks();
    if (ranks > 1)
        cluster.sync();
    else
        __syncthreads();
    if (blockIdx.x == 0 && warp == 0) {
        const int live = __reduce_add_sync(0xffffffffu, s_live[lane]);
        double total = 0.0;
        for (int k = 0; k < ranks; ++k) total += *cluster.map_shared_rank(&cta_loss, k);
        const double n = live;
        if (lane == 0) {
            *n_tokens = live;
            *loss = live ? (float)((double)coef * E * total / (topk * n * n)) : 0.0f;
        }
    }
    if (ranks > 1) cluster.sync();      // CTA 0 may still read the others' sums
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

template <typename LT, int LPT, int NV, bool VEC>
__global__ void __launch_bounds__(kBalThreads) moe_balance_bwd_kernel(const BalanceBwdArgs a) {
    pdl_begin();
    constexpr int kSubs = kBalThreads / LPT;
    const int sub = threadIdx.x / LPT, col = threadIdx.x % LPT;
    const LT* logits = static_cast<const LT*>(a.logits);
    auto row_of = [&](long long t) { return logits + min(t, (long long)a.T - 1) * a.ld; };
    const long long step = (long long)gridDim.x * kSubs;
    const long long t0 = (long long)blockIdx.x * kSubs + sub;
    RowRaw<LT, NV> next = load_row<LT, LPT, NV, VEC>(row_of(t0), a.E);

    // Since sum_e p_e = 1, c may be taken relative to any constant; relative
    // to its mean (to an integer) the difference below loses no digits to the
    // part that all counts share.
    float c[NV][4];
    int ci[NV][4];
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = 4 * (LPT * i + col) + k;
            ci[i][k] = a.counts[min(e, a.E - 1)];
            total += e < a.E ? (float)ci[i][k] : 0.0f;
        }
    const int mean = (int)(lanes_sum<LPT>(total) / (float)a.E);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) c[i][k] = (float)(ci[i][k] - mean);
    const float n = (float)*a.n_tokens;
    const float factor = n > 0.0f ? *a.grad_loss * a.coef * (float)a.E / (float)a.topk / n / n : 0.0f;

    const long long rounds = (a.T - (long long)blockIdx.x * kSubs + step - 1) / step;
    for (long long i0 = 0; i0 < rounds; ++i0) {
        const long long t = t0 + i0 * step;
        const RowRaw<LT, NV> row = next;
        if (i0 + 1 < rounds) next = load_row<LT, LPT, NV, VEC>(row_of(t + step), a.E);
        const bool live = t < a.T && (!a.mask || a.mask[t]);
        float p[NV][4], rest[NV][4];
        row_probs<LT, LPT, NV>(row, a.E, a.sigmoid, p, rest);
        float inner = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) inner = fmaf(p[i][k], c[i][k], inner);
        inner = lanes_sum<LPT>(inner);
        if (t >= a.T) continue;
        LT* out = static_cast<LT*>(a.dlogits) + t * a.E;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float d[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                d[k] = live ? p[i][k] * rest[i][k] * (c[i][k] - inner) * factor : 0.0f;
            store4<LT, VEC>(out, 4 * (LPT * i + col), a.E, d);
        }
    }
}

// Lanes per token and vectors per lane: the fewest lanes that hold a row in one
// vector each, and from 128 columns on the whole warp.
#define FERRET_BALANCE_SHAPE(KERNEL, LT, VEC, E, ...)                                   \
    ((E) <= 32    ? launch_kernel(KERNEL<LT, 8, 1, VEC>, __VA_ARGS__)                   \
     : (E) <= 64  ? launch_kernel(KERNEL<LT, 16, 1, VEC>, __VA_ARGS__)                  \
     : (E) <= 128 ? launch_kernel(KERNEL<LT, 32, 1, VEC>, __VA_ARGS__)                  \
     : (E) <= 256 ? launch_kernel(KERNEL<LT, 32, 2, VEC>, __VA_ARGS__)                  \
     : (E) <= 512 ? launch_kernel(KERNEL<LT, 32, 4, VEC>, __VA_ARGS__)                  \
                  : launch_kernel(KERNEL<LT, 32, 8, VEC>, __VA_ARGS__))

// Tokens that a CTA works on at once.
int balance_tokens(int E) { return kBalThreads / (E <= 32 ? 8 : E <= 64 ? 16 : 32); }

// Four rounds of tokens per CTA before a further CTA pays (the second launch reads a
// row for every CTA), four CTAs per SM at most.
int balance_ctas(int T, int E, int sms) {
    const int per = 4 * balance_tokens(E);
    return std::max(1, std::min((int)(((long long)T + per - 1) / per), sms * 4));
}

int balance_stride(int E) { return (E + 3) / 4 * 4; }

// Vector accesses: rows of whole vectors, each on a vector's boundary.
bool balance_vec(const void* logits, long long ld, int E, int size, const void* out) {
    return E % 4 == 0 && ld % 4 == 0 && aligned_to(logits, 4 * size) && aligned_to(out, 4 * size);
}

template <typename LT>
int run_balance(const BalanceArgs& a, int ctas, cudaStream_t s) {
    const dim3 grid(ctas), block(kBalThreads);
    return balance_vec(a.logits, a.ld, a.E, sizeof(LT), nullptr)
               ? FERRET_BALANCE_SHAPE(moe_balance_kernel, LT, true, a.E, grid, block, 0, s, a)
               : FERRET_BALANCE_SHAPE(moe_balance_kernel, LT, false, a.E, grid, block, 0, s, a);
}

template <typename LT>
int run_balance_bwd(const BalanceBwdArgs& a, int sms, cudaStream_t s) {
    const int per = balance_tokens(a.E);
    const dim3 grid((unsigned)std::min<long long>(((long long)a.T + per - 1) / per, sms * 6LL)),
        block(kBalThreads);
    return balance_vec(a.logits, a.ld, a.E, sizeof(LT), a.dlogits)
               ? FERRET_BALANCE_SHAPE(moe_balance_bwd_kernel, LT, true, a.E, grid, block, 0, s, a)
               : FERRET_BALANCE_SHAPE(moe_balance_bwd_kernel, LT, false, a.E, grid, block, 0, s, a);
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" size_t ferret_moe_balance_loss_workspace_size(int T, int E) {
    if (T <= 0 || E <= 0 || E > kBalMaxE) return 0;
    return (size_t)balance_ctas(T, E, kBalMaxCtas / 4) * (2 * (size_t)balance_stride(E) + 1) * 4;
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
        !aligned16(workspace))
        return FERRET_ERR_ALIGN;
    if (T > 0 && (!workspace || ws_bytes < ferret_moe_balance_loss_workspace_size(T, E)))
        return FERRET_ERR_WORKSPACE;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    const cudaStream_t s = as_stream(stream);
    const int ctas = T ? balance_ctas(T, E, std::min(info->num_sms, kBalMaxCtas / 4)) : 0;
    float* sums = static_cast<float*>(workspace);
    const int stride = balance_stride(E);
    int32_t* cnts = reinterpret_cast<int32_t*>(sums + (size_t)ctas * stride);
    int32_t* live = cnts + (size_t)ctas * stride;
    if (T) {
        const BalanceArgs a{logits, ld, topk_ids, token_mask, T, E, topk,
                            (flags & FERRET_ROUTE_SIGMOID) != 0, sums, cnts, live, stride};
        rc = dtype == FERRET_BF16   ? run_balance<__nv_bfloat16>(a, ctas, s)
             : dtype == FERRET_FP16 ? run_balance<__half>(a, ctas, s)
                                    : run_balance<float>(a, ctas, s);
        if (rc != FERRET_OK) return rc;
    }
    const int join = (E + kJoinCols - 1) / kJoinCols;        // at most 8: one cluster
    return launch_kernel_cluster(moe_balance_join_kernel, dim3(join), dim3(kJoinThreads), 0, join,
                                 s, sums, cnts, live, ctas, stride, E, topk, coef, loss, counts,
                                 prob_sums, n_tokens);
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
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_balance_bwd<__nv_bfloat16>(a, info->num_sms, s);
        case FERRET_FP16: return run_balance_bwd<__half>(a, info->num_sms, s);
        default: return run_balance_bwd<float>(a, info->num_sms, s);
    }
}
