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
// -inf or NaN have p = 0; so has, with sigmoids, a row of nothing but the type's
// lowest finite value (a mask that leaves nothing).
//
// HBM-bound: forward reads the logits once; backward reads them once and writes
// the gradient once.  LPT lanes share a token's row, NV vectors of 4 columns
// each, and the next token's row is loaded before the current one is used.  The
// forward kernel sums probabilities for its columns in registers over all its
// tokens, so the only reduction across CTAs is one [CTAs, E] table of partial
// sums and counts in the workspace.  A second launch (32 columns per CTA) adds its
// rows in a fixed order, and the CTA that finishes last adds the CTAs' shares of the
// loss: no floating-point atomics, the same bits every time.
//
// B200, 32768 x 256 fp32, loss and gradient: 30.7 us (floor 10.4; forward with its join
// 17.8, backward 12.0 apart), with sigmoids 31.8, with every row below -87 46.  The
// exponentials and the row sums bound the two large kernels (issue slots 64 % busy in
// both, DRAM under 30 %); four resident CTAs per SM, one wave of each.
#include <algorithm>
#include <type_traits>

#include "row_io.cuh"

namespace ferret {
namespace {

constexpr int kBalWarps = 8;
constexpr int kBalThreads = kBalWarps * 32;
constexpr int kBalMaxE = 1024;
constexpr int kBalMaxCtas = 256 * 4;   // partial rows, on the largest device (the join reads 1024)

struct BalanceArgs {
    const void* logits;
    long long ld;
    const int32_t* ids;
    const uint8_t* mask;
    int T, E, topk;
    float* part_sums;     // [ctas, E]
    int32_t* part_counts; // [ctas, E]
    int32_t* part_live;   // [ctas]
    int32_t* done;        // CTAs of the second launch that are through: zeroed here
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

// e^v as ex2(v log2(e)): the approximation (relative error 2^-22), and an exponent that
// the rounding of the product and of log2(e) moves by up to 1.25 |v| 2^-24 (expf's
// own steps would cost 8 % of the kernels' time).  Results below 2^-126 are 0.
__device__ __forceinline__ float exp_fast(float v) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * 1.44269504f));
    return e;
}

// The lowest finite value of a type: what a mask may put in place of -inf.
template <typename LT>
__device__ __forceinline__ float lowest() {
    return sizeof(LT) == 4 ? -3.402823466e38f
           : std::is_same<LT, __half>::value ? -65504.0f : -3.389531389e38f;
}

// Its probabilities (all zero for a row of closed logits), and the factor that
// the scoring adds to the gradient: 1 - sigmoid(z), or 1 for the softmax.  `row` is where
// the row was loaded from.
//
// Sigmoids of far negative logits underflow, their quotients do not.  Where a row's
// sigmoids add up to less than 1/2, all of its logits are negative, and it is read again
// and every sigmoid taken times e^-m, m the row's largest logit: e^(z - m) / (1 + e^z).
// In any other row what underflows has p < 2^-125.  Ordinary batches hold few such rows,
// so that the sum, and no maximum, is looked at (a maximum for every row: 18.0 instead
// of 16.0 us for 5003 x 160).  SIGMOID is a template parameter for the registers of the
// softmax (4096 x 1000 in bf16: 22.3 instead of 28.6 us).
template <typename LT, int LPT, int NV, bool VEC, bool SIGMOID>
__device__ __forceinline__ void row_probs(const RowRaw<LT, NV>& r, const LT* row, int E,
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
    if (SIGMOID) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float z = p[i][k], e = exp_fast(-fabsf(z));
                float inv;                                // 1 ulp
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(1.0f + e));
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
                p[i][k] = exp_fast(p[i][k] - shift);
                rest[i][k] = 1.0f;
                sum += p[i][k];
            }
    }
    sum = lanes_sum<LPT>(sum);
    if (SIGMOID && __any_sync(0xffffffffu, sum < 0.5f)) {
        const bool far = LPT == 32 || sum < 0.5f;     // of the whole warp, or of this lane's row
        const RowRaw<LT, NV> again = load_row<LT, LPT, NV, VEC>(row, E);
        float z[NV][4], total = 0.0f;
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                z[i][k] = clean_logit(to_f32(again.e[i][k]));
                if (4 * (LPT * i + sub) + k >= E) z[i][k] = -INFINITY;
                m = fmaxf(m, z[i][k]);
            }
        m = lanes_max<LPT>(m);
        // nothing but -inf, NaN and the lowest finite value: closed
        const bool closed = m <= lowest<LT>();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float inv;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(1.0f + exp_fast(z[i][k])));
                const float v = closed ? 0.0f : exp_fast(z[i][k] - m) * inv;
                total += v;
                p[i][k] = far ? v : p[i][k];
            }
        total = lanes_sum<LPT>(total);
        if (far) sum = total;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) p[i][k] *= inv;
}

template <typename LT, int LPT, int NV, bool VEC, bool SIGMOID>
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
        row_probs<LT, LPT, NV, VEC, SIGMOID>(row, row_of(t), a.E, p, rest);
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
        a.part_sums[(long long)blockIdx.x * a.E + e] = s;
        a.part_counts[(long long)blockIdx.x * a.E + e] = counts[e];
    }
    if (threadIdx.x == 0) {
        a.part_live[blockIdx.x] = live;
        if (blockIdx.x == 0) *a.done = 0;
    }
}

// Adds the partial tables' rows in a fixed order and forms the loss.  A CTA takes
// 32 columns; warp w adds rows w, w + 32, ..., eight of them in flight at a time.
constexpr int kJoinThreads = 1024;
constexpr int kJoinAhead = 8;
constexpr int kJoinMaxCtas = kBalMaxE / 32;

struct JoinArgs {
    const float* part_sums;
    const int32_t* part_counts;
    const int32_t* part_live;
    int32_t* done;
    double* part_loss;    // [CTAs of this launch]
    int ctas, E, topk;
    float coef;
    float* loss;
    int32_t* counts;
    float* prob_sums;
    int32_t* n_tokens;
};

__global__ void __launch_bounds__(kJoinThreads) moe_balance_join_kernel(const JoinArgs a) {
    pdl_begin();
    __shared__ float s_sum[32][33];
    __shared__ int s_cnt[32][33];
    __shared__ int s_live[32];
    __shared__ bool last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int e = blockIdx.x * 32 + lane, col = min(e, a.E - 1);
    float s = 0.0f;
    int c = 0;
    for (int i = warp; i < a.ctas; i += 32 * kJoinAhead) {
        float f[kJoinAhead];
        int n[kJoinAhead];
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const long long at = (long long)min(i + 32 * j, a.ctas - 1) * a.E + col;
            f[j] = a.part_sums[at];
            n[j] = a.part_counts[at];
        }
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            s += i + 32 * j < a.ctas ? f[j] : 0.0f;
            c += i + 32 * j < a.ctas ? n[j] : 0;
        }
    }
    s_sum[warp][lane] = s;
    s_cnt[warp][lane] = c;
    int live = tid < a.ctas ? a.part_live[tid] : 0;       // at most 1024 rows
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) s_live[warp] = live;
    __syncthreads();
    if (warp > 0) return;
    s = 0.0f;
    c = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
        s += s_sum[w][lane];
        c += s_cnt[w][lane];
    }
    double part = 0.0;
    if (e < a.E) {
        a.prob_sums[e] = s;
        a.counts[e] = c;
        part = (double)c * (double)s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    if (lane == 0) {
        a.part_loss[blockIdx.x] = part;
        __threadfence();
        last = atomicAdd(a.done, 1) == (int)gridDim.x - 1;
        __threadfence();
    }
    __syncwarp();
    if (!last) return;
    live = __reduce_add_sync(0xffffffffu, s_live[lane]);
    if (lane == 0) {
        double total = 0.0;
        for (int k = 0; k < (int)gridDim.x; ++k) total += __ldcg(a.part_loss + k);
        const double n = live;
        *a.n_tokens = live;
        *a.loss = live ? (float)((double)a.coef * a.E * total / (a.topk * n * n)) : 0.0f;
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
    void* dlogits;
};

template <typename LT, int LPT, int NV, bool VEC, bool SIGMOID>
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
        row_probs<LT, LPT, NV, VEC, SIGMOID>(row, row_of(t), a.E, p, rest);
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
#define FERRET_BALANCE_SHAPE(KERNEL, LT, VEC, SIG, E, ...)                              \
    ((E) <= 32    ? launch_kernel(KERNEL<LT, 8, 1, VEC, SIG>, __VA_ARGS__)              \
     : (E) <= 64  ? launch_kernel(KERNEL<LT, 16, 1, VEC, SIG>, __VA_ARGS__)             \
     : (E) <= 128 ? launch_kernel(KERNEL<LT, 32, 1, VEC, SIG>, __VA_ARGS__)             \
     : (E) <= 256 ? launch_kernel(KERNEL<LT, 32, 2, VEC, SIG>, __VA_ARGS__)             \
     : (E) <= 512 ? launch_kernel(KERNEL<LT, 32, 4, VEC, SIG>, __VA_ARGS__)             \
                  : launch_kernel(KERNEL<LT, 32, 8, VEC, SIG>, __VA_ARGS__))

// Tokens that a CTA works on at once.
int balance_tokens(int E) { return kBalThreads / (E <= 32 ? 8 : E <= 64 ? 16 : 32); }

// Two rounds of tokens per CTA before a further CTA pays (the second launch reads a
// row for every CTA), four CTAs per SM at most.
int balance_ctas(int T, int E, int sms) {
    const int per = 2 * balance_tokens(E);
    return std::max(1, std::min((int)(((long long)T + per - 1) / per), sms * 4));
}

// Vector accesses: rows of whole vectors, each on a vector's boundary.
bool balance_vec(const void* logits, long long ld, int E, int size, const void* out) {
    return E % 4 == 0 && ld % 4 == 0 && aligned_to(logits, 4 * size) && aligned_to(out, 4 * size);
}

template <typename LT, bool SIG>
int run_balance(const BalanceArgs& a, int ctas, cudaStream_t s) {
    const dim3 grid(ctas), block(kBalThreads);
    return balance_vec(a.logits, a.ld, a.E, sizeof(LT), nullptr)
               ? FERRET_BALANCE_SHAPE(moe_balance_kernel, LT, true, SIG, a.E, grid, block, 0, s, a)
               : FERRET_BALANCE_SHAPE(moe_balance_kernel, LT, false, SIG, a.E, grid, block, 0, s, a);
}

template <typename LT>
int run_balance(const BalanceArgs& a, bool sigmoid, int ctas, cudaStream_t s) {
    return sigmoid ? run_balance<LT, true>(a, ctas, s) : run_balance<LT, false>(a, ctas, s);
}

template <typename LT, bool SIG>
int run_balance_bwd(const BalanceBwdArgs& a, int sms, cudaStream_t s) {
    const int per = balance_tokens(a.E);
    const dim3 grid((unsigned)std::min<long long>(((long long)a.T + per - 1) / per, sms * 4LL)),
        block(kBalThreads);
    return balance_vec(a.logits, a.ld, a.E, sizeof(LT), a.dlogits)
               ? FERRET_BALANCE_SHAPE(moe_balance_bwd_kernel, LT, true, SIG, a.E, grid, block, 0, s, a)
               : FERRET_BALANCE_SHAPE(moe_balance_bwd_kernel, LT, false, SIG, a.E, grid, block, 0, s, a);
}

template <typename LT>
int run_balance_bwd(const BalanceBwdArgs& a, bool sigmoid, int sms, cudaStream_t s) {
    return sigmoid ? run_balance_bwd<LT, true>(a, sms, s) : run_balance_bwd<LT, false>(a, sms, s);
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" size_t ferret_moe_balance_loss_workspace_size(int T, int E) {
    if (T <= 0 || E <= 0 || E > kBalMaxE) return 0;
    return kJoinMaxCtas * sizeof(double) + 16 +
           (size_t)balance_ctas(T, E, kBalMaxCtas / 4) * (2 * (size_t)E + 1) * 4;
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
    if (T == 0) {
        if (cudaMemsetAsync(loss, 0, 4, s) != cudaSuccess ||
            cudaMemsetAsync(counts, 0, (size_t)E * 4, s) != cudaSuccess ||
            cudaMemsetAsync(prob_sums, 0, (size_t)E * 4, s) != cudaSuccess ||
            cudaMemsetAsync(n_tokens, 0, 4, s) != cudaSuccess) {
            cudaGetLastError();
            return FERRET_ERR_CUDA;
        }
        return FERRET_OK;
    }
    const int ctas = balance_ctas(T, E, std::min(info->num_sms, kBalMaxCtas / 4));
    // loss shares, the counter, then the tables
    double* shares = static_cast<double*>(workspace);
    int32_t* done = reinterpret_cast<int32_t*>(shares + kJoinMaxCtas);
    float* sums = reinterpret_cast<float*>(done + 4);
    int32_t* cnts = reinterpret_cast<int32_t*>(sums + (size_t)ctas * E);
    int32_t* live = cnts + (size_t)ctas * E;
    const BalanceArgs a{logits, ld, topk_ids, token_mask, T, E, topk, sums, cnts, live, done};
    const bool sigmoid = (flags & FERRET_ROUTE_SIGMOID) != 0;
    rc = dtype == FERRET_BF16   ? run_balance<__nv_bfloat16>(a, sigmoid, ctas, s)
         : dtype == FERRET_FP16 ? run_balance<__half>(a, sigmoid, ctas, s)
                                : run_balance<float>(a, sigmoid, ctas, s);
    if (rc != FERRET_OK) return rc;
    const JoinArgs j{sums, cnts, live, done, shares, ctas, E, topk, coef, loss, counts, prob_sums,
                     n_tokens};
    return launch_kernel(moe_balance_join_kernel, dim3((E + 31) / 32), dim3(kJoinThreads), 0, s, j);
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
                           grad_logits};
    const bool sigmoid = (flags & FERRET_ROUTE_SIGMOID) != 0;
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_balance_bwd<__nv_bfloat16>(a, sigmoid, info->num_sms, s);
        case FERRET_FP16: return run_balance_bwd<__half>(a, sigmoid, info->num_sms, s);
        default: return run_balance_bwd<float>(a, sigmoid, info->num_sms, s);
    }
}
