// moe_route.cu -- from router logits to the ids and weights the expert path
// reads (moe_permute, moe_combine), and the gradient of the logits.
//
// Per token, over E experts with logits z:
//   scores   s = softmax(z) or sigmoid(z)
//   keys     c = s + bias (the bias picks experts, it never enters a weight)
//   groups   with n_group > 1, only the topk_group groups whose group_top best
//            keys have the largest sum stay open
//   choice   the topk open experts with the largest keys, largest first, the
//            lower id first among equals
//   weights  scale * s[id], divided by their sum when renormalized
// A logit of -inf or NaN closes its expert (score 0); slots with no open
// expert left, and every slot of a token outside the mask, get id -1 and
// weight 0, which the permutation and the combine skip.
//
// Which of two keys is larger decides an integer, so the order has to be that
// of the exact keys.  Without a bias the score is monotone in z and z itself
// is compared.  Otherwise keys carry the rounding of exp and of the sum; the
// selection runs on fp32 keys and also looks at the gap between each chosen
// key and the next: a gap below the bound on that rounding sends the token to
// a second selection with keys in fp64 (under one token in a hundred).
//
// HBM-bound at large T (the logits are read once), latency-bound at small T.
// One warp per token with the keys in registers: a round of the choice is a
// compare of a lane's keys plus two warp reductions (redux.sync) on an
// order-preserving integer image of the key.  Groups are whole lane segments
// (n_group is a power of two), so a group's best two keys need
// log2(32 / n_group) shuffles.
#include "row_io.cuh"

namespace ferret {
namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxE = 1024;
constexpr unsigned kFull = 0xffffffffu;

struct RouteArgs {
    const void* logits;
    long long ld;
    const float* bias;
    const uint8_t* mask;
    int T, E, topk, n_group, topk_group, group_top;
    bool sigmoid, renorm;
    float scale;
    float* weights;
    int32_t* ids;
};

// sigmoid(z) without cancellation or overflow on either side.
__device__ __forceinline__ float sigmoid_f(float z) {
    const float e = expf(-fabsf(z));
    return (z >= 0.0f ? 1.0f : e) / (1.0f + e);
}
__device__ __forceinline__ double sigmoid_d(double z) {
    const double e = exp(-fabs(z));
    return (z >= 0.0 ? 1.0 : e) / (1.0 + e);
}

// Order-preserving image of a float: a < b <=> order(a) < order(b), -0 == +0.
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned u = __float_as_uint(v + 0.0f);
    return u ^ ((int)u < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o) {
    return __uint_as_float(o ^ ((int)o < 0 ? 0x80000000u : 0xffffffffu));
}

// The largest v over the warp, and the smallest idx among the lanes that have it.
__device__ __forceinline__ void warp_best(float& v, int& idx) {
    const unsigned o = order_of(v);
    const unsigned m = __reduce_max_sync(kFull, o);
    idx = (int)__reduce_min_sync(kFull, o == m ? (unsigned)idx : 0x7fffffffu);
    v = value_of(m);
}
__device__ __forceinline__ void warp_best(double& v, int& idx) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double w = __shfl_xor_sync(kFull, v, o);
        const int i = __shfl_xor_sync(kFull, idx, o);
        if (w > v || (w == v && i < idx)) v = w, idx = i;
    }
}

// Where a lane's experts are: group lane / lpg, `n` of them from `base` on.
struct Span {
    int base, n;
};

__device__ __forceinline__ Span lane_span(int E, int n_group) {
    const int lane = threadIdx.x & 31, lpg = 32 / n_group, G = E / n_group;
    const int vpl = (G + lpg - 1) / lpg, off = (lane % lpg) * vpl;
    return {lane / lpg * G + off, max(0, min(vpl, G - off))};
}

// Closes the keys of all but the topk_group best groups.  Returns true if the
// border between the last open and the first closed group is closer than tol.
template <typename F, int VPL>
__device__ __forceinline__ bool close_groups(F (&key)[VPL], const RouteArgs& a, F tol) {
    const int lane = threadIdx.x & 31, lpg = 32 / a.n_group;
    F b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        b2 = fmax(b2, fmin(b1, key[k]));
        b1 = fmax(b1, key[k]);
    }
    for (int o = 1; o < lpg; o <<= 1) {
        const F c1 = __shfl_xor_sync(kFull, b1, o), c2 = __shfl_xor_sync(kFull, b2, o);
        b2 = fmax(fmin(b1, c1), fmax(b2, c2));
        b1 = fmax(b1, c1);
    }
    F score = b1;
    if (a.group_top == 2 && b2 > -INFINITY) score += b2;
    bool open = false;
    F last = INFINITY;
    bool near = false;
    for (int i = 0; i <= a.topk_group && i < a.n_group; ++i) {
        F v = open ? (F)-INFINITY : score;
        int g = lane / lpg;
        warp_best(v, g);
        if (!(v > -INFINITY)) break;
        if (i == a.topk_group) {
            near = last - v <= tol;
            break;
        }
        if (g == lane / lpg) open = true;
        last = v;
    }
    if (!open)
#pragma unroll
        for (int k = 0; k < VPL; ++k) key[k] = -INFINITY;
    return near;
}

template <typename LT>
__device__ __forceinline__ bool same_expert(const RouteArgs& a, const LT* row, int i, int j) {
    return clean_logit(to_f32(row[i])) == clean_logit(to_f32(row[j])) &&
           (!a.bias || a.bias[i] == a.bias[j]);
}

// Picks up to topk experts; lane j gets the id of slot j (-1: none left).
// With tol >= 0 the gaps down to the first key not chosen are watched: returns
// true where one is within tol and the two experts are not equal by input.
template <typename F, int VPL, typename LT>
__device__ __forceinline__ bool pick(F (&key)[VPL], const Span sp, const RouteArgs& a,
                                     const LT* row, F tol, int& my_id) {
    const int lane = threadIdx.x & 31;
    F last = INFINITY;
    int last_id = -1;
    my_id = -1;
    const int rounds = a.topk + (tol >= 0 ? 1 : 0);
    for (int j = 0; j < rounds; ++j) {
        F v = -INFINITY;
        int k0 = 0;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if (key[k] > v) v = key[k], k0 = k;
        int id = sp.base + k0;
        warp_best(v, id);
        if (!(v > -INFINITY)) break;
        if (tol >= 0 && j > 0 && last - v <= tol && !same_expert(a, row, last_id, id)) return true;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if (sp.base + k == id && k < sp.n) key[k] = -INFINITY;
        if (j == lane && j < a.topk) my_id = id;
        last = v;
        last_id = id;
    }
    return false;
}

// The selection with keys in fp64, for tokens whose fp32 keys are too close.
template <typename LT, int VPL>
__device__ __noinline__ int pick_exact(const RouteArgs& a, const LT* row) {
    const Span sp = lane_span(a.E, a.n_group);
    double key[VPL];
    double m = -INFINITY, sum = 0.0;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        key[k] = k < sp.n ? (double)clean_logit(to_f32(row[sp.base + k])) : -INFINITY;
        m = fmax(m, key[k]);
    }
    if (!a.sigmoid) {
        int unused = 0;
        warp_best(m, unused);
#pragma unroll
        for (int k = 0; k < VPL; ++k) sum += key[k] > -INFINITY ? exp(key[k] - m) : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    }
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        if (!(key[k] > -INFINITY)) continue;
        key[k] = a.sigmoid ? sigmoid_d(key[k]) : exp(key[k] - m) / sum;
        if (a.bias) {
            key[k] += (double)a.bias[sp.base + k];
            if (!(key[k] > -INFINITY)) key[k] = -INFINITY;
        }
    }
    if (a.n_group > 1) close_groups<double, VPL>(key, a, -1.0);
    int id;
    pick<double, VPL>(key, sp, a, row, -1.0, id);
    return id;
}

template <typename LT, int VPL>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_kernel(const RouteArgs a) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const Span sp = lane_span(a.E, a.n_group);
    const bool bare = !a.bias && (a.n_group == 1 || a.group_top == 1);   // z orders the experts
    for (long long t = (long long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < a.T;
         t += (long long)gridDim.x * kRouteWarps) {
        const LT* row = static_cast<const LT*>(a.logits) + t * a.ld;
        int id = -1;
        float m = -INFINITY, sum = 0.0f;
        if (!a.mask || a.mask[t]) {
            float key[VPL];
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                key[k] = k < sp.n ? clean_logit(to_f32(row[sp.base + k])) : -INFINITY;
                m = fmaxf(m, key[k]);
            }
            m = warp_max(m);
            // Two keys further apart than tol are in their exact order: a
            // sigmoid is within 2^-22 of the exact one (expf 2 ulp, two
            // roundings), a softmax within (VPL + 12) 2^-24 (VPL + 5 additions
            // in the sum, expf, the division), and the sum with the bias adds
            // half an ulp of the key.
            float tol = -1.0f;
            if (m > -INFINITY && !a.sigmoid && (!bare || !a.renorm)) {
#pragma unroll
                for (int k = 0; k < VPL; ++k)
                    sum += key[k] > -INFINITY ? expf(key[k] - m) : 0.0f;
                sum = warp_sum(sum);
            }
            if (!bare) {
                float big = 1.0f;
#pragma unroll
                for (int k = 0; k < VPL; ++k) {
                    if (!(key[k] > -INFINITY)) continue;
                    key[k] = a.sigmoid ? sigmoid_f(key[k]) : expf(key[k] - m) / sum;
                    if (a.bias) {
                        key[k] += a.bias[sp.base + k];
                        if (!(key[k] > -INFINITY)) key[k] = -INFINITY;
                        if (fabsf(key[k]) < INFINITY) big = fmaxf(big, fabsf(key[k]));
                    }
                }
                tol = (a.sigmoid ? 0x1p-20f : (VPL + 12) * 0x1p-23f) + 0x1p-22f * warp_max(big);
            }
            bool near = false;
            if (a.n_group > 1) near = close_groups<float, VPL>(key, a, bare ? -1.0f : 2.0f * tol);
            if (!near) near = pick<float, VPL>(key, sp, a, row, tol, id);
            if (near) id = pick_exact<LT, VPL>(a, row);
        }
        // lane j: slot j
        float w = 0.0f;
        if (a.sigmoid) {
            if (id >= 0) w = sigmoid_f(clean_logit(to_f32(row[id])));
            if (a.renorm) {
                const float total = warp_sum(w);
                w = total > 0.0f ? w / total : 0.0f;
            }
        } else {
            const float z = id >= 0 ? clean_logit(to_f32(row[id])) : -INFINITY;
            const float top = a.renorm ? warp_max(z) : m;     // shifted by the largest chosen one
            if (id >= 0) w = expf(z - top);
            const float total = a.renorm ? warp_sum(w) : sum;
            w = id >= 0 ? w / total : 0.0f;
        }
        if (lane < a.topk) {
            a.weights[t * a.topk + lane] = a.scale * w;
            a.ids[t * a.topk + lane] = id;
        }
    }
}

// ------------------------------------------------------------------ backward
//
// With g_j the gradient of weight j times scale, over the token's valid slots:
//   softmax              dz_e = p_e * (G_e - sum_j g_j p_(id_j)),  G_e: the sum
//                        of the g_j with id_j = e
//   softmax, renormalized, w'_j = s_j / sum s:  dz_(id_j) += w'_j (g_j - sum_i g_i w'_i)
//   sigmoid              dz_(id_j) += g_j s_j (1 - s_j)
//   sigmoid, renormalized      dz_(id_j) += w'_j (1 - s_j) (g_j - sum_i g_i w'_i)
// and zero elsewhere.  Slots that repeat an id add up, in slot order; slots
// outside [0, E) count for nothing.  A warp writes a token's row first and the
// chosen columns over it (its own writes, ordered by __syncwarp).
struct RouteBwdArgs {
    const float* grad;
    const void* logits;
    long long ld;
    const int32_t* ids;
    int T, E, topk;
    bool sigmoid, renorm;
    float scale;
    void* dlogits;
};

template <typename LT>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_bwd_kernel(const RouteBwdArgs a) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const bool dense = !a.sigmoid && !a.renorm;
    for (long long t = (long long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5); t < a.T;
         t += (long long)gridDim.x * kRouteWarps) {
        const LT* row = static_cast<const LT*>(a.logits) + t * a.ld;
        LT* out = static_cast<LT*>(a.dlogits) + t * a.E;
        int id = lane < a.topk ? a.ids[t * a.topk + lane] : -1;
        if (id >= a.E) id = -1;
        const float g = id >= 0 ? a.scale * a.grad[t * a.topk + lane] : 0.0f;
        const float z = id >= 0 ? clean_logit(to_f32(row[id])) : -INFINITY;

        float m = 0.0f, sum = 1.0f;
        if (dense) {
            m = -INFINITY;
            for (int e = lane; e < a.E; e += 32) m = fmaxf(m, clean_logit(to_f32(row[e])));
            m = warp_max(m);
            sum = 0.0f;
            if (m > -INFINITY)
                for (int e = lane; e < a.E; e += 32) sum += expf(clean_logit(to_f32(row[e])) - m);
            sum = warp_sum(sum);
        }
        // d: this slot's contribution to dz at its id
        float d = 0.0f, inner = 0.0f;
        if (dense) {
            const float p = z > -INFINITY ? expf(z - m) / sum : 0.0f;
            inner = warp_sum(g * p);
            d = p * g;                                    // - p * inner, once per id, below
        } else if (!a.renorm) {
            const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
            d = z > -INFINITY ? g * e * r * r : 0.0f;     // s (1 - s)
        } else {
            float w, rest = 1.0f;
            if (a.sigmoid) {
                w = z > -INFINITY ? sigmoid_f(z) : 0.0f;
                rest = sigmoid_f(-z);                     // 1 - s
            } else {
                const float top = warp_max(z);
                w = z > -INFINITY ? expf(z - top) : 0.0f;
            }
            const float total = warp_sum(w);
            w = total > 0.0f ? w / total : 0.0f;
            d = w * (g - warp_sum(g * w)) * rest;
            if (!(z > -INFINITY)) d = 0.0f;
        }
        // slots with the same id: the first of them writes the sum
        float all = 0.0f;
        bool first = id >= 0;
        for (int j = 0; j < a.topk; ++j) {
            const int other = __shfl_sync(kFull, id, j);
            const float dj = __shfl_sync(kFull, d, j);
            if (other == id) {
                all += dj;
                if (j < lane) first = false;
            }
        }
        if (dense) {
            for (int e = lane; e < a.E; e += 32) {
                const float ze = clean_logit(to_f32(row[e]));
                out[e] = from_f32<LT>(ze > -INFINITY ? -(expf(ze - m) / sum) * inner : 0.0f);
            }
            if (z > -INFINITY) all -= expf(z - m) / sum * inner;
        } else {
            for (int e = lane; e < a.E; e += 32) out[e] = from_f32<LT>(0.0f);
        }
        __syncwarp();
        if (first) out[id] = from_f32<LT>(all);
    }
}

template <typename LT>
int run_route(const RouteArgs& a, int sms, cudaStream_t s) {
    const int lpg = 32 / a.n_group, G = a.E / a.n_group, vpl = (G + lpg - 1) / lpg;
    const long long want = ((long long)a.T + kRouteWarps - 1) / kRouteWarps;
    const long long most = (long long)sms * 64;
    const dim3 grid((unsigned)(want < most ? want : most)), block(kRouteWarps * 32);
    if (vpl <= 2) return launch_kernel(moe_route_kernel<LT, 2>, grid, block, 0, s, a);
    if (vpl <= 4) return launch_kernel(moe_route_kernel<LT, 4>, grid, block, 0, s, a);
    if (vpl <= 8) return launch_kernel(moe_route_kernel<LT, 8>, grid, block, 0, s, a);
    if (vpl <= 16) return launch_kernel(moe_route_kernel<LT, 16>, grid, block, 0, s, a);
    return launch_kernel(moe_route_kernel<LT, 32>, grid, block, 0, s, a);
}

template <typename LT>
int run_route_bwd(const RouteBwdArgs& a, int sms, cudaStream_t s) {
    const long long want = ((long long)a.T + kRouteWarps - 1) / kRouteWarps;
    const long long most = (long long)sms * 64;
    const dim3 grid((unsigned)(want < most ? want : most)), block(kRouteWarps * 32);
    return launch_kernel(moe_route_bwd_kernel<LT>, grid, block, 0, s, a);
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" int ferret_moe_route(const void* logits, long long ld, int dtype, const float* bias,
                                const uint8_t* token_mask, int T, int E, int topk, int n_group,
                                int topk_group, int group_top, float scale, int flags,
                                float* weights, int32_t* ids, void* stream) {
    const int size = dtype_size(dtype);
    if (!size || T < 0 || E <= 0 || E > kRouteMaxE || topk <= 0 || topk > 32 || topk > E ||
        ld < E || (long long)T * topk >= (1ll << 31))
        return FERRET_ERR_SHAPE;
    if (n_group <= 0 || n_group > 32 || (n_group & (n_group - 1)) || E % n_group ||
        topk_group <= 0 || topk_group > n_group || (group_top != 1 && group_top != 2) ||
        topk > topk_group * (E / n_group))
        return FERRET_ERR_SHAPE;
    if (T == 0) return FERRET_OK;
    if (!logits || !weights || !ids) return FERRET_ERR_NULL;
    if (!aligned_to(logits, size) || !aligned_to(bias, 4) || !aligned_to(weights, 4) ||
        !aligned_to(ids, 4))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    // every group open: the groups decide nothing
    if (topk_group == n_group) n_group = topk_group = 1;
    const RouteArgs a{logits, ld, bias, token_mask, T, E, topk, n_group, topk_group, group_top,
                      (flags & FERRET_ROUTE_SIGMOID) != 0, (flags & FERRET_ROUTE_RENORM) != 0,
                      scale, weights, ids};
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_route<__nv_bfloat16>(a, info->num_sms, s);
        case FERRET_FP16: return run_route<__half>(a, info->num_sms, s);
        default: return run_route<float>(a, info->num_sms, s);
    }
}

extern "C" int ferret_moe_route_backward(const float* grad_weights, const void* logits,
                                         long long ld, int dtype, const int32_t* ids, int T, int E,
                                         int topk, float scale, int flags, void* grad_logits,
                                         void* stream) {
    const int size = dtype_size(dtype);
    if (!size || T < 0 || E <= 0 || E > kRouteMaxE || topk <= 0 || topk > 32 || ld < E ||
        (long long)T * topk >= (1ll << 31))
        return FERRET_ERR_SHAPE;
    if (T == 0) return FERRET_OK;
    if (!grad_weights || !logits || !ids || !grad_logits) return FERRET_ERR_NULL;
    if (!aligned_to(grad_weights, 4) || !aligned_to(logits, size) || !aligned_to(ids, 4) ||
        !aligned_to(grad_logits, size))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    const RouteBwdArgs a{grad_weights, logits, ld, ids, T, E, topk,
                         (flags & FERRET_ROUTE_SIGMOID) != 0, (flags & FERRET_ROUTE_RENORM) != 0,
                         scale, grad_logits};
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_route_bwd<__nv_bfloat16>(a, info->num_sms, s);
        case FERRET_FP16: return run_route_bwd<__half>(a, info->num_sms, s);
        default: return run_route_bwd<float>(a, info->num_sms, s);
    }
}
