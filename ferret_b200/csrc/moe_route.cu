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
//   weights  scale * s[id], divided by the sum of the chosen s when renormalized
// A logit of -inf or NaN closes its expert (score 0); slots with no open
// expert left, and every slot of a token outside the mask, get id -1 and
// weight 0, which the permutation and the combine skip.
//
// Which of two keys is larger decides an integer, so the order has to be that
// of the exact keys.  The selection runs on approximate keys (fast fp32
// scores, the low bits of a key's integer image traded for the expert's place in
// its lane) and looks at the gap between each chosen key and the next: where a gap is
// below the bound on the approximation, and the two experts are not both chosen
// and equal by their inputs, the experts in reach are ordered by keys in fp64
// (under one token in a hundred of fp32 logits).  Without a bias the score is
// monotone in z, and z itself is the key.
//
// HBM-bound at large T (the logits are read once), latency-bound at small T; in
// between the instructions of the selection bound it.  One warp per token, the
// keys of a lane in registers, sorted once (a merge-sorting network of the
// lane's keys).  A round of the choice is then one warp maximum (redux.sync) of
// the lanes' heads, a ballot that finds the lowest lane that has it, and a shift of
// that lane's list; the gaps are looked at once, after the rounds, by all
// slots together.  Lanes hold consecutive experts and groups are whole lane
// segments (n_group is a power of two), so the lowest lane has the lowest id, and
// a group's best two keys need log2(32 / n_group) shuffles.
//
// B200, 32768 tokens x 256 experts, 8 groups, sigmoid and bias: forward 41 us, with the
// gradient 54 (floor 10.7); 810 warp instructions a token at 74 % of the issue slots.
// 384 experts without groups 53 us, 1024 172 us; tokens whose logits are all equal take
// the full fp64 selection (107 us).  128 tokens: 4.7-5.2 us, the host's share included.
// 80 registers for up to 8 keys a lane, for six CTAs per SM: 72 to 176 bytes a thread are
// spilled with 8 keys.
#include <algorithm>

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
    int lpg_log;          // log2 of the lanes per group
    int slots_log;        // log2 of the lanes per token of the last step (2^slots_log >= topk)
    bool sigmoid, renorm;
    bool bare;            // z orders the experts
    float scale;
    float* weights;
    int32_t* ids;
};

// sigmoid(z) / e^shift, shift <= 0: with the shift of the largest of several z a
// quotient of sigmoids does not underflow.
__device__ __forceinline__ float sigmoid_over(float z, float shift) {
    return expf(fminf(z, 0.0f) - shift) / (1.0f + expf(-fabsf(z)));
}
__device__ __forceinline__ double sigmoid_d(double z) {
    const double e = exp(-fabs(z));
    return (z >= 0.0 ? 1.0 : e) / (1.0 + e);
}

// Fast sigmoid for keys, within 2^-22: ex2 (relative error 2^-22, weighted with
// s (1 - s); the rounding of its argument weighs |z| e^-|z| 2^-23), one addition and
// a reciprocal approximation (1 ulp).
__device__ __forceinline__ float sigmoid_key(float z) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

// Order-preserving image of a float that is not -0: a < b <=> order(a) < order(b).
// No float above -inf maps to 0, which stands for a closed expert.
__device__ __forceinline__ unsigned order_of(float v) {
    const int u = __float_as_int(v);
    return (unsigned)(u ^ ((u >> 31) | (int)0x80000000));
}
__device__ __forceinline__ float value_of(unsigned o) {
    const int u = (int)~o;
    return __int_as_float((int)o ^ ((u >> 31) | (int)0x80000000));
}

// Where a lane's experts are: `n` of its group's (lane >> lpg_log) from `base` on.
struct Span {
    int base, n;
};

__device__ __forceinline__ Span lane_span(const RouteArgs& a) {
    const int lane = threadIdx.x & 31, lpg = 1 << a.lpg_log, G = a.E / a.n_group;
    const int vpl = (G + lpg - 1) >> a.lpg_log, off = (lane & (lpg - 1)) * vpl;
    return {(lane >> a.lpg_log) * G + off, max(0, min(vpl, G - off))};
}

// ---- the selection with keys in fp64, for tokens whose approximate keys are too
// close: plain rounds over the lane's keys

__device__ __forceinline__ void warp_best(double& v, int& idx) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double w = __shfl_xor_sync(kFull, v, o);
        const int i = __shfl_xor_sync(kFull, idx, o);
        if (w > v || (w == v && i < idx)) v = w, idx = i;
    }
}

template <typename LT, int VPL>
__device__ __noinline__ int pick_exact(const RouteArgs& a, const LT* row) {
    const Span sp = lane_span(a);
    const int lane = threadIdx.x & 31, lpg = 1 << a.lpg_log, group = lane >> a.lpg_log;
    double key[VPL];
    double m = -INFINITY, sum = 0.0;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        key[k] = k < sp.n ? (double)clean_logit(to_f32(row[sp.base + k])) : -INFINITY;
        m = fmax(m, key[k]);
    }
    if (!a.bare) {
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
    }
    if (a.n_group > 1) {
        double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            b2 = fmax(b2, fmin(b1, key[k]));
            b1 = fmax(b1, key[k]);
        }
        for (int o = 1; o < lpg; o <<= 1) {
            const double c1 = __shfl_xor_sync(kFull, b1, o), c2 = __shfl_xor_sync(kFull, b2, o);
            b2 = fmax(fmin(b1, c1), fmax(b2, c2));
            b1 = fmax(b1, c1);
        }
        double score = b1;
        if (a.group_top == 2 && b2 > -INFINITY) score += b2;
        bool open = false;
        for (int i = 0; i < a.topk_group; ++i) {
            double v = open ? -INFINITY : score;
            int g = group;
            warp_best(v, g);
            if (v > -INFINITY && g == group) open = true;
        }
        if (!open)
#pragma unroll
            for (int k = 0; k < VPL; ++k) key[k] = -INFINITY;
    }
    int my_id = -1;
    for (int j = 0; j < a.topk; ++j) {
        double v = -INFINITY;
        int id = sp.base;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if (key[k] > v) v = key[k], id = sp.base + k;
        warp_best(v, id);
        if (!(v > -INFINITY)) break;
#pragma unroll
        for (int k = 0; k < VPL; ++k)
            if (sp.base + k == id && k < sp.n) key[k] = -INFINITY;
        if (j == lane) my_id = id;
    }
    return my_id;
}

// Orders n <= 32 candidates (ids) by their exact keys and returns slot lane's: for
// tokens whose groups are settled.  One candidate per lane; its place is the number
// of candidates before it.
template <typename LT>
__device__ __noinline__ int order_exact(const RouteArgs& a, const LT* row, int* ids, int n) {
    const int lane = threadIdx.x & 31;
    const int id = lane < n ? ids[lane] : -1;
    double key = id >= 0 ? (double)clean_logit(to_f32(row[id])) : -INFINITY;
    if (!a.bare) {
        if (a.sigmoid) {
            if (id >= 0) key = sigmoid_d(key);
        } else {
            float m = -INFINITY;
            for (int e = lane; e < a.E; e += 32) m = fmaxf(m, clean_logit(to_f32(row[e])));
            m = warp_max(m);
            double sum = 0.0;
            for (int e = lane; e < a.E; e += 32)
                sum += exp((double)clean_logit(to_f32(row[e])) - (double)m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
            if (id >= 0) key = exp(key - (double)m) / sum;
        }
        if (a.bias && id >= 0) key += (double)a.bias[id];
    }
    int place = 0;
    for (int i = 0; i < n; ++i) {
        const double other = __shfl_sync(kFull, key, i);
        const int other_id = __shfl_sync(kFull, id, i);
        place += other > key || (other == key && other_id < id);
    }
    __syncwarp();
    if (id >= 0) ids[place] = id;
    __syncwarp();
    return lane < min(n, a.topk) ? ids[lane] : -1;
}

// ---- the usual selection

__device__ __forceinline__ void sort_two(unsigned& a, unsigned& b) {
    const unsigned hi = max(a, b);
    b = min(a, b);
    a = hi;
}

// The power of two from VPL up.
template <int VPL>
constexpr int places = VPL <= 2 ? 2 : VPL <= 4 ? 4 : VPL <= 8 ? 8 : VPL <= 16 ? 16 : 32;

// Descending odd-even merge sort (Batcher) of M registers (padded with zeros, whose
// comparisons fold away).
template <int M>
__device__ __forceinline__ void sort_down(unsigned (&list)[M]) {
    constexpr int N = places<M>;
    unsigned v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < M ? list[i] : 0u;
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q > 0; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p))
                        sort_two(v[i + j], v[i + j + q]);
#pragma unroll
    for (int i = 0; i < M; ++i) list[i] = v[i];
}

// A lane's logits as loaded.
template <typename LT, int VPL>
struct LaneRow {
    LT e[VPL];
};

// VEC: the lane holds exactly VPL experts, at a vector's boundary.
template <typename LT, int VPL, bool VEC>
__device__ __forceinline__ LaneRow<LT, VPL> load_lane(const LT* row, const Span sp, int E) {
    LaneRow<LT, VPL> r;
    if (VEC) {
#pragma unroll
        for (int k = 0; k < VPL / 4; ++k) {
            LT v[4];
            load4<LT, true>(row, sp.base + 4 * k, E, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) r.e[4 * k + i] = v[i];
        }
    } else {
#pragma unroll
        for (int k = 0; k < VPL; ++k) r.e[k] = row[min(sp.base + k, E - 1)];
    }
    return r;
}

template <typename LT, int VPL, bool VEC>
__global__ void __launch_bounds__(kRouteWarps * 32, VPL <= 8 ? 6 : VPL <= 16 ? 4 : 2)
    moe_route_kernel(const __grid_constant__ RouteArgs a) {
    pdl_begin();
    constexpr unsigned kPlaces = places<VPL> - 1;     // a key's low bits: kPlaces - place
    __shared__ int picked[kRouteWarps][33];      // the ids in the order of the rounds
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned below = (1u << lane) - 1u;
    const Span sp = lane_span(a);
    const LT* logits = static_cast<const LT*>(a.logits);
    // A warp takes runs of `per` tokens; their weights are computed together, lane
    // (i << slots_log) + j for slot j of token i.
    const int per = 32 >> a.slots_log;
    const long long step = ((long long)gridDim.x * kRouteWarps - 1) * per;   // past a run
    long long t = ((long long)blockIdx.x * kRouteWarps + warp) * per;
    if (t >= a.T) return;
    LaneRow<LT, VPL> next = load_lane<LT, VPL, VEC>(logits + t * a.ld, sp, a.E);
    float bias[VPL];
    float size = 1.0f;                            // no key is larger (unless z is the key)
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        bias[k] = a.bias ? a.bias[min(sp.base + k, a.E - 1)] : 0.0f;
        if (fabsf(bias[k]) < INFINITY) size = fmaxf(size, 1.0f + fabsf(bias[k]));
    }
    size = warp_max(size);
    // Two keys further apart than abs_off + rel * size are in their exact order.
    // Both lose their low bits to the place in the lane downwards, so these move
    // the difference by less than places 2^-23 of the size; the sums with the
    // bias round by half an ulp each; and a score, at most 1, may be off: the
    // fast sigmoid by less than 2^-22, the softmax (VPL + 5 additions in the sum,
    // the exponentials, the quotient) by (VPL + 16) 2^-24.
    const float rel = (places<VPL> + 2) * 0x1p-23f;
    const float abs_off = a.bare ? 0.0f : 2.0f * (a.sigmoid ? 0x1p-22f : (VPL + 16) * 0x1p-24f);
    // A key's integer image with its place in the lane, 0 for a closed expert
    // (bias 0 turns -0 into +0; the largest finite value stands for +inf).
    auto image = [&](float v, int k, bool open) {
        const unsigned o = (order_of(fminf(v, 3.402823466e38f)) & ~kPlaces) | (kPlaces - k);
        return open && v > -INFINITY && (VEC || k < sp.n) ? o : 0u;
    };
    int in_run = 0, run_id = -1;
    float run_m = 0.0f, run_sum = 1.0f;
    while (t < a.T) {
        const LT* row = logits + t * a.ld;
        const LaneRow<LT, VPL> raw = next;
        const long long t_next = t + 1 + (in_run + 1 == per ? step : 0);
        if (t_next < a.T) next = load_lane<LT, VPL, VEC>(logits + t_next * a.ld, sp, a.E);
        int id = -1;
        float m = -INFINITY, sum = 0.0f;
        if (!a.mask || a.mask[t]) {
            unsigned list[VPL];
            if (a.sigmoid && !a.bare) {
#pragma unroll
                for (int k = 0; k < VPL; ++k) {
                    const float z = to_f32(raw.e[k]);
                    list[k] = image(sigmoid_key(z) + bias[k], k, z > -INFINITY);
                }
            } else {
                float z[VPL], e[VPL];
#pragma unroll
                for (int k = 0; k < VPL; ++k) {
                    z[k] = clean_logit(to_f32(raw.e[k]));
                    if (!VEC && k >= sp.n) z[k] = -INFINITY;
                    e[k] = z[k];
                }
                if (!a.sigmoid && (!a.bare || !a.renorm)) {
#pragma unroll
                    for (int k = 0; k < VPL; ++k) m = fmaxf(m, z[k]);
                    m = warp_max(m);
                    const float shift = m > -INFINITY ? m : 0.0f;
#pragma unroll
                    for (int k = 0; k < VPL; ++k) {
                        e[k] = expf(z[k] - shift);
                        sum += e[k];
                    }
                    sum = warp_sum(sum);
                    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                    for (int k = 0; k < VPL; ++k) e[k] = a.bare ? z[k] : e[k] * inv;
                }
#pragma unroll
                for (int k = 0; k < VPL; ++k)
                    list[k] = image(e[k] + bias[k], k, z[k] > -INFINITY);
            }
            sort_down<VPL>(list);
            bool near = false;
            if (a.n_group > 1) {
                const int lpg = 1 << a.lpg_log;
                unsigned b1 = list[0] & ~kPlaces, b2 = VPL > 1 ? list[1] & ~kPlaces : 0u;
                for (int o = 1; o < lpg; o <<= 1) {
                    const unsigned c1 = __shfl_xor_sync(kFull, b1, o),
                                   c2 = __shfl_xor_sync(kFull, b2, o);
                    b2 = max(min(b1, c1), max(b2, c2));
                    b1 = max(b1, c1);
                }
                // half the sum of two keys: biases near the largest finite value may not
                // overflow it
                float sc = value_of(b1);
                if (a.group_top == 2) sc = 0.5f * sc + (b2 ? 0.5f * value_of(b2) : 0.0f);
                // Distinct images: the lower group first among equals.  A group
                // is open if fewer than topk_group come before it.
                const int group = lane >> a.lpg_log;
                const unsigned last = a.n_group - 1, rank = last - group;
                const unsigned score = b1 ? (order_of(sc) & ~last) | rank : rank;
                int before = 0;
#pragma unroll 4
                for (int g = 0; g < 32; g += lpg) before += __shfl_sync(kFull, score, g) > score;
                const bool open = before < a.topk_group;
                if (!open)
#pragma unroll
                    for (int k = 0; k < VPL; ++k) list[k] = 0u;
                // the border between open and closed groups: two sums of two keys,
                // rounded, with log2(n_group) bits of up to twice the size given away
                // (or half of all this)
                const unsigned lo = __reduce_min_sync(kFull, open ? score : 0xffffffffu);
                const unsigned hi = __reduce_max_sync(kFull, open ? 0u : score);
                if (hi > last) {
                    const float vl = value_of(lo), vh = value_of(hi);
                    const float big = a.bare ? fmaxf(fabsf(vl), fabsf(vh)) : size;
                    near = vl - vh <= (a.group_top == 2 ? 0.5f : 1.0f) *
                           (2.0f * abs_off + (2.0f * rel + (2 * a.n_group + 6) * 0x1p-23f) * big);
                }
            }
            unsigned mine = 0u, more = 0u;        // slot lane's key; the first key not chosen
            for (int j = 0; j <= a.topk; ++j) {
                // equal keys: the lowest lane, and in it the lowest place (sorted first)
                const unsigned head = list[0] & ~kPlaces;
                const unsigned best = __reduce_max_sync(kFull, head);
                const unsigned have = __ballot_sync(kFull, head == best);
                if (head == best && !(have & below)) {
                    picked[warp][j] = sp.base + (int)(kPlaces - (list[0] & kPlaces));
                    // up to topk + 1 <= kShort keys of a lane can be called for
                    constexpr int kShort = VPL < 9 ? VPL : 9;
#pragma unroll
                    for (int k = 0; k + 1 < kShort; ++k) list[k] = list[k + 1];
                    if (VPL > kShort && a.topk < kShort) {
                        list[kShort - 1] = 0u;
                    } else {
#pragma unroll
                        for (int k = kShort - 1; k + 1 < VPL; ++k) list[k] = list[k + 1];
                        list[VPL - 1] = 0u;
                    }
                }
                if (j == lane) mine = best;
                more = best;
            }
            __syncwarp();
            // slot lane against the one after it
            const unsigned down = __shfl_down_sync(kFull, mine, 1);
            const unsigned after = lane == a.topk - 1 ? more : down;
            bool close = false;
            if (lane < a.topk && mine) {
                id = picked[warp][lane];
                if (after) {
                    const float v = value_of(mine), w = value_of(after);
                    const float big = a.bare ? fmaxf(fabsf(v), fabsf(w)) : size;
                    if (v - w <= abs_off + rel * big) {
                        // Two chosen experts equal by their inputs are in order.  At the
                        // border a third one, in reach but not looked at, may differ.
                        const int other = picked[warp][lane + 1];
                        close = lane == a.topk - 1 ||
                                clean_logit(to_f32(row[id])) != clean_logit(to_f32(row[other])) ||
                                (a.bias && a.bias[id] != a.bias[other]);
                    }
                }
            }
            if (near) {
                id = pick_exact<LT, VPL>(a, row);
            } else if (__any_sync(kFull, close)) {
                // Every expert that can be among the chosen: those taken (the first one
                // not chosen, too) and what is left within reach of the last slot's key.
                int n = min(__popc(__ballot_sync(kFull, mine != 0u)), a.topk) + (more != 0u);
                const float v = value_of(__shfl_sync(kFull, mine, a.topk - 1));
                const float big = a.bare ? fabsf(v) : size;
                const unsigned reach = more ? order_of(v - (abs_off + 2.0f * rel * big)) : ~0u;
#pragma unroll
                for (int k = 0; k < VPL; ++k) {
                    const unsigned in = __ballot_sync(kFull, list[k] != 0u && list[k] >= reach);
                    if ((in >> lane & 1u) && n + __popc(in & below) < 32)
                        picked[warp][n + __popc(in & below)] =
                            sp.base + (int)(kPlaces - (list[k] & kPlaces));
                    n += __popc(in);
                }
                __syncwarp();
                id = n <= 32 ? order_exact<LT>(a, row, picked[warp], n)
                             : pick_exact<LT, VPL>(a, row);
            }
            __syncwarp();
        }
        // this token's slots to their lanes of the run
        const int from = lane & ((1 << a.slots_log) - 1);
        const int moved = __shfl_sync(kFull, id, from);
        if (lane >> a.slots_log == in_run) {
            run_id = from < a.topk ? moved : -1;
            run_m = m;
            run_sum = sum;
        }
        if (++in_run == per || t + 1 == a.T) {
            const long long token = t + 1 - in_run + (lane >> a.slots_log);
            const bool mine = lane >> a.slots_log < in_run;
            float w = 0.0f;
            const float z = mine && run_id >= 0 ? clean_logit(to_f32(logits[token * a.ld + run_id]))
                                                : -INFINITY;
            float top = a.sigmoid ? 0.0f : run_m;
            if (a.renorm) {                                  // shifted by the largest chosen
                top = z;
                for (int o = 1 << a.slots_log >> 1; o > 0; o >>= 1)
                    top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
            }
            if (z > -INFINITY) w = a.sigmoid ? sigmoid_over(z, fminf(top, 0.0f)) : expf(z - top);
            float total = a.sigmoid ? 1.0f : run_sum;
            if (a.renorm) {
                total = w;
                for (int o = 1 << a.slots_log >> 1; o > 0; o >>= 1)
                    total += __shfl_xor_sync(kFull, total, o);
            }
            w = total > 0.0f ? w / total : 0.0f;
            if (mine && from < a.topk) {
                a.weights[token * a.topk + from] = a.scale * w;
                a.ids[token * a.topk + from] = run_id;
            }
            in_run = 0;
        }
        t = t_next;
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
    int slots;            // lanes per token: the power of two from topk up
    bool sigmoid, renorm;
    float scale;
    void* dlogits;
};

// A warp takes 32 / P tokens at a time, P the power of two from topk up: lane
// P i + j holds slot j of token i.  Rows are written by the whole warp.  NV: vectors
// of 4 columns per lane, columns 4 (32 i + lane) ..+3.
template <typename LT, int NV, bool VEC>
__global__ void __launch_bounds__(kRouteWarps * 32)
    moe_route_bwd_kernel(const __grid_constant__ RouteBwdArgs a) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int P = a.slots, per = 32 / P, slot = lane % P;
    const bool dense = !a.sigmoid && !a.renorm;
    auto slots_sum = [&](float v) {
        for (int o = P >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        return v;
    };
    for (long long t0 = ((long long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5)) * per; t0 < a.T;
         t0 += (long long)gridDim.x * kRouteWarps * per) {
        const long long t = t0 + lane / P;
        const int tokens = (int)min((long long)per, a.T - t0);
        const LT* row = static_cast<const LT*>(a.logits) + t * a.ld;
        LT* out = static_cast<LT*>(a.dlogits) + t * a.E;
        int id = -1;
        float g = 0.0f;
        if (slot < a.topk && t < a.T) {
            id = a.ids[t * a.topk + slot];
            g = a.scale * a.grad[t * a.topk + slot];
        }
        if (id < 0 || id >= a.E) id = -1, g = 0.0f;
        const float z = id >= 0 ? clean_logit(to_f32(row[id])) : -INFINITY;

        // d: this slot's contribution to dz at its id; once: what comes off once per id
        float d = 0.0f, once = 0.0f;
        if (dense) {
            for (int i = 0; i < tokens; ++i) {
                const LT* r = static_cast<const LT*>(a.logits) + (t0 + i) * a.ld;
                LT e[NV][4];
                float p[NV][4];
                float m = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NV; ++n) load4<LT, VEC>(r, 4 * (32 * n + lane), a.E, e[n]);
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        p[n][k] = 4 * (32 * n + lane) + k < a.E ? clean_logit(to_f32(e[n][k]))
                                                                : -INFINITY;
                        m = fmaxf(m, p[n][k]);
                    }
                m = warp_max(m);
                if (!(m > -INFINITY)) m = 0.0f;
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        p[n][k] = expf(p[n][k] - m);
                        sum += p[n][k];
                    }
                sum = warp_sum(sum);
                const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
                const float p_id = expf(z - m) * inv;        // of the lanes of token i
                const float inner = __shfl_sync(kFull, slots_sum(g * p_id), i * P);
                if (lane / P == i) d = p_id * g, once = p_id * inner;
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    float v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = -(p[n][k] * inv) * inner;
                    store4<LT, VEC>(static_cast<LT*>(a.dlogits) + (t0 + i) * a.E,
                                    4 * (32 * n + lane), a.E, v);
                }
            }
        } else {
            const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int i = 0; i < tokens; ++i)
#pragma unroll
                for (int n = 0; n < NV; ++n)
                    store4<LT, VEC>(static_cast<LT*>(a.dlogits) + (t0 + i) * a.E,
                                    4 * (32 * n + lane), a.E, none);
            if (!a.renorm) {
                const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
                d = g * e * r * r;                        // s (1 - s); -inf: e = 0
            } else {
                float top = z, w = 0.0f;
                for (int o = P >> 1; o > 0; o >>= 1)
                    top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
                if (z > -INFINITY)
                    w = a.sigmoid ? sigmoid_over(z, fminf(top, 0.0f)) : expf(z - top);
                const float rest = a.sigmoid ? sigmoid_over(-z, 0.0f) : 1.0f;      // 1 - s
                const float total = slots_sum(w);
                w = total > 0.0f ? w / total : 0.0f;
                d = w * (g - slots_sum(g * w)) * rest;
            }
        }
        // slots of a token with the same id add up in slot order; the first writes the sum
        const unsigned same = __match_any_sync(kFull, id < 0 ? -1 - lane : id + lane / P * a.E);
        float all = d;
        if (__any_sync(kFull, __popc(same) > 1)) {
            all = 0.0f;
            for (int j = 0; j < 32; ++j) {
                const float dj = __shfl_sync(kFull, d, j);
                if (same >> j & 1u) all += dj;
            }
        }
        __syncwarp();
        if (id >= 0 && __ffs(same) - 1 == lane) out[id] = from_f32<LT>(all - once);
        __syncwarp();
    }
}

template <typename LT, int VPL, bool VEC>
int launch_route(const RouteArgs& a, int sms, cudaStream_t s) {
    // as many CTAs as are resident at once
    static const int per_sm = [] {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, moe_route_kernel<LT, VPL, VEC>,
                                                          kRouteWarps * 32, 0) != cudaSuccess)
            cudaGetLastError();
        return n > 0 ? n : 4;
    }();
    const int per = kRouteWarps * (32 >> a.slots_log);
    const long long want = ((long long)a.T + per - 1) / per;
    const dim3 grid((unsigned)std::min(want, (long long)sms * per_sm)), block(kRouteWarps * 32);
    return launch_kernel(moe_route_kernel<LT, VPL, VEC>, grid, block, 0, s, a);
}

template <typename LT, int VPL>
int launch_route(const RouteArgs& a, bool vec, int sms, cudaStream_t s) {
    return vec ? launch_route<LT, VPL, true>(a, sms, s) : launch_route<LT, VPL, false>(a, sms, s);
}

template <typename LT>
int run_route(const RouteArgs& a, int sms, cudaStream_t s) {
    const int lpg = 32 / a.n_group, G = a.E / a.n_group, vpl = (G + lpg - 1) / lpg;
    const bool rows = a.ld % 4 == 0 && aligned_to(a.logits, 4 * sizeof(LT));
    const bool full = G == vpl * lpg;          // every lane holds the same number
    if (vpl <= 2) return launch_route<LT, 2>(a, false, sms, s);
    if (vpl <= 4) return launch_route<LT, 4>(a, rows && full && vpl == 4, sms, s);
    if (vpl <= 8) return launch_route<LT, 8>(a, rows && full && vpl == 8, sms, s);
    if (vpl <= 12) return launch_route<LT, 12>(a, rows && full && vpl == 12, sms, s);
    if (vpl <= 16) return launch_route<LT, 16>(a, rows && full && vpl == 16, sms, s);
    return launch_route<LT, 32>(a, rows && full && vpl == 32, sms, s);
}

template <typename LT, int NV>
int launch_route_bwd(const RouteBwdArgs& a, bool vec, int sms, cudaStream_t s) {
    const int per = kRouteWarps * (32 / a.slots);
    const long long want = ((long long)a.T + per - 1) / per;
    const dim3 grid((unsigned)std::min(want, (long long)sms * 64)), block(kRouteWarps * 32);
    return vec ? launch_kernel(moe_route_bwd_kernel<LT, NV, true>, grid, block, 0, s, a)
               : launch_kernel(moe_route_bwd_kernel<LT, NV, false>, grid, block, 0, s, a);
}

template <typename LT>
int run_route_bwd(const RouteBwdArgs& a, int sms, cudaStream_t s) {
    const bool vec = a.E % 4 == 0 && a.ld % 4 == 0 && aligned_to(a.logits, 4 * sizeof(LT)) &&
                     aligned_to(a.dlogits, 4 * sizeof(LT));
    if (a.E <= 128) return launch_route_bwd<LT, 1>(a, vec, sms, s);
    if (a.E <= 256) return launch_route_bwd<LT, 2>(a, vec, sms, s);
    if (a.E <= 512) return launch_route_bwd<LT, 4>(a, vec, sms, s);
    return launch_route_bwd<LT, 8>(a, vec, sms, s);
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
    int lpg_log = 5, slots_log = 0;
    while (32 >> lpg_log < n_group) --lpg_log;
    while (1 << slots_log < topk) ++slots_log;
    // shorter runs while there are too few of them for every SM's 24 warps
    while (slots_log < 5 && T >> (5 - slots_log) < info->num_sms * 24) ++slots_log;
    const RouteArgs a{logits, ld, bias, token_mask, T, E, topk, n_group, topk_group, group_top,
                      lpg_log, slots_log,
                      (flags & FERRET_ROUTE_SIGMOID) != 0, (flags & FERRET_ROUTE_RENORM) != 0,
                      !bias && (n_group == 1 || group_top == 1), scale, weights, ids};
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
    int slots = 1;
    while (slots < topk) slots *= 2;
    const RouteBwdArgs a{grad_weights, logits, ld, ids, T, E, topk, slots,
                         (flags & FERRET_ROUTE_SIGMOID) != 0, (flags & FERRET_ROUTE_RENORM) != 0,
                         scale, grad_logits};
    const cudaStream_t s = as_stream(stream);
    switch (dtype) {
        case FERRET_BF16: return run_route_bwd<__nv_bfloat16>(a, info->num_sms, s);
        case FERRET_FP16: return run_route_bwd<__half>(a, info->num_sms, s);
        default: return run_route_bwd<float>(a, info->num_sms, s);
    }
}
