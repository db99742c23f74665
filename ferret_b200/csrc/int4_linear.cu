// int4_linear.cu -- y = x W (+ bias) for a few tokens and one dense 4-bit weight
// matrix in the compressed-tensors layout (the layout ferret_int4_repack_w13
// takes, baselines/kimi-moe-w13-int4/baseline_marlin.py:62-89, for one matrix):
// w int32 [K/8, N], eight offset-binary nibbles along K per word, low nibble
// first; scale [K/g, N]; W[k, n] = scale[k/g, n] * (nibble - zero[k/g, n]) with
// zero = 8 where no zero points are given.
//
// HBM-bound on the weights (K N / 2 bytes) for up to ~32 tokens, so the weights
// go from global memory to registers once, 16 bytes per lane, and nowhere
// else; no repack is needed, the raw layout already streams.
//
// Arithmetic.  nibble - zero is an integer of at most five bits, exact in bf16
// and fp16: one lop3 plants a nibble pair under an exponent (128 + n or
// 1024 + n) and one packed subtraction takes 128 + zero (1024 + zero) off.
// The warp-level mma.sync.m16n8k16 multiplies these integers with the
// activations (products exact, sums in fp32), 16 columns of W by 8 tokens by
// 16 of K.  The group's scale multiplies the group's fp32 sum, so scales are
// never rounded into weights.
//
// Fragments.  A warp covers 32 columns and walks its K range in blocks of 32.
// Lane (r = lane / 4, c = lane % 4) loads word row c of the block for columns
// 4r .. 4r+3: 8 lanes read 128 contiguous bytes.  The MMA's reduction order is
// free as long as both operands share it, so nibbles j and j + 4 of a word (the
// pair one lop3 extracts) meet activations j and j + 4.  Columns 4r and 4r+1
// are rows r and r + 8 of one MMA, 4r+2 and 4r+3 of another; the accumulators
// of lane (r, c) then belong to the same four columns, tokens 2c and 2c+1, and
// a lane needs the scales of its own four columns only (8 bytes per group).
//
// Split.  K is split over the warps of a CTA and, where the columns alone cannot
// fill the SMs, over the CTAs of a cluster; partial sums meet in shared memory
// (the cluster's through distributed shared memory) and are added in a fixed
// order, so results repeat bit for bit and no workspace is needed.
#include <algorithm>
#include <cooperative_groups.h>

#include "int4_common.cuh"
#include "row_io.cuh"

namespace ferret {
namespace {

namespace cg = cooperative_groups;

constexpr int kLinWarps = 8;
constexpr int kLinThreads = kLinWarps * 32;
constexpr int kLinCols = 32;          // columns of a CTA
constexpr int kLinMaxCluster = 8;
constexpr int kLinDepth = 4;          // 32-wide K blocks a warp loads ahead

struct LinearArgs {
    const void* x;
    long long ldx;
    const int32_t* w;
    const void* scale;
    const int32_t* zero;   // nullable: packed [K/g, N/8]
    const void* bias;      // nullable
    void* y;
    int T, K, N, group_blocks;   // 32-wide blocks of a group
};

template <typename T>
struct Half2Ops;
template <>
struct Half2Ops<__nv_bfloat16> {
    static constexpr uint32_t kMagic = 0x43004300u;       // 128, 128
    static constexpr uint32_t kOne = 0x00010001u;         // one integer step at 128
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        return bf16x2_sub(a, b);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Half2Ops<__half> {
    static constexpr uint32_t kMagic = 0x64006400u;       // 1024, 1024
    static constexpr uint32_t kOne = 0x00010001u;
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// NT: groups of 8 tokens that one pass over the weights serves.
template <typename T, int NT>
__global__ void __launch_bounds__(kLinThreads) int4_linear_kernel(const LinearArgs a) {
    pdl_begin();
    using Ops = Half2Ops<T>;
    __shared__ float part[kLinWarps][NT * 8][kLinCols];
    cg::cluster_group cluster = cg::this_cluster();
    const int splits = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.y * kLinCols, n = n0 + 4 * r;
    const int t0 = blockIdx.z * (NT * 8);
    const bool col_live = n < a.N;

    // this warp's 32-wide K blocks
    const int blocks = a.K >> 5, slots = splits * kLinWarps, slot = rank * kLinWarps + warp;
    const int b0 = (int)((long long)blocks * slot / slots);
    const int b1 = (int)((long long)blocks * (slot + 1) / slots);

    float acc[NT][2][4], sum[NT][2][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][h][q] = sum[i][h][q] = 0.0f;

    const int32_t* wp = a.w + n + (long long)c * a.N;
    const T* xp[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int t = t0 + 8 * i + r;
        xp[i] = t < a.T ? static_cast<const T*>(a.x) + (long long)t * a.ldx + 8 * c : nullptr;
    }

    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t off[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) off[q] = Ops::kMagic + 8u * Ops::kOne;
    int group = -1;
    for (int b = b0; b < b1; b += kLinDepth) {
        uint4 wv[kLinDepth];
#pragma unroll
        for (int d = 0; d < kLinDepth; ++d)
            wv[d] = b + d < b1 && col_live
                        ? ld16_stream(wp + (long long)(b + d) * 4 * a.N)
                        : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int d = 0; d < kLinDepth; ++d) {
            if (b + d >= b1) break;
            const int g = (b + d) / a.group_blocks;
            if (g != group) {
                // the finished group's sums, scaled, and the new group's scales
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            sum[i][h][q] = fmaf(s[2 * h + (q >> 1)], acc[i][h][q], sum[i][h][q]);
                            acc[i][h][q] = 0.0f;
                        }
                group = g;
                if (col_live) {
                    uint2 raw = __ldg(reinterpret_cast<const uint2*>(
                        static_cast<const T*>(a.scale) + (long long)g * a.N + n));
                    T e[4];
                    memcpy(e, &raw, 8);
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[q] = to_f32(e[q]);
                    if (a.zero) {
                        const uint32_t z =
                            (uint32_t)__ldg(a.zero + (long long)g * (a.N >> 3) + (n >> 3)) >>
                            (4 * (n & 7));
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            off[q] = Ops::kMagic + ((z >> (4 * q)) & 15u) * Ops::kOne;
                    }
                }
            }
            const uint32_t word[4] = {wv[d].x, wv[d].y, wv[d].z, wv[d].w};
            uint32_t q4[4][4];      // [column][nibble pair j, j + 4]
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q4[q][j] = Ops::sub(lop3_and_or(word[q] >> (4 * j), 0x000F000Fu, Ops::kMagic),
                                        off[q]);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                uint4 xv = make_uint4(0u, 0u, 0u, 0u);
                if (xp[i]) xv = __ldg(reinterpret_cast<const uint4*>(xp[i] + (b + d) * 32));
                // natural pairs (0,1) (2,3) (4,5) (6,7) -> (0,4) (1,5) (2,6) (3,7)
                const uint32_t p0 = __byte_perm(xv.x, xv.z, 0x5410),
                               p1 = __byte_perm(xv.x, xv.z, 0x7632),
                               p2 = __byte_perm(xv.y, xv.w, 0x5410),
                               p3 = __byte_perm(xv.y, xv.w, 0x7632);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t lo[4] = {q4[2 * h][0], q4[2 * h + 1][0], q4[2 * h][1],
                                            q4[2 * h + 1][1]};
                    const uint32_t hi[4] = {q4[2 * h][2], q4[2 * h + 1][2], q4[2 * h][3],
                                            q4[2 * h + 1][3]};
                    Ops::mma(acc[i][h], lo, p0, p1);
                    Ops::mma(acc[i][h], hi, p2, p3);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                // MMA row r or r + 8 (q >> 1) is column 4r + 2h + (q >> 1), token 2c + (q & 1)
                part[warp][8 * i + 2 * c + (q & 1)][4 * r + 2 * h + (q >> 1)] =
                    fmaf(s[2 * h + (q >> 1)], acc[i][h][q], sum[i][h][q]);
    __syncthreads();

    // The CTA's sum over its warps, in place of warp 0's partials.
    constexpr int kOut = NT * 8 * kLinCols;
    float* flat = &part[0][0][0];
    for (int i = threadIdx.x; i < kOut; i += kLinThreads) {
        float v = flat[i];
#pragma unroll
        for (int w = 1; w < kLinWarps; ++w) v += flat[w * kOut + i];
        flat[i] = v;
    }
    if (splits > 1)
        cluster.sync();
    else
        __syncthreads();
    // The cluster's sums, added in rank order: warp w of CTA `rank` finishes
    // token rows rank + splits * (w, w + 8, ...), a lane one column.
    for (int t = warp * splits + rank; t < NT * 8; t += splits * kLinWarps) {
        if (t0 + t >= a.T || n0 + lane >= a.N) continue;
        float v = 0.0f;
        for (int k = 0; k < splits; ++k)
            v += cluster.map_shared_rank(flat, k)[t * kLinCols + lane];
        if (a.bias) v += to_f32(static_cast<const T*>(a.bias)[n0 + lane]);
        static_cast<T*>(a.y)[(long long)(t0 + t) * a.N + n0 + lane] = from_f32<T>(v);
    }
    if (splits > 1) cluster.sync();      // peers may still read this CTA's sums
}

template <typename T, int NT>
int launch_linear(const LinearArgs& a, int splits, cudaStream_t s) {
    const dim3 grid(splits, (a.N + kLinCols - 1) / kLinCols, (a.T + NT * 8 - 1) / (NT * 8));
    return launch_kernel_cluster(int4_linear_kernel<T, NT>, grid, dim3(kLinThreads), 0, splits, s,
                                 a);
}

template <typename T>
int run_linear(const LinearArgs& a, int sms, cudaStream_t s) {
    // Enough CTAs for about four on every SM, as long as each warp keeps at
    // least two blocks of K.
    const long long tiles = ((long long)a.N + kLinCols - 1) / kLinCols;
    int splits = 1;
    while (splits < kLinMaxCluster && tiles * splits * 2 <= (long long)sms * 4 &&
           a.K / 32 >= splits * 2 * kLinWarps * 2)
        splits *= 2;
    if (a.T <= 8) return launch_linear<T, 1>(a, splits, s);
    if (a.T <= 16) return launch_linear<T, 2>(a, splits, s);
    return launch_linear<T, 4>(a, splits, s);
}

}  // namespace
}  // namespace ferret

using namespace ferret;

extern "C" int ferret_int4_linear(const void* x, long long ldx, const int32_t* w,
                                  const void* w_scale, const int32_t* w_zero, const void* bias,
                                  int dtype, int T, int K, int N, int group, void* y,
                                  void* stream) {
    if ((dtype != FERRET_BF16 && dtype != FERRET_FP16) || T < 0 || K <= 0 || N <= 0 ||
        group <= 0 || group % 32 || K % group || N % 8 || ldx < K || ldx % 8)
        return FERRET_ERR_SHAPE;
    // grid limits: 65535 column tiles and token passes
    if (N > 65535 * kLinCols || T > 65535 * 32) return FERRET_ERR_SHAPE;
    if (T == 0) return FERRET_OK;
    if (!x || !w || !w_scale || !y) return FERRET_ERR_NULL;
    if (!aligned16(x) || !aligned16(w) || !aligned_to(w_scale, 8) || !aligned_to(w_zero, 4) ||
        !aligned_to(bias, 2) || !aligned_to(y, 2))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    const LinearArgs a{x, ldx, w, w_scale, w_zero, bias, y, T, K, N, group / 32};
    const cudaStream_t s = as_stream(stream);
    return dtype == FERRET_BF16 ? run_linear<__nv_bfloat16>(a, info->num_sms, s)
                                : run_linear<__half>(a, info->num_sms, s);
}
