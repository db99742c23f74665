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
// Feeding.  A CTA covers 128 columns with 4 column warps times 4 K warps and
// walks its K range in chunks of 512 (4 blocks of 32 for each K warp).  While a
// chunk is computed, the next one's weights, scales and zero points are in
// flight into registers, and its activations on their way to the other half of a
// shared buffer, already in the order of the nibble pairs; the four column warps
// read them from there.  One barrier per chunk.
//
// Split.  Where the columns alone give too few CTAs, K is split over the CTAs of
// a cluster.  Partial sums of the K warps meet in shared memory, those of the
// cluster through distributed shared memory, added in a fixed order: results
// repeat bit for bit and no workspace is needed.
#include <algorithm>
#include <cooperative_groups.h>

#include "int4_common.cuh"
#include "row_io.cuh"

namespace ferret {
namespace {

namespace cg = cooperative_groups;

constexpr int kLinColWarps = 4;
constexpr int kLinKWarps = 4;
constexpr int kLinThreads = kLinColWarps * kLinKWarps * 32;
constexpr int kLinCols = 32 * kLinColWarps;   // columns of a CTA
constexpr int kLinDepth = 4;                  // 32-wide K blocks of a warp per chunk
constexpr int kLinChunk = kLinKWarps * kLinDepth;   // blocks of a chunk
constexpr int kLinMaxCluster = 8;
// A token's row of a chunk in shared memory: 64 bytes past a multiple of 128, so
// that the 16-byte reads of two tokens x four K pieces hit all banks once.
constexpr int kLinRowBytes = kLinChunk * 64 + 64;

struct LinearArgs {
    const void* x;
    long long ldx;
    const int32_t* w;
    const void* scale;
    const int32_t* zero;   // nullable: packed [K/g, N/8]
    const void* bias;      // nullable
    void* y;
    int T, K, N;
    uint32_t group_inv;    // block b is in group b for 0, else in group umulhi(b, group_inv)
};

template <typename T>
struct Half2Ops;
template <>
struct Half2Ops<__nv_bfloat16> {
    static constexpr uint32_t kMagic = 0x43004300u;       // 128, 128
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
template <typename T, int NT, bool ZERO>
__global__ void __launch_bounds__(kLinThreads) int4_linear_kernel(const LinearArgs a) {
    pdl_begin();
    using Ops = Half2Ops<T>;
    extern __shared__ __align__(16) uint8_t smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int splits = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cw = warp % kLinColWarps, kw = warp / kLinColWarps;
    const int r = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.y * kLinCols;
    const int n = n0 + 32 * cw + 4 * r;
    const int nc = min(n, a.N - 4);                 // columns past N read valid memory, unused
    const int t0 = blockIdx.z * (NT * 8);
    const int tokens = min(a.T - t0, NT * 8);

    // this CTA's 32-wide K blocks
    const int blocks = a.K >> 5;
    const int b0 = (int)((long long)blocks * rank / splits);
    const int b1 = (int)((long long)blocks * (rank + 1) / splits);

    uint4 w[kLinDepth];
    uint2 sc[kLinDepth];
    uint32_t zp[kLinDepth];
    auto load_weights = [&](int first) {
#pragma unroll
        for (int d = 0; d < kLinDepth; ++d) {
            const int b = min(first + kw * kLinDepth + d, b1 - 1);
            const int g = a.group_inv ? (int)__umulhi((uint32_t)b, a.group_inv) : b;
            w[d] = ld16_stream(a.w + (long long)(4 * b + c) * a.N + nc);
            sc[d] = __ldg(reinterpret_cast<const uint2*>(static_cast<const T*>(a.scale) +
                                                         (long long)g * a.N + nc));
            if (ZERO)
                zp[d] = (uint32_t)__ldg(a.zero + (long long)g * (a.N >> 3) + (nc >> 3)) >>
                        (4 * (nc & 7));
        }
    };
    // Activations of a chunk: 64 pieces of 8 elements per token, NT per thread.
    uint4 xr[NT];
    auto load_x = [&](int first) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int p = threadIdx.x + i * kLinThreads, t = p / (kLinChunk * 4),
                      k = p % (kLinChunk * 4);
            xr[i] = make_uint4(0u, 0u, 0u, 0u);
            if (t < tokens && first + (k >> 2) < b1)
                xr[i] = __ldg(reinterpret_cast<const uint4*>(
                    static_cast<const T*>(a.x) + (long long)(t0 + t) * a.ldx + first * 32 + k * 8));
        }
    };
    auto store_x = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int p = threadIdx.x + i * kLinThreads, t = p / (kLinChunk * 4),
                      k = p % (kLinChunk * 4);
            // natural pairs (0,1) (2,3) (4,5) (6,7) -> (0,4) (1,5) (2,6) (3,7)
            const uint4 v = xr[i];
            const uint4 q = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                                       __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
            *reinterpret_cast<uint4*>(smem + (buf * NT * 8 + t) * kLinRowBytes + k * 16) = q;
        }
    };

    float sum[NT][2][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[i][h][q] = 0.0f;

    load_weights(b0);
    load_x(b0);
    store_x(0);
    __syncthreads();
    int buf = 0;
    for (int first = b0; first < b1; first += kLinChunk, buf ^= 1) {
        uint4 wc[kLinDepth];
        uint2 scc[kLinDepth];
        uint32_t zpc[kLinDepth];
#pragma unroll
        for (int d = 0; d < kLinDepth; ++d) {
            wc[d] = w[d];
            scc[d] = sc[d];
            if (ZERO) zpc[d] = zp[d];
        }
        const bool more = first + kLinChunk < b1;
        if (more) {
            load_weights(first + kLinChunk);
            load_x(first + kLinChunk);
        }
        const uint8_t* xs = smem + (buf * NT * 8 + r) * kLinRowBytes + c * 16;
#pragma unroll
        for (int d = 0; d < kLinDepth; ++d) {
            const int kb = kw * kLinDepth + d;
            if (first + kb >= b1) break;
            T e[4];
            memcpy(e, &scc[d], 8);
            float s[4];
            uint32_t off[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                s[q] = to_f32(e[q]);
                off[q] = Ops::kMagic + (ZERO ? (zpc[d] >> (4 * q)) & 15u : 8u) * 0x00010001u;
            }
            const uint32_t word[4] = {wc[d].x, wc[d].y, wc[d].z, wc[d].w};
            uint32_t q4[4][4];      // [column][nibble pair j, j + 4]
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q4[q][j] = Ops::sub(lop3_and_or(word[q] >> (4 * j), 0x000F000Fu, Ops::kMagic),
                                        off[q]);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint4 x = *reinterpret_cast<const uint4*>(xs + i * 8 * kLinRowBytes + kb * 64);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t lo[4] = {q4[2 * h][0], q4[2 * h + 1][0], q4[2 * h][1],
                                            q4[2 * h + 1][1]};
                    const uint32_t hi[4] = {q4[2 * h][2], q4[2 * h + 1][2], q4[2 * h][3],
                                            q4[2 * h + 1][3]};
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    Ops::mma(acc, lo, x.x, x.y);
                    Ops::mma(acc, hi, x.z, x.w);
                    // MMA row r or r + 8 (q >> 1) is column 2h + (q >> 1) of the lane's four
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        sum[i][h][q] = fmaf(s[2 * h + (q >> 1)], acc[q], sum[i][h][q]);
                }
            }
        }
        if (more) store_x(buf ^ 1);
        __syncthreads();
    }

    // Partial sums [K warp][token][column] over the activations' memory.
    float* part = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                part[(kw * NT * 8 + 8 * i + 2 * c + (q & 1)) * kLinCols + 32 * cw + 4 * r + 2 * h +
                     (q >> 1)] = sum[i][h][q];
    __syncthreads();
    const int live = tokens * kLinCols;
    if (splits > 1) {
        for (int i = threadIdx.x; i < live; i += kLinThreads) {
            float v = part[i];
#pragma unroll
            for (int k = 1; k < kLinKWarps; ++k) v += part[k * NT * 8 * kLinCols + i];
            part[i] = v;
        }
        cluster.sync();
    }
    // Output elements of this CTA: every splits-th run of a warp's 32 columns.
    for (int i = (warp * splits + rank) * 32 + lane; i < live; i += kLinThreads * splits) {
        const int t = i / kLinCols, col = n0 + i % kLinCols;
        if (col >= a.N) continue;
        float v = 0.0f;
        if (splits > 1) {
            for (int k = 0; k < splits; ++k) v += cluster.map_shared_rank(part, k)[i];
        } else {
#pragma unroll
            for (int k = 0; k < kLinKWarps; ++k) v += part[k * NT * 8 * kLinCols + i];
        }
        if (a.bias) v += to_f32(static_cast<const T*>(a.bias)[col]);
        static_cast<T*>(a.y)[(long long)(t0 + t) * a.N + col] = from_f32<T>(v);
    }
    if (splits > 1) cluster.sync();      // peers may still read this CTA's sums
}

template <typename T, int NT, bool ZERO>
int launch_linear(const LinearArgs& a, int splits, cudaStream_t s) {
    const dim3 grid(splits, (a.N + kLinCols - 1) / kLinCols, (a.T + NT * 8 - 1) / (NT * 8));
    constexpr size_t smem = std::max(2 * NT * 8 * kLinRowBytes,
                                     kLinKWarps * NT * 8 * kLinCols * (int)sizeof(float));
    auto kern = int4_linear_kernel<T, NT, ZERO>;
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
            cudaSuccess) {
        cudaGetLastError();
        return FERRET_ERR_CUDA;
    }
    return launch_kernel_cluster(kern, grid, dim3(kLinThreads), smem, splits, s, a);
}

template <typename T, int NT>
int launch_linear(const LinearArgs& a, int splits, cudaStream_t s) {
    return a.zero ? launch_linear<T, NT, true>(a, splits, s)
                  : launch_linear<T, NT, false>(a, splits, s);
}

template <typename T>
int run_linear(const LinearArgs& a, int sms, cudaStream_t s) {
    // The fewest splits that give every SM about four CTAs in turn, as long as
    // a CTA keeps a whole chunk of K.
    const long long tiles = ((long long)a.N + kLinCols - 1) / kLinCols;
    int splits = 1;
    while (splits < kLinMaxCluster && tiles * splits < (long long)sms * 4 &&
           a.K / 32 >= splits * 2 * kLinChunk)
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
    // exact group numbers; 65535 column tiles and token passes in a grid
    if (K > (1 << 20) || N > 65535 * kLinCols || T > 65535 * 32) return FERRET_ERR_SHAPE;
    if (T == 0) return FERRET_OK;
    if (!x || !w || !w_scale || !y) return FERRET_ERR_NULL;
    if (!aligned16(x) || !aligned16(w) || !aligned_to(w_scale, 8) || !aligned_to(w_zero, 4) ||
        !aligned_to(bias, 2) || !aligned_to(y, 2))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    // ceil(2^32 / blocks of a group): exact quotients as long as the product of
    // block number and group length stays below 2^32 (K <= 2^20)
    const uint32_t blocks = group / 32;
    const uint32_t inv = blocks == 1 ? 0u : (uint32_t)(((1ull << 32) + blocks - 1) / blocks);
    const LinearArgs a{x, ldx, w, w_scale, w_zero, bias, y, T, K, N, inv};
    const cudaStream_t s = as_stream(stream);
    return dtype == FERRET_BF16 ? run_linear<__nv_bfloat16>(a, info->num_sms, s)
                                : run_linear<__half>(a, info->num_sms, s);
}
