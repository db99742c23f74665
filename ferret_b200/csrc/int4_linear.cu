// int4_linear.cu -- y = x W (+ bias) for a few tokens and one dense 4-bit weight
// matrix in the compressed-tensors layout (the layout ferret_int4_repack_w13
// takes, baselines/kimi-moe-w13-int4/baseline_marlin.py:62-89, for one matrix):
// w int32 [K/8, N], eight offset-binary nibbles along K per word, low nibble
// first; scale [K/g, N]; W[k, n] = scale[k/g, n] * (nibble - zero[k/g, n]) with
// zero = 8 where no zero points are given.
//
// HBM-bound on the weights (K N / 2 bytes) for up to ~32 tokens, so the weights
// are copied on chip once, as they are, and dequantized in registers; no repack is
// needed, the raw layout already streams.
//
// Arithmetic.  nibble - zero is an integer of at most five bits, exact in bf16
// and fp16: one lop3 plants a nibble pair under an exponent (128 + n or
// 1024 + n) and one packed subtraction takes 128 + zero (1024 + zero) off.
// The warp-level mma.sync.m16n8k16 multiplies these integers with the
// activations (products exact, sums in fp32), 16 columns of W by 8 tokens by
// 16 of K.  The group's scale multiplies the group's fp32 sum, so scales are
// never rounded into weights.
//
// Fragments.  A warp covers 32 columns and takes K in blocks of 32.  Lane
// (r = lane / 4, c = lane % 4) reads word row c of the block for four adjacent
// columns (16 bytes).  The MMA's reduction order is free as long as both
// operands share it, so nibbles j and j + 4 of a word (the pair one lop3
// extracts) meet activations j and j + 4.  The lane's columns 0 and 1 are rows
// r and r + 8 of one MMA, 2 and 3 of another; the accumulators of lane (r, c)
// then belong to the same four columns, and a lane needs the scales of its own
// four columns only.
//
// Feeding.  A CTA covers 128 columns: a copy warp and two groups of four math
// warps.  The copy warp fills a shared-memory ring of 128-wide K stages with
// tensor-map boxes (word rows and token rows of 128 bytes, 128-byte swizzle;
// the groups' scale rows); the math groups take the stages in turn.  Bytes in
// flight thus cost no registers, and few copies carry them: one bulk copy per
// 512-byte word row left the copy unit at half the HBM rate.  Two CTAs per SM: with
// three, 72 registers a thread made the compiler compute fragments and scales again
// (158 warp instructions per 32 x 32 block for 16 tokens against 130).  Two leave 96 (18
// warps put five on one sub-partition), in which the kernels for 9 to 16 tokens spill 4
// to 28 bytes a thread, those for more tokens 24 to 72.  The eight lanes of
// a 16-byte shared-memory read phase hold r = 2q, 2q + 1 and all c; with r
// standing for 16-byte piece (token) q or q + 4, the swizzle spreads them over
// all banks.
//
// Split.  Where the columns alone give too few CTAs, K is split over the CTAs of
// a cluster.  Partial sums of the math groups meet in shared memory, those of the
// cluster through distributed shared memory, added in a fixed order: results
// repeat bit for bit and no workspace is needed.
//
// B200: 1 token x 7168 x 4096 8.8 us, 16 x 7168 x 32768 52 us (floors 2.5 and 20.4; the
// copies alone 5.5 and 22.6).  The large case issues on 59 % of the slots with 3.7
// warps per scheduler: the dequantization, not the stream, bounds it.
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

#include "int4_common.cuh"
#include "row_io.cuh"

namespace ferret {
namespace {

namespace cg = cooperative_groups;

constexpr int kLinColWarps = 4;
constexpr int kLinKGroups = 2;                          // math groups
constexpr int kLinMath = kLinColWarps * kLinKGroups;    // math warps
constexpr int kLinThreads = (kLinMath + 1) * 32;        // and the copy warp
constexpr int kLinCols = 32 * kLinColWarps;             // columns of a CTA
constexpr int kLinDepth = 4;                            // 32-wide K blocks of a stage
constexpr int kLinMaxCluster = 8;
// Stages of the ring.  A multiple of the math groups, so that a slot always
// belongs to the same group: a group that met a slot only every other lap could
// take the completion of the lap before last for its own (the wait sees a lap's
// parity, not its number).
constexpr int kLinStages = 6;
static_assert(kLinStages % kLinKGroups == 0);
// Stage layout: a box of word rows per column warp, token rows in boxes of 64
// activations, scale rows; boxes on 1024 bytes (the swizzle's period).
constexpr int kLinWordBox = 4 * kLinDepth * 128;
constexpr int kLinTokenAt = kLinColWarps * kLinWordBox;
constexpr int kLinScaleRow = kLinCols * 2;
constexpr int kLinScaleRows = kLinDepth + 1;            // groups that a stage can touch

template <int NT>
constexpr int kLinTokenBox = NT * 8 * 128;
template <int NT>
constexpr int kLinScaleAt = kLinTokenAt + kLinDepth / 2 * kLinTokenBox<NT>;
template <int NT>
constexpr int kLinStageBytes = (kLinScaleAt<NT> + kLinScaleRows * kLinScaleRow + 1023) / 1024 * 1024;

struct LinearArgs {
    const int32_t* zero;   // nullable: packed [K/g, N/8]
    const void* bias;      // nullable
    void* y;
    int T, K, N;
    uint32_t group_inv;    // block b is in group b for 0, else in group umulhi(b, group_inv)
    int scale_rows;        // rows of a scale box
    bool even_groups;      // scale_rows groups of equal length in every stage
};

template <typename T>
struct Half2Ops;
template <>
struct Half2Ops<__nv_bfloat16> {
    static constexpr uint32_t kMagic = 0x43004300u;       // 128, 128
    static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
        return bf16x2_sub(a, b);
    }
    static __device__ __forceinline__ void unpack(uint2 v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xFFFF0000u);
        f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xFFFF0000u);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1, const float (&c)[4]) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
              "f"(c[2]), "f"(c[3]));
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
    static __device__ __forceinline__ void unpack(uint2 v, float (&f)[4]) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)),
                     b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
        f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1, const float (&c)[4]) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
            "{%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]),
              "f"(c[2]), "f"(c[3]));
    }
};

// What lane group r stands for: 16-byte piece of a word row, token of a group.
__device__ __forceinline__ int spread(int r) { return (r >> 1) + 4 * (r & 1); }

// NT: groups of 8 tokens that one pass over the weights serves.
template <typename T, int NT, bool ZERO>
__global__ void __launch_bounds__(kLinThreads, 2)
    int4_linear_kernel(const __grid_constant__ CUtensorMap w_map,
                       const __grid_constant__ CUtensorMap x_map,
                       const __grid_constant__ CUtensorMap s_map, const LinearArgs a,
                       const DevCtl ctl) {
    pdl_begin();
    using Ops = Half2Ops<T>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~(uintptr_t)1023);
    __shared__ uint64_t full[kLinStages], empty[kLinStages];
    __shared__ int abort_flag;
    cg::cluster_group cluster = cg::this_cluster();
    const int splits = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    const int n0 = blockIdx.y * kLinCols;
    const int t0 = blockIdx.z * (NT * 8);
    const int tokens = min(a.T - t0, NT * 8);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kLinStages; ++i) {
            mbar_init(smem_addr(&full[i]), 1);
            mbar_init(smem_addr(&empty[i]), kLinColWarps);
        }
        abort_flag = 0;
        mbar_init_fence();
    }
    __syncthreads();

    // this CTA's stages of four 32-wide K blocks (the last one may be short)
    const int blocks = a.K >> 5, all = (blocks + kLinDepth - 1) / kLinDepth;
    const int s0 = (int)((long long)all * rank / splits);
    const int stages = (int)((long long)all * (rank + 1) / splits) - s0;
    auto group_of = [&](int b) {
        return a.group_inv ? (int)__umulhi((uint32_t)b, a.group_inv) : b;
    };

    float sum[NT][2][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[i][h][q] = 0.0f;

    int issued = 0;                      // copy warp: stages filled
    if (warp == kLinMath) {
        // ---- copy warp
        const uint64_t once = policy_evict_first(), keep = policy_evict_last();
        const uint32_t bytes = kLinColWarps * kLinWordBox + kLinDepth / 2 * kLinTokenBox<NT> +
                               a.scale_rows * kLinScaleRow;
        RingPos pos;
        for (int s = 0; s < stages; ++s, pos.advance(kLinStages)) {
            if (s >= kLinStages &&
                !__all_sync(0xffffffffu, mbar_wait(smem_addr(&empty[pos.slot]), pos.phase ^ 1u,
                                                   &abort_flag, ctl, 23)))
                break;
            issued = s + 1;
            if (lane == 0) {
                const int b = (s0 + s) * kLinDepth;
                const uint32_t bar = smem_addr(&full[pos.slot]);
                const uint32_t dst = smem_addr(smem) + pos.slot * kLinStageBytes<NT>;
                mbar_expect_tx(bar, bytes);
#pragma unroll
                for (int i = 0; i < kLinColWarps; ++i)
                    tma_load_2d_hint(dst + i * kLinWordBox, &w_map, n0 + 32 * i, 4 * b, bar, once);
                tma_load_2d_hint(dst + kLinScaleAt<NT>, &s_map, n0, group_of(b), bar, once);
#pragma unroll
                for (int i = 0; i < kLinDepth / 2; ++i)
                    tma_load_2d_hint(dst + kLinTokenAt + i * kLinTokenBox<NT>, &x_map,
                                     b * 32 + 64 * i, t0, bar, keep);
            }
            __syncwarp();
        }
    } else {
        // ---- math warps
        const int cw = warp % kLinColWarps, kg = warp / kLinColWarps;
        const int r = lane >> 2, c = lane & 3, piece = spread(r);
        const int nc = min(n0 + 32 * cw + 4 * piece, a.N - 4);
        const int swz[2] = {(piece ^ c) << 4, (piece ^ (4 + c)) << 4};
        RingPos pos;
        for (int s = 0; s < stages; ++s, pos.advance(kLinStages)) {
            if (s % kLinKGroups != kg) continue;
            // Blocks past K multiply zero-filled activations with zero-filled scales.
            const int b = (s0 + s) * kLinDepth;
            uint32_t zp[kLinDepth];
            if (ZERO)
#pragma unroll
                for (int d = 0; d < kLinDepth; ++d)
                    zp[d] = (uint32_t)__ldg(a.zero + (long long)group_of(min(b + d, blocks - 1)) *
                                                         (a.N >> 3) + (nc >> 3)) >> (4 * (nc & 7));
            if (!__all_sync(0xffffffffu, mbar_wait(smem_addr(&full[pos.slot]), pos.phase,
                                                   &abort_flag, ctl, 24)))
                break;
            const uint8_t* stage = smem + pos.slot * kLinStageBytes<NT>;
            const uint8_t* ws = stage + cw * kLinWordBox + c * 128;
            const uint8_t* ss = stage + kLinScaleAt<NT> + cw * 64 + piece * 8;
            const uint8_t* xs = stage + kLinTokenAt + piece * 128;
#pragma unroll
            for (int d = 0; d < kLinDepth; ++d) {
                // word row 4 d + c: its 16-byte pieces are XORed with the row number
                const uint4 wv = *reinterpret_cast<const uint4*>(ws + d * 512 + swz[d & 1]);
                const int row = a.even_groups ? d * a.scale_rows >> 2
                                                                  : group_of(b + d) - group_of(b);
                const uint2 sv = *reinterpret_cast<const uint2*>(ss + row * kLinScaleRow);
                float sf[4];
                Ops::unpack(sv, sf);
                const uint32_t word[4] = {wv.x, wv.y, wv.z, wv.w};
                uint32_t q4[4][4];      // [column][nibble pair j, j + 4]
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t off =
                        Ops::kMagic + (ZERO ? (zp[d] >> (4 * q)) & 15u : 8u) * 0x00010001u;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        q4[q][j] =
                            Ops::sub(lop3_and_or(word[q] >> (4 * j), 0x000F000Fu, Ops::kMagic), off);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint4 x = *reinterpret_cast<const uint4*>(
                        xs + (d >> 1) * kLinTokenBox<NT> + i * 1024 + swz[d & 1]);
                    // natural pairs (0,1) (2,3) (4,5) (6,7) -> (0,4) (1,5) (2,6) (3,7)
                    const uint32_t x0 = __byte_perm(x.x, x.z, 0x5410),
                                   x1 = __byte_perm(x.x, x.z, 0x7632),
                                   x2 = __byte_perm(x.y, x.w, 0x5410),
                                   x3 = __byte_perm(x.y, x.w, 0x7632);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t lo[4] = {q4[2 * h][0], q4[2 * h + 1][0], q4[2 * h][1],
                                                q4[2 * h + 1][1]};
                        const uint32_t hi[4] = {q4[2 * h][2], q4[2 * h + 1][2], q4[2 * h][3],
                                                q4[2 * h + 1][3]};
                        const float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        float half[4], acc[4];
                        Ops::mma(half, lo, x0, x1, none);
                        Ops::mma(acc, hi, x2, x3, half);
                        // MMA row r or r + 8 (q >> 1) is column 2h + (q >> 1) of the lane's four
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            sum[i][h][q] =
                                fmaf(sf[2 * h + (q >> 1)], acc[q], sum[i][h][q]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&empty[pos.slot]));
        }
    }
    // After a wait that ran out (status word set, results undefined) the last
    // copies have to land before their memory is used again.
    __syncthreads();
    if (abort_flag && warp == kLinMath)
        for (int s = max(0, issued - kLinStages); s < issued; ++s)
            mbar_wait(smem_addr(&full[s % kLinStages]), (s / kLinStages) & 1, &abort_flag, ctl, 24,
                      false);
    __syncthreads();

    // Partial sums [math group][token][column] over the ring's memory.
    float* part = reinterpret_cast<float*>(smem);
    if (warp < kLinMath) {
        const int cw = warp % kLinColWarps, kg = warp / kLinColWarps;
        const int piece = spread(lane >> 2), c = lane & 3;
        // MMA column 2c + (q & 1) is token spread(2c + (q & 1)) = c + 4 (q & 1) of its eight
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    part[(kg * NT * 8 + 8 * i + c + 4 * (q & 1)) * kLinCols + 32 * cw + 4 * piece +
                         2 * h + (q >> 1)] = sum[i][h][q];
    }
    __syncthreads();
    constexpr int kOther = NT * 8 * kLinCols;       // the second math group's sums
    if (splits > 1) cluster.sync();
    // Output elements of this CTA: every splits-th run of a warp's 32 columns.
    for (int i = (warp * splits + rank) * 32 + lane; i < tokens * kLinCols;
         i += kLinThreads * splits) {
        const int t = i / kLinCols, col = n0 + i % kLinCols;
        if (col >= a.N) continue;
        float v = 0.0f;
        for (int k = 0; k < splits; ++k) {
            const float* p = cluster.map_shared_rank(part, k);
            v += p[i] + p[kOther + i];
        }
        if (a.bias) v += to_f32(static_cast<const T*>(a.bias)[col]);
        static_cast<T*>(a.y)[(long long)(t0 + t) * a.N + col] = from_f32<T>(v);
    }
    if (splits > 1) cluster.sync();      // peers may still read this CTA's sums
}

struct LinearIn {
    const void *x, *w, *scale;
    long long ldx;
    int groups;
};

template <typename T, int NT, bool ZERO>
int launch_linear(const LinearIn& in, const LinearArgs& a, int splits, const DeviceInfo* info,
                  cudaStream_t s) {
    constexpr CUtensorMapDataType dt = std::is_same<T, __half>::value
                                           ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap w_map, x_map, s_map;
    int rc;
    if ((rc = make_tmap_2d(&w_map, in.w, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, a.K / 8, a.N,
                           (uint64_t)a.N * 4, 32, 4 * kLinDepth, true)) != FERRET_OK ||
        (rc = make_tmap_2d(&x_map, in.x, dt, 2, a.T, a.K, (uint64_t)in.ldx * 2, 64, NT * 8,
                           true)) != FERRET_OK ||
        (rc = make_tmap_2d(&s_map, in.scale, dt, 2, in.groups, a.N, (uint64_t)a.N * 2, kLinCols,
                           a.scale_rows, false)) != FERRET_OK)
        return rc;
    const dim3 grid(splits, (a.N + kLinCols - 1) / kLinCols, (a.T + NT * 8 - 1) / (NT * 8));
    constexpr size_t smem = kLinStages * kLinStageBytes<NT> + 1024;
    static_assert(smem >= kLinKGroups * NT * 8 * kLinCols * sizeof(float) + 1024);
    auto kern = int4_linear_kernel<T, NT, ZERO>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess) {
        cudaGetLastError();
        return FERRET_ERR_CUDA;
    }
    return launch_kernel_cluster(kern, grid, dim3(kLinThreads), smem, splits, s, w_map, x_map,
                                 s_map, a, make_ctl(info));
}

template <typename T, int NT>
int launch_linear(const LinearIn& in, const LinearArgs& a, int splits, const DeviceInfo* info,
                  cudaStream_t s) {
    return a.zero ? launch_linear<T, NT, true>(in, a, splits, info, s)
                  : launch_linear<T, NT, false>(in, a, splits, info, s);
}

template <typename T>
int run_linear(const LinearIn& in, const LinearArgs& a, const DeviceInfo* info, cudaStream_t s) {
    // The fewest splits that give every SM a CTA, as long as a CTA keeps four
    // stages of K: a split costs its two cluster barriers (16 tokens x 7168 x
    // 32768: 53 us unsplit, 57 us split in two or four).
    const long long tiles = ((long long)a.N + kLinCols - 1) / kLinCols;
    int splits = 1;
    while (splits < kLinMaxCluster && tiles * splits < (long long)info->num_sms &&
           a.K / 32 >= splits * 2 * 4 * kLinDepth)
        splits *= 2;
    if (a.T <= 8) return launch_linear<T, 1>(in, a, splits, info, s);
    if (a.T <= 16) return launch_linear<T, 2>(in, a, splits, info, s);
    return launch_linear<T, 4>(in, a, splits, info, s);
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
    if (!aligned16(x) || !aligned16(w) || !aligned16(w_scale) || !aligned_to(w_zero, 4) ||
        !aligned_to(bias, 2) || !aligned_to(y, 2))
        return FERRET_ERR_ALIGN;
    DeviceInfo* info = nullptr;
    int rc = current_device(&info);
    if (rc != FERRET_OK) return rc;
    // ceil(2^32 / blocks of a group): exact quotients as long as the product of
    // block number and group length stays below 2^32 (K <= 2^20)
    const uint32_t blocks = group / 32;
    const uint32_t inv = blocks == 1 ? 0u : (uint32_t)(((1ull << 32) + blocks - 1) / blocks);
    // a stage starts at a multiple of 128: the groups it can touch
    const int rows = 128 % group == 0 ? 128 / group : group % 128 == 0 ? 1 : 128 / group + 2;
    const LinearIn in{x, w, w_scale, ldx, K / group};
    const LinearArgs a{w_zero, bias, y, T, K, N, inv, rows,
                       128 % group == 0 || group % 128 == 0};
    const cudaStream_t s = as_stream(stream);
    return dtype == FERRET_BF16 ? run_linear<__nv_bfloat16>(in, a, info, s)
                                : run_linear<__half>(in, a, info, s);
}
