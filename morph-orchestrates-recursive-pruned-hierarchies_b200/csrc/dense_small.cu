// Products for a few tokens (1 to 32 rows): bound by reading the weights once.
//
// A warp multiplies 16 weight rows by up to 8, 16 or 32 tokens with mma.sync (M = 16 weight rows, N = 8
// tokens): at these sizes the tensor cores idle either way, and operands that go straight from
// memory into registers need no staging, so every warp keeps its own loads in flight.  Which k a
// register holds is free as long as both operands agree, so a lane takes 16 neighbouring bytes of its
// row (8 values of 16 bits, 16 of 8 bits), four lanes a 64-byte piece of a row, and word i of the 16
// bytes is the i-th operand register.  With the gate, a warp's 16 rows are 8 gate rows and the 8 up rows
// of the same hidden columns: a thread then holds both sums of its outputs.
//
// The warps of a CTA take the pieces of k in turn and add their sums through shared memory in warp
// order; where there are too few row tiles for the SMs, a cluster of CTAs shares a tile's k and adds
// in rank order.  The order is fixed, so the same call gives the same bits.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.h"
#include "dense_small.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;

enum Kind { kBf16 = 0, kF16 = 1, k8 = 2 };

__device__ __forceinline__ uint4 load_stream(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <int KIND, int XT, int WT>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
#define SMALL_MMA(SHAPE_TYPES)                                                                                       \
    asm volatile("mma.sync.aligned." SHAPE_TYPES " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"           \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if constexpr (KIND == kBf16) SMALL_MMA("m16n8k16.row.col.f32.bf16.bf16.f32");
    else if constexpr (KIND == kF16) SMALL_MMA("m16n8k16.row.col.f32.f16.f16.f32");
    else if constexpr (WT == MORTAR_E4M3 && XT == MORTAR_E4M3) SMALL_MMA("m16n8k32.row.col.f32.e4m3.e4m3.f32");
    else if constexpr (WT == MORTAR_E4M3) SMALL_MMA("m16n8k32.row.col.f32.e4m3.e5m2.f32");
    else if constexpr (XT == MORTAR_E4M3) SMALL_MMA("m16n8k32.row.col.f32.e5m2.e4m3.f32");
    else SMALL_MMA("m16n8k32.row.col.f32.e5m2.e5m2.f32");
#undef SMALL_MMA
}

__device__ __forceinline__ float silu(float g) { return __fdividef(g, 1.f + __expf(-g)); }

__device__ __forceinline__ void store(const small::Params &p, long long idx, float v) {
    if (p.out_dtype == MORTAR_F32) reinterpret_cast<float *>(p.out)[idx] = v;
    else if (p.out_dtype == MORTAR_BF16) reinterpret_cast<__nv_bfloat16 *>(p.out)[idx] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half *>(p.out)[idx] = __float2half_rn(v);
}

// NT: groups of 8 tokens.  A piece is 64 bytes of k; `kUnroll` pieces of a warp are in flight together (for 8-bit
// operands two pieces make a block with its own scales).
template <int KIND, int XT, int WT, int NT, bool GATED>
__global__ void __launch_bounds__(kThreads)
small_kernel(const __grid_constant__ small::Params p) {
    constexpr int kUnroll = 4;
    __shared__ float part[kWarps][16][8 * NT + 1];
    __shared__ float tile[16][8 * NT];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int tile_id = blockIdx.x / ranks, n0 = tile_id * (GATED ? 8 : 16);
    // rows of w of this thread: accumulator rows g and g + 8
    const int row_a = n0 + g, row_b = GATED ? p.up_row + n0 + g : n0 + g + 8;
    const bool in_a = row_a < p.n, in_b = GATED ? in_a : row_b < p.n;
    const uint8_t *wa = p.w + (long long)row_a * p.ldw + 16 * t, *wb = p.w + (long long)row_b * p.ldw + 16 * t;
    const int pieces = (p.k_bytes + 63) >> 6;
    const int step = KIND == k8 ? 2 : 1;                             // pieces that stay with one warp
    const int slots = kWarps * ranks, slot = rank * kWarps + warp;

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;

    // the j-th piece of this warp
    auto piece_of = [&](int j) { return KIND == k8 ? ((j >> 1) * slots + slot) * 2 + (j & 1) : j * slots + slot; };
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 a[kUnroll], b[kUnroll];
    auto fetch = [&](int j0) {
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int at = piece_of(j0 + j) * 64, in = at + 16 * t < p.k_bytes;
            a[j] = in && in_a ? load_stream(wa + at) : zero;
            b[j] = in && in_b ? load_stream(wb + at) : zero;
        }
    };
    fetch(0);
    if (p.after_previous) asm volatile("griddepcontrol.wait;\n" ::: "memory");
    else asm volatile("griddepcontrol.launch_dependents;\n");
    for (int j0 = 0; piece_of(j0) < pieces; j0 += kUnroll) {
        uint4 x[NT][kUnroll];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) {
                const int at = piece_of(j0 + j) * 64 + 16 * t, m = 8 * i + g;
                x[i][j] = at < p.k_bytes && m < p.rows ? *reinterpret_cast<const uint4 *>(p.x + m * p.ldx + at) : zero;
            }
        uint4 ca[kUnroll], cb[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) { ca[j] = a[j]; cb[j] = b[j]; }
        fetch(j0 + kUnroll);
        if constexpr (KIND != k8) {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    mma<KIND, XT, WT>(acc[i], ca[j].x, cb[j].x, ca[j].y, cb[j].y, x[i][j].x, x[i][j].y);
                    mma<KIND, XT, WT>(acc[i], ca[j].z, cb[j].z, ca[j].w, cb[j].w, x[i][j].z, x[i][j].w);
                }
        } else {
#pragma unroll
            for (int j = 0; j < kUnroll; j += 2) {
                const int blk = piece_of(j0 + j) >> 1;
                if (2 * blk >= pieces) continue;
                const float sa = in_a ? __ldg(p.ws + (long long)(row_a >> 7) * p.ld_ws + blk) : 0.f;
                const float sb = in_b ? __ldg(p.ws + (long long)(row_b >> 7) * p.ld_ws + blk) : 0.f;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mma<KIND, XT, WT>(d, ca[j + h].x, cb[j + h].x, ca[j + h].y, cb[j + h].y, x[i][j + h].x, x[i][j + h].y);
                        mma<KIND, XT, WT>(d, ca[j + h].z, cb[j + h].z, ca[j + h].w, cb[j + h].w, x[i][j + h].z, x[i][j + h].w);
                    }
                    const int m = 8 * i + 2 * t;
                    const float x0 = m < p.rows ? p.xs[m * p.ld_xs + blk] : 0.f, x1 = m + 1 < p.rows ? p.xs[(m + 1) * p.ld_xs + blk] : 0.f;
                    acc[i][0] = fmaf(d[0], sa * x0, acc[i][0]);
                    acc[i][1] = fmaf(d[1], sa * x1, acc[i][1]);
                    acc[i][2] = fmaf(d[2], sb * x0, acc[i][2]);
                    acc[i][3] = fmaf(d[3], sb * x1, acc[i][3]);
                }
            }
        }
    }
    (void)step;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        part[warp][g][8 * i + 2 * t] = acc[i][0];
        part[warp][g][8 * i + 2 * t + 1] = acc[i][1];
        part[warp][g + 8][8 * i + 2 * t] = acc[i][2];
        part[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += kThreads) {
        const int r = i & 15, m = i >> 4;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += part[w][r][m];
        tile[r][m] = s;
    }
    if (ranks > 1) {
        cluster.sync();                                              // every rank's sums are there
        if (rank == 0)
            for (int i = threadIdx.x; i < 16 * 8 * NT; i += kThreads) {
                float s = tile[i & 15][i >> 4];
                for (int r = 1; r < ranks; ++r) s += cluster.map_shared_rank(&tile[0][0], r)[(i & 15) * 8 * NT + (i >> 4)];
                tile[i & 15][i >> 4] = s;                            // read by this thread's peers after the barrier below
            }
        cluster.sync();                                              // and no rank leaves before they have been read
        if (rank) return;
    } else {
        __syncthreads();
    }
    constexpr int kOut = GATED ? 8 : 16;
    for (int i = threadIdx.x; i < kOut * 8 * NT; i += kThreads) {
        const int r = i % kOut, m = i / kOut;
        if (m < p.rows && n0 + r < p.n) {
            const float v = GATED ? silu(tile[r][m]) * tile[r + 8][m] : tile[r][m];
            store(p, m * p.ld_out + n0 + r, v);
        }
    }
}

template <int KIND, int XT, int WT, int NT, bool GATED>
int run(const small::Params &p, int sms, cudaStream_t st) {
    const int tiles = (p.n + (GATED ? 7 : 15)) / (GATED ? 8 : 16);
    const int pieces = (p.k_bytes + 63) / 64;
    // four CTAs an SM, as long as a warp keeps two pieces (a whole scaled block) to itself
    int ranks = 1;
    while (ranks < 8 && tiles * ranks * 2 <= 4 * sms && pieces >= 2 * kWarps * ranks * 2) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.after_previous ? 2 : 1;
    MORTAR_CUDA_CHECK(cudaLaunchKernelEx(&cfg, small_kernel<KIND, XT, WT, NT, GATED>, p));
    return MORTAR_OK;
}

template <int KIND, int XT, int WT>
int pick(const small::Params &p, int sms, cudaStream_t st) {
    if (p.up_row) {
        if (p.rows <= 8) return run<KIND, XT, WT, 1, true>(p, sms, st);
        if (p.rows <= 16) return run<KIND, XT, WT, 2, true>(p, sms, st);
        return run<KIND, XT, WT, 4, true>(p, sms, st);
    }
    if (p.rows <= 8) return run<KIND, XT, WT, 1, false>(p, sms, st);
    if (p.rows <= 16) return run<KIND, XT, WT, 2, false>(p, sms, st);
    return run<KIND, XT, WT, 4, false>(p, sms, st);
}

}  // namespace

int small::launch(const small::Params &p, int sms, cudaStream_t st) {
    if (p.w_dtype == MORTAR_BF16) return pick<kBf16, 0, 0>(p, sms, st);
    if (p.w_dtype == MORTAR_F16) return pick<kF16, 0, 0>(p, sms, st);
    if (p.w_dtype == MORTAR_E4M3)
        return p.x_dtype == MORTAR_E4M3 ? pick<k8, MORTAR_E4M3, MORTAR_E4M3>(p, sms, st)
                                        : pick<k8, MORTAR_E5M2, MORTAR_E4M3>(p, sms, st);
    return p.x_dtype == MORTAR_E4M3 ? pick<k8, MORTAR_E4M3, MORTAR_E5M2>(p, sms, st)
                                    : pick<k8, MORTAR_E5M2, MORTAR_E5M2>(p, sms, st);
}
