// Products for a few tokens (up to 32 rows; 8-bit operands of more than 16 only where the weight is narrow): bound by reading the weights once.
//
// A warp multiplies 16 weight rows by up to 8, 16 or 32 tokens with mma.sync (M = 16 weight rows, N = 8
// tokens): at these sizes the tensor cores idle either way, and operands that go straight from
// memory into registers need no staging, so every warp keeps its own loads in flight.  Which k a
// register holds is free as long as both operands agree, so a lane takes 16 neighbouring bytes of its
// row (8 values of 16 bits, 16 of 8 bits), four lanes a 64-byte piece of a row, and word i of the 16
// bytes is the i-th operand register.  With the gate, a warp's 16 rows are 8 gate rows and the 8 up rows
// of the same hidden columns: a thread then holds both sums of its outputs.
//
// One CTA of sixteen warps an SM walks the row tiles; its warps take the pieces of k in turn, the next
// tile's weights are on their way while this one's sums are added through shared memory, in warp order.
// Where there are too few row tiles for the SMs, a cluster of CTAs shares a tile's k and adds in rank
// order.  The order is fixed, so the same call gives the same bits.
//
// One token, 2048/5632: gate/up (46 MB) 13.7 us = 3.4 TB/s, down (23 MB) 11.1 us, 18.3 us together since the second
// fetches weights while the first ends.  4 tokens against the 8-bit 2048 -> 11264 matrix (23 MB): 11.6 us.  With
// several microseconds of launch and first access in each, a longer queue of weights (64 KB an SM here) has
// nothing left to hide; CTAs of one tile each instead of a queue across tiles took 24.6 us for the block.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.h"
#include "dense_small.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kWarps = 16;
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

// Weights of one batch: `kUnroll` pieces of two rows, and their block scales.
template <int N> struct Batch { uint4 a[N], b[N]; float sa, sb; };

// NT: groups of 8 tokens.  A piece is 64 bytes of k, a batch `kUnroll` of them a warp, and `kSlots` batches, of this tile
// and the next ones, are on their way or at work: about 64 KB an SM in flight (for 8-bit operands a batch is one block
// with its own scales).
template <int KIND, int XT, int WT, int NT, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
small_kernel(const __grid_constant__ small::Params p) {
    constexpr int kUnroll = KIND != k8 && NT == 1 ? 4 : 2;
    constexpr int kSlots = kUnroll == 4 || NT == 4 ? 2 : 3;
    __shared__ float part[kWarps][16][8 * NT + 1];
    __shared__ float tile_s[16][8 * NT];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int kTileRows = GATED ? 8 : 16;
    const int tiles = (p.n + kTileRows - 1) / kTileRows, tile_step = (int)gridDim.x / ranks;
    const int pieces = (p.k_bytes + 63) >> 6, slots = kWarps * ranks, slot = rank * kWarps + warp;

    // the j-th piece of this warp; every warp makes the same number of batches, the last ones empty-handed
    auto piece_of = [&](int j) { return KIND == k8 ? ((j >> 1) * slots + slot) * 2 + (j & 1) : j * slots + slot; };
    const int batches = KIND == k8 ? (pieces + 2 * slots - 1) / (2 * slots) : (pieces + kUnroll * slots - 1) / (kUnroll * slots);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    Batch<kUnroll> w[kSlots];
    int next_tile = (int)blockIdx.x / ranks, next_batch = 0;             // what is fetched next
    auto fetch = [&](Batch<kUnroll> &s) {
        if (next_tile >= tiles) return;
        // rows of w of this thread: accumulator rows g and g + 8
        const int row_a = next_tile * kTileRows + g, row_b = GATED ? p.up_row + row_a : row_a + 8;
        const bool in_a = row_a < p.n, in_b = GATED ? in_a : row_b < p.n;
        const uint8_t *wa = p.w + (long long)row_a * p.ldw + 16 * t, *wb = p.w + (long long)row_b * p.ldw + 16 * t;
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int at = piece_of(next_batch * kUnroll + j) * 64;
            const bool in = at + 16 * t < p.k_bytes;
            s.a[j] = in && in_a ? load_stream(wa + at) : zero;
            s.b[j] = in && in_b ? load_stream(wb + at) : zero;
        }
        if constexpr (KIND == k8) {
            const int blk = piece_of(next_batch * kUnroll) >> 1;
            const bool in = 2 * blk < pieces;
            s.sa = in && in_a ? __ldg(p.ws + (long long)(row_a >> 7) * p.ld_ws + blk) : 0.f;
            s.sb = in && in_b ? __ldg(p.ws + (long long)(row_b >> 7) * p.ld_ws + blk) : 0.f;
        }
        if (++next_batch == batches) {
            next_batch = 0;
            next_tile += tile_step;
        }
    };
#pragma unroll
    for (int s = 0; s < kSlots; ++s) fetch(w[s]);
    if (p.after_previous) asm volatile("griddepcontrol.wait;\n" ::: "memory");
    else asm volatile("griddepcontrol.launch_dependents;\n");

    uint4 x[NT][kUnroll];
    float xs[NT][2];
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    int tile = (int)blockIdx.x / ranks, batch = 0;
    bool have_x = false;                                                 // one batch a tile: its tokens stay
    while (tile < tiles) {
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
            if (tile >= tiles) break;
            if (!have_x) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
#pragma unroll
                    for (int j = 0; j < kUnroll; ++j) {
                        const int at = piece_of(batch * kUnroll + j) * 64 + 16 * t, m = 8 * i + g;
                        x[i][j] = at < p.k_bytes && m < p.rows ? *reinterpret_cast<const uint4 *>(p.x + m * p.ldx + at) : zero;
                    }
                    if constexpr (KIND == k8) {
                        const int blk = piece_of(batch * kUnroll) >> 1, m = 8 * i + 2 * t;
                        const bool in = 2 * blk < pieces;
                        xs[i][0] = in && m < p.rows ? p.xs[m * p.ld_xs + blk] : 0.f;
                        xs[i][1] = in && m + 1 < p.rows ? p.xs[(m + 1) * p.ld_xs + blk] : 0.f;
                    }
                }
                have_x = batches == 1;
            }
            Batch<kUnroll> &c = w[s];
            if constexpr (KIND != k8) {
#pragma unroll
                for (int j = 0; j < kUnroll; ++j)
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        mma<KIND, XT, WT>(acc[i], c.a[j].x, c.b[j].x, c.a[j].y, c.b[j].y, x[i][j].x, x[i][j].y);
                        mma<KIND, XT, WT>(acc[i], c.a[j].z, c.b[j].z, c.a[j].w, c.b[j].w, x[i][j].z, x[i][j].w);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        mma<KIND, XT, WT>(d, c.a[h].x, c.b[h].x, c.a[h].y, c.b[h].y, x[i][h].x, x[i][h].y);
                        mma<KIND, XT, WT>(d, c.a[h].z, c.b[h].z, c.a[h].w, c.b[h].w, x[i][h].z, x[i][h].w);
                    }
                    acc[i][0] = fmaf(d[0], c.sa * xs[i][0], acc[i][0]);
                    acc[i][1] = fmaf(d[1], c.sa * xs[i][1], acc[i][1]);
                    acc[i][2] = fmaf(d[2], c.sb * xs[i][0], acc[i][2]);
                    acc[i][3] = fmaf(d[3], c.sb * xs[i][1], acc[i][3]);
                }
            }
            fetch(c);
            if (++batch < batches) continue;
            batch = 0;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                part[warp][g][8 * i + 2 * t] = acc[i][0];
                part[warp][g][8 * i + 2 * t + 1] = acc[i][1];
                part[warp][g + 8][8 * i + 2 * t] = acc[i][2];
                part[warp][g + 8][8 * i + 2 * t + 1] = acc[i][3];
                acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * 8 * NT; i += kThreads) {
                const int r = i & 15, m = i >> 4;
                float sum = 0.f;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) sum += part[v][r][m];
                tile_s[r][m] = sum;
            }
            if (ranks > 1) cluster.sync();                           // every rank's sums are there
            else __syncthreads();
            if (rank == 0)
                for (int i = threadIdx.x; i < kTileRows * 8 * NT; i += kThreads) {
                    const int r = i % kTileRows, m = i / kTileRows;
                    if (m >= p.rows || tile * kTileRows + r >= p.n) continue;
                    float v = tile_s[r][m], u = GATED ? tile_s[r + 8][m] : 0.f;
                    for (int q = 1; q < ranks; ++q) {
                        const float *other = cluster.map_shared_rank(&tile_s[0][0], q);
                        v += other[r * 8 * NT + m];
                        if (GATED) u += other[(r + 8) * 8 * NT + m];
                    }
                    if (GATED) v = silu(v) * u;
                    store(p, m * p.ld_out + tile * kTileRows + r, v);
                }
            // a tile's sums are not written again, and no rank leaves, before they have been read; in one CTA the next
            // tile's first barrier sees to that
            if (ranks > 1) cluster.sync();
            tile += tile_step;
        }
    }
}

template <int KIND, int XT, int WT, int NT, bool GATED>
int run(const small::Params &p, int sms, cudaStream_t st) {
    const int tiles = (p.n + (GATED ? 7 : 15)) / (GATED ? 8 : 16);
    const int pieces = (p.k_bytes + 63) / 64;
    // a CTA an SM, as long as a warp keeps a piece (a whole scaled block) to itself
    int ranks = 1;
    while (ranks < 8 && tiles * ranks * 2 <= sms && pieces >= (KIND == k8 ? 2 : 1) * kWarps * ranks * 2) ranks *= 2;
    const int at_once = sms / ranks < tiles ? sms / ranks : tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(at_once * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    cfg.attrs = at;
    if (ranks > 1) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)ranks;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
    }
    if (p.after_previous) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
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
