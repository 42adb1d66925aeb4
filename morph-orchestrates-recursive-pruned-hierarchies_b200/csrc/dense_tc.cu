// The dense gated feed-forward block, forward and backward, on the 5th-generation tensor cores.
//
//   gu = x Wgu^T (gate columns first), h = silu(g) * u, y = h Wd^T
//   dh = dy Wd,  dg = dh u (s + a (1 - s)),  du = dh a   with s = sigmoid(g), a = g s
//   dx = [dg, du] Wgu,  dWgu = [dg, du]^T x,  dWd = dy^T h
//
// (`_SwiGLUMortar.forward` before it is carved, morph/model/transformer.py:402-431, and its
// gradient).  All six products run in one kernel, C[M][N] = sum_k A[m][k] B[n][k], whose operands lie
// in memory with either index contiguous: the tile copies and the matrix descriptors take both, so
// nothing is transposed.  Gate and up products of the same hidden columns are the two halves of one
// accumulator tile, so the gate is applied where the sums are read, and the backward of the gate is
// the epilogue of dh.
//
// One cluster of two CTAs computes a tile of 256 rows and 256 or 128 columns (each CTA 128 rows; the B operand is
// split between their shared memories): per SM and 64-wide step 16 KB of A and 64 bytes a column of B cross from L2,
// half of what two single CTAs would read, which is what keeps the copies ahead of the MMAs.  Warp 0
// issues the copies of its CTA, one thread of CTA 0 issues the MMAs of both, warps 2..17 read the
// accumulators (two sets, so that a tile's epilogue runs under the next tile's MMAs).
// Every wait is bounded.
//
// What bounds it: at 8192 x 2048/5632 every launch draws its operands from L2 at 12.2 to 12.4 TB/s (128 KB a
// 128-wide step and cluster of 256 columns), which is all that L2 gives: gate/up 236 us = 1600 TFLOP/s without and 278 us with
// the kept sums, down 137 us = 1380, dh 194 us (its epilogue moves 0.7 GB more), the three last products
// together 594 us = 1590 TFLOP/s with the tensor pipe busy 88% of the time.  A hand-off of 64-wide steps with
// one wait for four MMAs reached 1200.  Under the power cap of a long run the whole step comes to 1150 of the
// library product's sustained 1400 TFLOP/s.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>
#include "common.h"
#include "dense_small.cuh"
#include "tc_pair.cuh"

namespace {

constexpr int kStageA = 128 * 256;               // this CTA's 128 rows, 128 elements of 2 bytes each
constexpr int kEpiWarps = 16;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr int kMaxProblems = 3;
constexpr int kClusters = 74;                    // CTA pairs that run at once

// BN: accumulator columns of a tile, 256 or 128
template <int BN> struct Shape {
    static constexpr int kStages = BN == 256 ? 3 : 4;
    static constexpr int kStageB = BN / 2 * 256;
    static constexpr int kStage = kStageA + kStageB;
    static constexpr int kSmem = kStages * kStage + (2 * kStages + 4) * 8 + 1024;
    static_assert(kSmem <= 227 * 1024, "shared memory budget");
};

__device__ int g_dense_error;

enum Epilogue { kStore = 0, kSwiglu = 1, kSwigluBackward = 2 };

struct Problem {
    void *out;               // 16-bit [m][n]
    long long ld_out;
    long long m;             // rows of C
    int n;                   // columns of C (hidden columns for kSwiglu)
    int tiles_m, tiles_n;
    int k_steps;             // 128-wide steps of the reduction
    int a_mn, b_mn;          // 1: the operand's row index is the contiguous one in memory
    int first_item;
    int splits;              // parts of the reduction, an item each (kStore only)
    float *partial;          // splits > 1: fp32 [splits][m][n] instead of `out`
};

struct DenseParams {
    CUtensorMap map_a[kMaxProblems], map_b[kMaxProblems];
    Problem prob[kMaxProblems];
    int n_problems, n_items;
    int half;                // 1: fp16, 0: bf16
    int d_ff;                // kSwiglu / kSwigluBackward: rows between a gate row and its up row
    float *gu;               // kSwiglu: where gate and up sums are kept ([m][2 d_ff], or NULL); kSwigluBackward: read
    void *hidden;            // unused by kStore
    long long ld_gu;
};

// exp2-based exponential and an approximate quotient, off by 2^-22 (1 + |g|) at worst; the result is rounded to 16 bits
__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// 16 accumulator columns -> 16 16-bit values of one row, 32 bytes at a time: every row starts on 32 bytes and every
// width is a multiple of 16
__device__ __forceinline__ void store16(void *base, long long idx, const uint32_t (&v)[16], bool half) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = tc::pack16(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), half);
    tc::store_v8(reinterpret_cast<uint16_t *>(base) + idx, w);
}

// 16 accumulator columns as they are
__device__ __forceinline__ void store16_f32(float *dst, const uint32_t (&v)[16]) {
    uint32_t lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { lo[i] = v[i]; hi[i] = v[8 + i]; }
    tc::store_v8(dst, lo);
    tc::store_v8(dst + 8, hi);
}

struct TileId { int p, tm, tn, split, k_begin, k_end; };

// Items walk a problem's tiles in bands of 8 tile rows, column by column, so that the clusters at work
// share few A and B panels.
__device__ __forceinline__ TileId tile_of(const DenseParams &p, int item) {
    TileId t;
    t.p = 0;
    while (t.p + 1 < p.n_problems && item >= p.prob[t.p + 1].first_item) ++t.p;
    const Problem &q = p.prob[t.p];
    int i = item - q.first_item;
    t.split = q.splits > 1 ? i % q.splits : 0;
    t.k_begin = 0;
    t.k_end = q.k_steps;
    if (q.splits > 1) {
        i /= q.splits;
        t.k_begin = (int)((long long)q.k_steps * t.split / q.splits);
        t.k_end = (int)((long long)q.k_steps * (t.split + 1) / q.splits);
    }
    const int band = i / (8 * q.tiles_n), r = i - band * 8 * q.tiles_n;
    const int h = min(8, q.tiles_m - band * 8);
    t.tn = r / h;
    t.tm = band * 8 + r - t.tn * h;
    return t;
}

template <int EPI, int kBN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
dense_pair_kernel(const __grid_constant__ DenseParams p) {
    constexpr int kStages = Shape<kBN>::kStages, kStageB = Shape<kBN>::kStageB, kStage = Shape<kBN>::kStage, kTmemCols = 2 * kBN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(stages + kStages * kStage), *empty = full + kStages;
    uint64_t *acc_full = empty + kStages, *acc_empty = acc_full + 2;
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < kStages; ++s) { tc::mbar_init(tc::smem_u32(&full[s]), 1); tc::mbar_init(tc::smem_u32(&empty[s]), 1); }
        for (int s = 0; s < 2; ++s) { tc::mbar_init(tc::smem_u32(&acc_full[s]), 1); tc::mbar_init(tc::smem_u32(&acc_empty[s]), 2 * kEpiWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(tc::smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();                                   // barriers of both CTAs are initialised
    tc::fence_after();
    tc::let_next();
    tc::after_previous();                                 // returns at once when this launch waits for none
    const uint32_t tmem = tmem_base_s;
    volatile int *abort_flag = &abort_s;

    if (warp == 0) {
        // ---------------- copies: one thread in each CTA, completing on CTA 0's barriers ----------------
        if (lane == 0) {
            const uint32_t full_lead = tc::cluster_addr(tc::smem_u32(full), 0);
            const uint32_t empty0 = tc::smem_u32(empty), stage0 = tc::smem_u32(stages);
            uint32_t s = 0, parity = 1;
            bool ok = true;
            for (int item = cluster_id; item < p.n_items && ok; item += n_clusters) {
                const TileId t = tile_of(p, item);
                const Problem &q = p.prob[t.p];
                const CUtensorMap *ma = &p.map_a[t.p], *mb = &p.map_b[t.p];
                const int row0 = t.tm * 256 + (int)rank * 128;
                const int col0 = EPI == kSwiglu ? t.tn * (kBN / 2) + (rank ? p.d_ff : 0) : t.tn * kBN + (int)rank * (kBN / 2);
                for (int k = t.k_begin; k < t.k_end; ++k) {
                    if (!tc::mbar_wait(empty0 + 8 * s, parity, abort_flag, &g_dense_error, 1)) { ok = false; break; }
                    const uint32_t bar = full_lead + 8 * s, dst = stage0 + s * kStage;
                    if (rank == 0) tc::mbar_arrive_expect_tx(tc::smem_u32(&full[s]), 2 * kStage);
                    // rows contiguous in memory: boxes of 64 rows x 128 k; k contiguous: 128 rows x 64 k
                    if (q.a_mn) {
                        tc::load_pair(dst, ma, row0, k * 128, bar);
                        tc::load_pair(dst + 16384, ma, row0 + 64, k * 128, bar);
                    } else {
                        tc::load_pair(dst, ma, k * 128, row0, bar);
                        tc::load_pair(dst + 16384, ma, k * 128 + 64, row0, bar);
                    }
                    if (q.b_mn) {
#pragma unroll
                        for (int i = 0; i < kBN / 128; ++i)
                            tc::load_pair(dst + kStageA + i * 16384, mb, col0 + i * 64, k * 128, bar);
                    } else {
                        tc::load_pair(dst + kStageA, mb, k * 128, col0, bar);
                        tc::load_pair(dst + kStageA + kStageB / 2, mb, k * 128 + 64, col0, bar);
                    }
                    if (++s == kStages) { s = 0; parity ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issue: one thread of CTA 0 for the pair ----------------
        if (rank == 0 && lane == 0) {
            // D fp32 (bit 4); A and B type at bits 7 and 10 (0 fp16, 1 bf16); M/N-major at bits 15 and 16;
            // N >> 3 at bit 17, M >> 4 at bit 24 (M = 256 over the pair)
            const uint32_t type = p.half ? 0u : (1u << 7) | (1u << 10);
            const uint32_t idesc0 = (1u << 4) | type | ((uint32_t)(kBN >> 3) << 17) | ((256u >> 4) << 24);
            const uint32_t full0 = tc::smem_u32(full), empty0 = tc::smem_u32(empty);
            const uint32_t stage0 = tc::smem_u32(stages);
            uint32_t s = 0, parity = 0;
            int it = 0;
            bool ok = true, ready = tc::mbar_try_wait(full0, 0);
            for (int item = cluster_id; item < p.n_items && ok; item += n_clusters, ++it) {
                const TileId t = tile_of(p, item);
                const Problem &q = p.prob[t.p];
                const int buf = it & 1, k_steps = t.k_end - t.k_begin;
                const uint32_t acc = tmem + buf * kBN;
                const uint32_t idesc = idesc0 | ((uint32_t)q.a_mn << 15) | ((uint32_t)q.b_mn << 16);
                // k contiguous: a row's 64 k are 128 bytes, 16 of them 32 bytes further, the next 64 k one box further.
                // Rows contiguous: one k is 128 bytes (64 rows), 16 of them 2048 bytes, the next 64 rows one box further
                const uint64_t da = tc::make_smem_desc(stage0, q.a_mn ? 16384 : 16, 1024, 2);
                const uint64_t db = tc::make_smem_desc(stage0 + kStageA, q.b_mn ? 16384 : 16, 1024, 2);
                const uint64_t step_a = q.a_mn ? 2048 >> 4 : 32 >> 4, step_b = q.b_mn ? 2048 >> 4 : 32 >> 4;
                const uint64_t half_a = q.a_mn ? 8192 >> 4 : 16384 >> 4, half_b = q.b_mn ? 8192 >> 4 : (uint64_t)(kStageB / 2) >> 4;
                if (!tc::mbar_wait(tc::smem_u32(&acc_empty[buf]), ((it >> 1) & 1) ^ 1u, abort_flag, &g_dense_error, 2)) break;
                tc::fence_after();
                for (int k = 0; k < k_steps; ++k) {
                    if (!ready && !tc::mbar_wait(full0 + 8 * s, parity, abort_flag, &g_dense_error, 3)) { ok = false; break; }
                    const uint64_t at = (uint64_t)(s * (kStage >> 4));
                    const uint32_t bar = empty0 + 8 * s;
                    if (++s == kStages) { s = 0; parity ^= 1; }
                    ready = tc::poll_mma8_f16(full0 + 8 * s, parity, acc, da + at, db + at, step_a, step_b, half_a, half_b, idesc, k);
                    tc::commit_both(bar);
                }
                if (!ok) break;
                tc::commit_both(tc::smem_u32(&acc_full[buf]));
            }
        }
    } else {
        // ---------------- epilogue: warp w reads tensor-memory lanes 32 (w % 4) .. +31 ----------------
        const int quarter = warp & 3, side = (warp - 2) >> 2;
        const bool half = p.half != 0;
        int it = 0;
        for (int item = cluster_id; item < p.n_items; item += n_clusters, ++it) {
            const TileId t = tile_of(p, item);
            const Problem &q = p.prob[t.p];
            const int buf = it & 1;
            const long long row = (long long)t.tm * 256 + (long long)rank * 128 + quarter * 32 + lane;
            if (!tc::mbar_wait(tc::smem_u32(&acc_full[buf]), (it >> 1) & 1, abort_flag, &g_dense_error, 4)) break;
            tc::fence_after();
            const uint32_t taddr = tmem + buf * kBN + ((uint32_t)(quarter * 32) << 16);
            // 16 columns at a time: sixteen warps of 96 registers hide each other's waits for tensor memory, the special
            // function unit and memory better than eight that take 32 (backward at 4093 x 768/2048: 100 -> 89 us).  Turning
            // the pieces in shared memory so that lanes lie side by side in memory changed nothing: see the header
            if (EPI == kStore) {
#pragma unroll 2
                for (int c = side * (kBN / 4); c < (side + 1) * (kBN / 4); c += 16) {
                    uint32_t v[16];
                    __syncwarp();                                     // lanes whose row does not exist are back
                    tc::ld16_ahead(taddr + c, v);
                    tc::wait_ld();
                    const int col = t.tn * kBN + c;
                    if (row >= q.m || col >= q.n) continue;
                    if (q.splits == 1) store16(q.out, row * q.ld_out + col, v, half);
                    else store16_f32(q.partial + ((long long)t.split * q.m + row) * q.n + col, v);
                }
            } else if (EPI == kSwiglu) {
#pragma unroll 1
                for (int c = side * (kBN / 8); c < (side + 1) * (kBN / 8); c += 16) {
                    uint32_t g[16], u[16];
                    __syncwarp();
                    tc::ld16_ahead(taddr + c, g);
                    tc::ld16_ahead(taddr + kBN / 2 + c, u);
                    tc::wait_ld();
                    const int col = t.tn * (kBN / 2) + c;
                    if (row >= q.m || col >= q.n) continue;
                    if (p.gu) {
                        // kept as fp32: rounded to 16 bits they would add a third rounding to the gradients (error
                        // 0.0030 instead of 0.0024 of the norm in bf16)
                        store16_f32(p.gu + row * p.ld_gu + col, g);
                        store16_f32(p.gu + row * p.ld_gu + p.d_ff + col, u);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float gv = __uint_as_float(g[i]);
                        g[i] = __float_as_uint(gv * sigmoid(gv) * __uint_as_float(u[i]));
                    }
                    store16(q.out, row * q.ld_out + col, g, half);
                }
            } else {
#pragma unroll 1
                for (int c = side * (kBN / 4); c < (side + 1) * (kBN / 4); c += 16) {
                    const int col = t.tn * kBN + c;
                    const bool in = row < q.m && col < q.n;
                    uint32_t gw[16], uw[16], dh[16];
                    __syncwarp();
                    tc::ld16_ahead(taddr + c, dh);
                    if (in) {
                        const float *gp = p.gu + row * p.ld_gu + col, *up = gp + p.d_ff;
                        tc::load_v8(gp, gw);
                        tc::load_v8(gp + 8, gw + 8);
                        tc::load_v8(up, uw);
                        tc::load_v8(up + 8, uw + 8);
                    }
                    tc::wait_ld();
                    if (!in) continue;
                    uint32_t dg[8], du[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float o[2], v[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float g = __uint_as_float(gw[2 * i + j]), u = __uint_as_float(uw[2 * i + j]);
                            const float s = sigmoid(g), a = g * s, d = __uint_as_float(dh[2 * i + j]);
                            o[j] = d * u * (s + a * (1.f - s));
                            v[j] = d * a;
                        }
                        dg[i] = tc::pack16(o[0], o[1], half);
                        du[i] = tc::pack16(v[0], v[1], half);
                    }
                    tc::store_v8(reinterpret_cast<uint16_t *>(q.out) + row * q.ld_out + col, dg);
                    tc::store_v8(reinterpret_cast<uint16_t *>(q.out) + row * q.ld_out + p.d_ff + col, du);
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::arrive_relaxed(tc::cluster_addr(tc::smem_u32(&acc_empty[buf]), 0));
        }
    }

    // neither CTA may leave (or free tensor memory) while its peer can still read its shared memory or
    // signal its barriers
    __syncwarp();
    if (*abort_flag) tc::drain_after_abort();
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

struct Join {
    const float *partial;    // [splits][m][n]
    void *out;               // 16-bit [m][n]
    long long m, ld_out;
    int n, splits;
    unsigned first_block;
};
struct Joins { Join part[kMaxProblems]; int count, half; };

// out[m][n] = the parts of its reduction added in order, 8 columns a thread, for all cut products of a launch.  The parts
// are read past L1: the kernel may start before the one that writes them has ended.
__global__ void __launch_bounds__(256)
dense_reduce_kernel(const __grid_constant__ Joins joins) {
    tc::let_next();
    tc::after_previous();
    int p = 0;
    while (p + 1 < joins.count && blockIdx.x >= joins.part[p + 1].first_block) ++p;
    const Join &q = joins.part[p];
    const float *partial = q.partial;
    const long long m = q.m;
    const int n = q.n, splits = q.splits, half = joins.half;
    const long long total = m * (n / 8), at = (long long)(blockIdx.x - q.first_block) * 256 + threadIdx.x;
    if (at >= total) return;
    const long long row = at / (n / 8);
    const int col = (int)(at - row * (n / 8)) * 8;
    const float4 *src = reinterpret_cast<const float4 *>(partial + row * n + col);
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // eight parts' loads are in flight together; loads under a condition would wait for one another, so the last part
    // stands in for those that do not exist
    const long long step = m * n / 4;
    for (int s0 = 0; s0 < splits; s0 += 8) {
        float4 a[8], b[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const float4 *at_s = src + min(s0 + s, splits - 1) * step;
            a[s] = __ldcg(at_s);
            b[s] = __ldcg(at_s + 1);
        }
#pragma unroll
        for (int s = 0; s < 8; ++s)
            if (s0 + s < splits) {
                v[0] += a[s].x; v[1] += a[s].y; v[2] += a[s].z; v[3] += a[s].w;
                v[4] += b[s].x; v[5] += b[s].y; v[6] += b[s].z; v[7] += b[s].w;
            }
    }
    *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(q.out) + row * q.ld_out + col) =
        make_uint4(tc::pack16(v[0], v[1], half), tc::pack16(v[2], v[3], half), tc::pack16(v[4], v[5], half), tc::pack16(v[6], v[7], half));
}

bool misaligned(const void *p, size_t a = 16) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// Adds C[m][n] = sum_k A[m][k] B[n][k] to a launch.  `a` is [m][k] (row stride lda) or, with a_mn, [k][m];
// `b` is [n][k] or, with b_mn, [k][n].  For kSwiglu n counts hidden columns and b has 2 n rows.
int add_problem(DenseParams &p, int epi, int bn, const void *a, int64_t lda, bool a_mn, const void *b, int64_t ldb, bool b_mn,
                int64_t m, int64_t n, int64_t k, void *out, int64_t ld_out) {
    const int i = p.n_problems;
    Problem &q = p.prob[i];
    const int64_t b_rows = epi == kSwiglu ? 2 * n : n, tile_n = epi == kSwiglu ? bn / 2 : bn;
    int rc = a_mn ? tc::encode_bf16_2d(&p.map_a[i], a, m, k, lda, 64, 128)
                  : tc::encode_bf16_2d(&p.map_a[i], a, k, m, lda, 64, 128);
    if (rc != MORTAR_OK) return rc;
    rc = b_mn ? tc::encode_bf16_2d(&p.map_b[i], b, b_rows, k, ldb, 64, 128)
              : tc::encode_bf16_2d(&p.map_b[i], b, k, b_rows, ldb, 64, (uint32_t)(bn / 2));
    if (rc != MORTAR_OK) return rc;
    const int64_t tm = (m + 255) / 256, tn = (n + tile_n - 1) / tile_n;
    if (tm * tn + p.n_items > 0x3fffffff) return MORTAR_ERR_CAPACITY;
    q.out = out; q.ld_out = ld_out; q.m = m; q.n = (int)n;
    q.tiles_m = (int)tm; q.tiles_n = (int)tn; q.k_steps = (int)((k + 127) / 128);
    q.a_mn = a_mn; q.b_mn = b_mn; q.first_item = p.n_items; q.splits = 1;
    p.n_items += (int)(tm * tn);
    ++p.n_problems;
    return MORTAR_OK;
}

std::mutex g_dense_mutex;

int64_t steps_of(int64_t k) { return (k + 127) / 128; }
int64_t tiles_of(int64_t m, int64_t n, int bn) { return ((m + 255) / 256) * ((n + bn - 1) / bn); }

// Tiles of 128 columns where all of a launch's run at once, else of 256: half the tile takes half the time, but reads three
// quarters of the memory.  Forward and backward of 333 x 768/2048 29.0 + 39.2 -> 24.8 + 33.1 us, 2048 x 512/512 30.9 + 41.1
// -> 26.7 + 26.9; with 128 columns also where three rounds of them replace two of 256: 2048 x 768/1536 56.0 -> 58.8 backward,
// 4096 x 2048/1280 74.3 + 132.5 -> 81.8 + 157.3.
int width_of(int64_t tiles_256) { return 2 * tiles_256 <= kClusters ? 128 : 256; }

// The parts that a reduction of `k_steps` 128-wide steps is cut into, where a launch takes `total` steps over all its
// tiles: more than one where a tile would run for twice the even share of a cluster or longer (few rows, or few columns
// of a weight gradient), no more than leave all parts of the launch running at once, and no more than the longest part
// needs.
int64_t parts_of(int64_t k_steps, int64_t total) {
    const int64_t most = total < kClusters ? k_steps : k_steps * kClusters / total;
    if (most < 2) return 1;
    const int64_t longest = (k_steps + most - 1) / most;
    return (k_steps + longest - 1) / longest;
}

struct Plan { int bn; int64_t parts[kMaxProblems], floats; };

// of up to three products m x n over k in one launch
Plan plan(const int64_t (*mnk)[3], int count) {
    Plan r = {};
    int64_t total = 0, tiles = 0;
    for (int i = 0; i < count; ++i) tiles += tiles_of(mnk[i][0], mnk[i][1], 256);
    r.bn = width_of(tiles);
    for (int i = 0; i < count; ++i) total += tiles_of(mnk[i][0], mnk[i][1], r.bn) * steps_of(mnk[i][2]);
    for (int i = 0; i < count; ++i) {
        r.parts[i] = parts_of(steps_of(mnk[i][2]), total);
        if (r.parts[i] > 1) r.floats += r.parts[i] * mnk[i][0] * mnk[i][1];
    }
    return r;
}

// Deals the scratch out to the products that are cut, and renumbers the items.
void cut(DenseParams &p, const Plan &plan, float *scratch) {
    p.n_items = 0;
    for (int i = 0; i < p.n_problems; ++i) {
        Problem &q = p.prob[i];
        q.splits = (int)plan.parts[i];
        q.partial = scratch;
        if (q.splits > 1) scratch += plan.parts[i] * q.m * q.n;
        q.first_item = p.n_items;
        p.n_items += q.tiles_m * q.tiles_n * q.splits;
    }
}

int join(const DenseParams &p, cudaStream_t st) {
    Joins j = {};
    int64_t blocks = 0;
    for (int i = 0; i < p.n_problems; ++i) {
        const Problem &q = p.prob[i];
        if (q.splits == 1) continue;
        j.part[j.count++] = {q.partial, q.out, q.m, q.ld_out, q.n, q.splits, (unsigned)blocks};
        blocks += (q.m * (q.n / 8) + 255) / 256;
    }
    if (j.count == 0) return MORTAR_OK;
    if (blocks > 0x7fffffffLL) return MORTAR_ERR_CAPACITY;
    j.half = p.half;
    return tc::launch_after(dense_reduce_kernel, (unsigned)blocks, 256u, 0, st, j);
}

template <int EPI, int BN>
int launch_width(const DenseParams &p, bool follows, cudaStream_t st) {
    static bool ready[64] = {false};
    constexpr int kSmem = Shape<BN>::kSmem;
    int sms = 0;
    int rc = tc::allow_smem(dense_pair_kernel<EPI, BN>, kSmem, ready, g_dense_mutex, nullptr);
    if (rc != MORTAR_OK) return rc;
    rc = tc::sm_count(&sms);
    if (rc != MORTAR_OK) return rc;
    const int clusters = p.n_items < sms / 2 ? p.n_items : sms / 2;
    if (follows) return tc::launch_after(dense_pair_kernel<EPI, BN>, (unsigned)(2 * clusters), (unsigned)kThreads, kSmem, st, p);
    dense_pair_kernel<EPI, BN><<<(unsigned)(2 * clusters), kThreads, kSmem, st>>>(p);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

// `follows`: the launch reads what the one before it in the call wrote, and may be set up while that one ends
template <int EPI>
int launch(const DenseParams &p, int bn, bool follows, cudaStream_t st) {
    return bn == 128 ? launch_width<EPI, 128>(p, follows, st) : launch_width<EPI, 256>(p, follows, st);
}

int check_shape(int32_t dtype, int64_t rows, int32_t d_model, int32_t d_ff) {
    if (rows < 0 || d_model <= 0 || d_ff <= 0 || d_model % 16 || d_ff % 16) return MORTAR_ERR_SHAPE;
    if (rows > 0x7fffff00LL || d_ff > (1 << 29) || d_model > (1 << 29)) return MORTAR_ERR_CAPACITY;
    if (dtype != MORTAR_BF16 && dtype != MORTAR_F16) return MORTAR_ERR_DTYPE;
    return MORTAR_OK;
}

}  // namespace

// products of the backward pass's last launch: dgate_up, dx, ddown
static Plan backward_plan(int64_t rows, int32_t d_model, int32_t d_ff, bool dgu, bool dx, bool ddn) {
    int64_t mnk[3][3];
    int n = 0;
    if (dx) { mnk[n][0] = rows; mnk[n][1] = d_model; mnk[n++][2] = 2LL * d_ff; }
    if (dgu) { mnk[n][0] = 2LL * d_ff; mnk[n][1] = d_model; mnk[n++][2] = rows; }
    if (ddn) { mnk[n][0] = d_model; mnk[n][1] = d_ff; mnk[n++][2] = rows; }
    return plan(mnk, n);
}

static Plan forward_plan(int64_t rows, int32_t d_model, int32_t d_ff) {
    const int64_t mnk[1][3] = {{rows, d_model, d_ff}};
    return plan(mnk, 1);
}

extern "C" int64_t mortar_mlp_dense_scratch_floats(int64_t rows, int32_t d_model, int32_t d_ff, int32_t keep_sums) {
    const int rc = check_shape(MORTAR_BF16, rows, d_model, d_ff);
    if (rc == MORTAR_OK && rows <= small::kMaxRows && !keep_sums) return 0;
    return rc != MORTAR_OK ? rc : forward_plan(rows, d_model, d_ff).floats;
}

extern "C" int64_t mortar_mlp_dense_backward_scratch_floats(int64_t rows, int32_t d_model, int32_t d_ff, int32_t want_dx,
                                                            int32_t want_dgate_up, int32_t want_ddown) {
    const int rc = check_shape(MORTAR_BF16, rows, d_model, d_ff);
    return rc != MORTAR_OK ? rc : backward_plan(rows, d_model, d_ff, want_dgate_up != 0, want_dx != 0, want_ddown != 0).floats;
}

extern "C" int mortar_mlp_dense(const void *x, int64_t ldx, int32_t dtype, int64_t rows, const void *gate_up,
                                int64_t ld_gate_up, const void *down, int64_t ld_down, int32_t d_model, int32_t d_ff,
                                void *hidden, float *gate_up_sums, void *y, int64_t ldy, float *scratch, int64_t scratch_floats,
                                void *stream) {
    if (!x || !gate_up || !down || !hidden || !y) return MORTAR_ERR_NULL;
    int rc = check_shape(dtype, rows, d_model, d_ff);
    if (rc != MORTAR_OK) return rc;
    if (ldx < d_model || ld_gate_up < d_model || ld_down < d_ff || ldy < d_model) return MORTAR_ERR_SHAPE;
    if (misaligned(x) || misaligned(gate_up) || misaligned(down) || misaligned(hidden, 32) || misaligned(gate_up_sums, 32) ||
        misaligned(y, 32) || misaligned(scratch, 32) || ldx % 8 || ld_gate_up % 8 || ld_down % 8 || ldy % 16)
        return MORTAR_ERR_ALIGN;
    if (rows == 0) return MORTAR_OK;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows <= small::kMaxRows && !gate_up_sums) {
        int sms = 0;
        rc = tc::sm_count(&sms);
        if (rc != MORTAR_OK) return rc;
        small::Params q = {};
        q.x = (const uint8_t *)x; q.ldx = 2 * ldx; q.w = (const uint8_t *)gate_up; q.ldw = 2 * ld_gate_up;
        q.rows = (int)rows; q.n = d_ff; q.up_row = d_ff; q.k_bytes = 2 * d_model;
        q.out = hidden; q.ld_out = d_ff; q.out_dtype = q.x_dtype = q.w_dtype = dtype;
        rc = small::launch(q, sms, st);
        if (rc != MORTAR_OK) return rc;
        q.x = (const uint8_t *)hidden; q.ldx = 2LL * d_ff; q.w = (const uint8_t *)down; q.ldw = 2 * ld_down;
        q.n = d_model; q.up_row = 0; q.k_bytes = 2 * d_ff;
        q.out = y; q.ld_out = ldy; q.after_previous = 1;
        return small::launch(q, sms, st);
    }
    const Plan parts = forward_plan(rows, d_model, d_ff);
    if (parts.floats > 0 && (!scratch || scratch_floats < parts.floats)) return MORTAR_ERR_CAPACITY;
    rc = tc::bind_context();
    if (rc != MORTAR_OK) return rc;
    alignas(64) DenseParams p = {};
    p.half = dtype == MORTAR_F16;
    p.d_ff = d_ff;
    p.gu = gate_up_sums;
    p.ld_gu = 2LL * d_ff;
    const int bn = width_of(tiles_of(rows, 2LL * d_ff, 256));
    rc = add_problem(p, kSwiglu, bn, x, ldx, false, gate_up, ld_gate_up, false, rows, d_ff, d_model, hidden, d_ff);
    if (rc == MORTAR_OK) rc = launch<kSwiglu>(p, bn, false, st);
    if (rc != MORTAR_OK) return rc;
    alignas(64) DenseParams p2 = {};
    p2.half = p.half;
    rc = add_problem(p2, kStore, parts.bn, hidden, d_ff, false, down, ld_down, false, rows, d_model, d_ff, y, ldy);
    if (rc != MORTAR_OK) return rc;
    cut(p2, parts, scratch);
    rc = launch<kStore>(p2, parts.bn, true, st);
    return rc == MORTAR_OK ? join(p2, st) : rc;
}

extern "C" int mortar_mlp_dense_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int32_t dtype,
                                         int64_t rows, const void *gate_up, int64_t ld_gate_up, const void *down,
                                         int64_t ld_down, int32_t d_model, int32_t d_ff, const void *hidden,
                                         const float *gate_up_sums, void *dgate_up_sums, void *dx, void *dgate_up,
                                         void *ddown, float *scratch, int64_t scratch_floats, void *stream) {
    if (!dy || !x || !gate_up || !down || !hidden || !gate_up_sums || !dgate_up_sums) return MORTAR_ERR_NULL;
    int rc = check_shape(dtype, rows, d_model, d_ff);
    if (rc != MORTAR_OK) return rc;
    if (lddy < d_model || ldx < d_model || ld_gate_up < d_model || ld_down < d_ff) return MORTAR_ERR_SHAPE;
    if (misaligned(dy) || misaligned(x) || misaligned(gate_up) || misaligned(down) || misaligned(hidden, 32) ||
        misaligned(gate_up_sums, 32) || misaligned(dgate_up_sums, 32) || misaligned(dx, 32) || misaligned(dgate_up, 32) ||
        misaligned(ddown, 32) || misaligned(scratch, 32) || lddy % 8 || ldx % 8 || ld_gate_up % 8 || ld_down % 8)
        return MORTAR_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {
        if (dgate_up) MORTAR_CUDA_CHECK(cudaMemsetAsync(dgate_up, 0, (size_t)4 * d_ff * d_model, st));
        if (ddown) MORTAR_CUDA_CHECK(cudaMemsetAsync(ddown, 0, (size_t)2 * d_ff * d_model, st));
        return MORTAR_OK;
    }
    const Plan parts = backward_plan(rows, d_model, d_ff, dgate_up != nullptr, dx != nullptr, ddown != nullptr);
    if (parts.floats > 0 && (!scratch || scratch_floats < parts.floats)) return MORTAR_ERR_CAPACITY;
    rc = tc::bind_context();
    if (rc != MORTAR_OK) return rc;
    const int64_t f2 = 2LL * d_ff;
    if (dx || dgate_up) {
        alignas(64) DenseParams p = {};
        p.half = dtype == MORTAR_F16;
        p.d_ff = d_ff;
        p.gu = const_cast<float *>(gate_up_sums);
        p.ld_gu = f2;
        const int bn = width_of(tiles_of(rows, d_ff, 256));
        rc = add_problem(p, kSwigluBackward, bn, dy, lddy, false, down, ld_down, true, rows, d_ff, d_model, dgate_up_sums, f2);
        if (rc == MORTAR_OK) rc = launch<kSwigluBackward>(p, bn, false, st);
        if (rc != MORTAR_OK) return rc;
    }
    alignas(64) DenseParams p = {};
    p.half = dtype == MORTAR_F16;
    // the longest reduction first
    if (dx) rc = add_problem(p, kStore, parts.bn, dgate_up_sums, f2, false, gate_up, ld_gate_up, true, rows, d_model, f2, dx, d_model);
    if (rc == MORTAR_OK && dgate_up)
        rc = add_problem(p, kStore, parts.bn, dgate_up_sums, f2, true, x, ldx, true, f2, d_model, rows, dgate_up, d_model);
    if (rc == MORTAR_OK && ddown)
        rc = add_problem(p, kStore, parts.bn, dy, lddy, true, hidden, d_ff, true, d_model, d_ff, rows, ddown, d_ff);
    if (rc != MORTAR_OK || p.n_problems == 0) return rc;
    cut(p, parts, scratch);
    rc = launch<kStore>(p, parts.bn, dx || dgate_up, st);
    return rc == MORTAR_OK ? join(p, st) : rc;
}

extern "C" int mortar_dense_error(int32_t *code, int32_t reset) {
    if (!code) return MORTAR_ERR_NULL;
    int v = 0;
    MORTAR_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_dense_error, sizeof(int)));
    *code = v;
    if (reset && v != 0) {
        const int zero = 0;
        MORTAR_CUDA_CHECK(cudaMemcpyToSymbol(g_dense_error, &zero, sizeof(int)));
    }
    return MORTAR_OK;
}
