// Matrix product of two 8-bit floating-point operands with one scale per block of 128, on the
// 5th-generation tensor cores:
//
//   y[m][n] = sum over blocks b of sx[m][b] * sw[n / 128][b] * sum_{k in block b} qx[m][k] qw[n][k]
//
// (activations scaled per 1 x 128, weights per 128 x 128), and with the gate applied,
// y = silu(y[:, :n/2]) * y[:, n/2:].
//
// The scales are any fp32 numbers, so a block's sum has to leave the accumulator before the next
// block's begins: one pipeline stage is one block (128 bytes of k, a swizzle row), its four MMAs
// (kind::f8f6f4, K = 32) write one of two accumulator sets, and the epilogue warps read the set,
// multiply by sx * sw (one factor per thread and 128 columns) and add it to fp32 sums in registers
// while the MMAs fill the other set.  A cluster of two CTAs computes 256 x 256: every thread of eight
// epilogue warps keeps 128 sums, for which the launch's registers are dealt out anew.
//
// What bounds it, at 8192 x 2048 -> 11264 with the gate (206 to 220 us, 1720 to 1830 TFLOP/s, 233 to 248 in
// a long run under the power cap): the epilogue warps.
// The same MMAs and copies with one sum per tile instead of one per block take 139 us.  A block's MMAs are
// 512 cycles; a warp needs about 800 for it: 150 to see that the block is there, twice 75 to read 64 columns
// and 150 to multiply and add them (3 cycles a packed multiply-add), 75 to hand the set back, the rest to
// walk on; and 4700 a tile for the gate and the stores (193 us without the gate).  Tried without gain: four sets of 128 columns (279
// us), reading 32 columns ahead (238), asking for the next block before the multiply-adds (the register it
// takes costs more than it hides), arrivals with release at cluster scope (630: they wait for the stores).
#include <cuda.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <cstdint>
#include <mutex>
#include <type_traits>
#include "common.h"
#include "dense_small.cuh"
#include "tc_pair.cuh"

namespace {

constexpr int kStages = 6;
constexpr int kStageA = 128 * 128;               // this CTA's 128 rows, one block of 128 bytes each
constexpr int kStageB = 128 * 128;               // this CTA's half of the 256 output columns
constexpr int kStage = kStageA + kStageB;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;   // warps 0..3: copies, MMAs, two that only lend their registers
constexpr int kTmemCols = 512;
constexpr int kTurn = 32 * 33;                   // floats a warp turns a 32 x 32 piece of the result in
constexpr int kSmem = kStages * kStage + (2 * kStages + 2) * 8 + kEpiWarps * kTurn * 4 + 1024;
static_assert(kSmem + 64 <= 227 * 1024, "shared memory budget");

__device__ int g_fp8_error;

struct Fp8Params {
    CUtensorMap map_x, map_w, map_w_half;      // boxes of 128, 128 and 64 rows
    const float *xs, *ws;
    long long ld_xs, ld_ws;
    long long rows;
    int n;                   // output columns (hidden columns with the gate)
    int tiles_m, tiles_n;
    int whole, n_items;      // items: the first `whole` tiles, then the others' left and right halves
    int k_blocks;
    int parts;               // of the reduction, an item each (all tiles are halves then); more than one: `out` holds fp32
    long long part_step;     // [parts][rows][ld_out], `part_step` elements from part to part
    int up_row;              // 0, or the first up row of w (gate applied)
    int w_blocks;            // rows of ws
    uint32_t types;          // operand type bits of the instruction descriptor
    void *out;
    long long ld_out;
    int out_dtype;
};

__device__ __forceinline__ float exp2_of(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float inverse_of(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

// silu(g) u of two columns, from the approximate power and inverse: off by 2^-22 (1 + |g|) of the result at worst.  A
// tile's 16384 a CTA keep the special function unit busy for 2000 of 19000 cycles; with __expf and __fdividef, which
// handle more than is needed here, the product of the header took 216 where it takes 206 us, with expf and a division 631.
__device__ __forceinline__ uint64_t gated(uint64_t g, uint64_t u) {
    const uint64_t t = tc::mul2(g, tc::both(-1.4426950408889634f));       // exp(-g) = 2^t
    const uint64_t d = tc::add2(tc::pair_of(__float_as_uint(exp2_of(tc::low_of(t))), __float_as_uint(exp2_of(tc::high_of(t)))),
                                tc::both(1.f));
    const uint64_t r = tc::pair_of(__float_as_uint(inverse_of(tc::low_of(d))), __float_as_uint(inverse_of(tc::high_of(d))));
    return tc::mul2(tc::mul2(g, r), u);
}

// A warp's 32 rows x 32 columns from (row0, col) on; v = this lane's row.  Rows that start on 32 bytes and end on a
// multiple of 32 columns are stored 32 bytes at a time, each lane its own.  Others (TURNED) are turned in shared memory, so that the lanes of a store lie side by side
// in a row (stored value by value from each lane's own row, a ragged tile took three times as long).
template <bool TURNED>
__device__ __forceinline__ void store_32x32(const Fp8Params &p, void *out, long long row0, int col, const float (&v)[32], float *turn) {
    const int left = p.n - col, lane = threadIdx.x & 31;
    if (left <= 0) return;
    const long long row = row0 + lane;
    if constexpr (!TURNED) {
        if (row >= p.rows) return;
        if (p.out_dtype == MORTAR_F32) {
            float *o = reinterpret_cast<float *>(out) + row * p.ld_out + col;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[8 * j + i]);
                tc::store_v8(o + 8 * j, w);
            }
            return;
        }
        uint16_t *o = reinterpret_cast<uint16_t *>(out) + row * p.ld_out + col;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = tc::pack16(v[16 * j + 2 * i], v[16 * j + 2 * i + 1], p.out_dtype == MORTAR_F16);
            tc::store_v8(o + 16 * j, w);
        }
        return;
    } else {
    __syncwarp();                                                     // the piece before has been read
#pragma unroll
    for (int i = 0; i < 32; ++i) turn[lane * 33 + i] = v[i];
    __syncwarp();
    if (lane >= left) return;
    const int rows = (int)min(32LL, p.rows - row0);
    const long long idx = row0 * p.ld_out + col + lane;
    if (p.out_dtype == MORTAR_F32) {
        float *o = reinterpret_cast<float *>(out) + idx;
        for (int r = 0; r < rows; ++r) o[r * p.ld_out] = turn[r * 33 + lane];
    } else {
        uint16_t *o = reinterpret_cast<uint16_t *>(out) + idx;
        for (int r = 0; r < rows; ++r) o[r * p.ld_out] = (uint16_t)tc::pack16(turn[r * 33 + lane], 0.f, p.out_dtype == MORTAR_F16);
    }
    }
}

__device__ __forceinline__ void tile_at(const Fp8Params &p, int i, int &tm, int &tn) {
    const int band = i / (8 * p.tiles_n), r = i - band * 8 * p.tiles_n;
    const int h = min(8, p.tiles_m - band * 8);
    tn = r / h;
    tm = band * 8 + r - tn * h;
}
// What a launch cuts: nothing, the tiles of its last round in two, or (all tiles being halves) their reductions too.
enum Cut { kWhole = 0, kHalves = 1, kParts = 2 };
// The tile of an item of halves; returns which half of its columns.
template <int CUT>
__device__ __forceinline__ int half_at(const Fp8Params &p, int item, int &tm, int &tn) {
    const int over = CUT == kParts ? item / p.parts : item - p.whole;
    tile_at(p, CUT == kParts ? over >> 1 : p.whole + (over >> 1), tm, tn);
    return over & 1;
}
// The blocks of an item: all, or its part of them.
template <int CUT> __device__ __forceinline__ int first_block(const Fp8Params &p, int item) {
    return CUT == kParts ? (int)((long long)p.k_blocks * (item % p.parts) / p.parts) : 0;
}
template <int CUT> __device__ __forceinline__ int end_block(const Fp8Params &p, int item) {
    return CUT == kParts ? (int)((long long)p.k_blocks * (item % p.parts + 1) / p.parts) : p.k_blocks;
}

template <bool TURNED, int CUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
fp8_pair_kernel(const __grid_constant__ Fp8Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    // full: a stage's copies have landed (CTA 0's count for both); done: its MMAs have ended, so the stage is free and
    // its sums are there; acc_empty (CTA 0's): the warps of both have read the sums
    uint64_t *full = reinterpret_cast<uint64_t *>(stages + kStages * kStage), *done = full + kStages;
    uint64_t *acc_empty = done + kStages;
    float *turns = reinterpret_cast<float *>(acc_empty + 2);
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < kStages; ++s) { tc::mbar_init(tc::smem_u32(&full[s]), 1); tc::mbar_init(tc::smem_u32(&done[s]), 1); }
        for (int s = 0; s < 2; ++s) tc::mbar_init(tc::smem_u32(&acc_empty[s]), 2 * kEpiWarps);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(tc::smem_u32(&tmem_base_s)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::fence_after();
    if constexpr (CUT == kParts) tc::let_next();
    const uint32_t tmem = tmem_base_s;
    volatile int *abort_flag = &abort_s;

    // 384 threads start with 168 registers each; before any of them waits for another they are dealt
    // out anew: 128 * 64 + 256 * 216 <= 384 * 168
    if (warp < 4) {
        tc::registers_down<64>();
        if (warp == 0 && lane == 0) {
            const uint32_t full_lead = tc::cluster_addr(tc::smem_u32(full), 0);
            const uint32_t done0 = tc::smem_u32(done), stage0 = tc::smem_u32(stages);
            uint32_t s = 0, parity = 1;
            bool ok = true;
            for (int item = cluster_id; item < p.n_items && ok; item += n_clusters) {
                int tm, tn;
                int part = -1;
                if (CUT == kWhole || (CUT == kHalves && item < p.whole)) tile_at(p, item, tm, tn);
                else part = half_at<CUT>(p, item, tm, tn);
                const int end = end_block<CUT>(p, item);
                const int row0 = tm * 256 + (int)rank * 128;
                const int wide = part < 0 ? 128 : 64;                 // this CTA's columns
                const int col0 = (p.up_row ? tn * 128 + (rank ? p.up_row : 0) + (part > 0 ? 64 : 0)
                                           : tn * 256 + (part > 0 ? 128 : 0) + (int)rank * wide);
                for (int k = first_block<CUT>(p, item); k < end; ++k) {
                    if (!tc::mbar_wait(done0 + 8 * s, parity, abort_flag, &g_fp8_error, 1)) { ok = false; break; }
                    const uint32_t bar = full_lead + 8 * s, dst = stage0 + s * kStage;
                    if (rank == 0) tc::mbar_arrive_expect_tx(tc::smem_u32(&full[s]), 2 * (kStageA + wide * 128));
                    tc::load_pair(dst, &p.map_x, k * 128, row0, bar);
                    tc::load_pair(dst + kStageA, part < 0 ? &p.map_w : &p.map_w_half, k * 128, col0, bar);
                    if (++s == kStages) { s = 0; parity ^= 1; }
                }
            }
        } else if (warp == 1 && rank == 0 && lane == 0) {
            const uint32_t idesc_256 = (1u << 4) | p.types | ((256u >> 3) << 17) | ((256u >> 4) << 24);
            const uint32_t idesc_128 = idesc_256 - ((128u >> 3) << 17);
            const uint32_t full0 = tc::smem_u32(full), done0 = tc::smem_u32(done), acc_empty0 = tc::smem_u32(acc_empty);
            const uint64_t da = tc::make_smem_desc(tc::smem_u32(stages), 16, 1024, 2);
            const uint64_t db = tc::make_smem_desc(tc::smem_u32(stages) + kStageA, 16, 1024, 2);
            uint32_t s = 0, parity = 0, g = 0;
            bool ok = true, ready = tc::mbar_try_wait(full0, 0);
            for (int item = cluster_id; item < p.n_items && ok; item += n_clusters) {
                const uint32_t idesc = CUT == kWhole || (CUT == kHalves && item < p.whole) ? idesc_256 : idesc_128;
                const int blocks = end_block<CUT>(p, item) - first_block<CUT>(p, item);
                for (int k = 0; k < blocks; ++k, ++g) {
                    const uint32_t buf = g & 1;
                    if ((!ready && !tc::mbar_wait(full0 + 8 * s, parity, abort_flag, &g_fp8_error, 3)) ||
                        !tc::mbar_wait(acc_empty0 + 8 * buf, ((g >> 1) & 1) ^ 1u, abort_flag, &g_fp8_error, 2)) { ok = false; break; }
                    tc::fence_after();
                    const uint64_t at = (uint64_t)(s * (kStage >> 4));
                    const uint32_t bar = done0 + 8 * s;
                    if (++s == kStages) { s = 0; parity ^= 1; }
                    ready = tc::poll_mma4_f8(full0 + 8 * s, parity, tmem + buf * 256, da + at, db + at, idesc);
                    tc::commit_both(bar);
                }
            }
        }
    } else {
        tc::registers_up<216>();
        // warp w: accumulator lanes 32 (w % 4) .. +31, columns 64 side .. +63 of either 128-column half (of a
        // half tile 32 side .. +31 of either 64-column half), so that a thread holds the gate and the up sum
        // of its hidden columns
        const int quarter = warp & 3, side = (warp - 4) >> 2;
        const uint32_t done0 = tc::smem_u32(done), lead_empty = tc::cluster_addr(tc::smem_u32(acc_empty), 0);
        const uint32_t taddr0 = tmem + ((uint32_t)(quarter * 32) << 16) + side * 64;
        uint32_t g = 0, s = 0, parity = 0;
        // HALF: a thread holds 32 columns of either half of the tile instead of 64
        auto finish = [&](int item, auto half) -> bool {
            constexpr bool HALF = decltype(half)::value;
            constexpr int kPer = HALF ? 1 : 2;                    // pieces of 32 columns in either half
            // positions in the scale arrays: 32 bits, and the tile's place is worked out again for the stores, since the sums
            // and what is being read leave few registers (229 -> 213 us)
            uint32_t at_x, at_w0, at_w1;
            {
                int tm, tn;
                int part = 0;
                if constexpr (HALF) part = half_at<CUT>(p, item, tm, tn);
                else tile_at(p, item, tm, tn);
                const long long row = (long long)tm * 256 + (long long)rank * 128 + quarter * 32 + lane;
                const int wb0 = p.up_row ? tn : HALF ? min(2 * tn + part, p.w_blocks - 1) : 2 * tn;
                const int wb1 = p.up_row ? p.up_row / 128 + tn : HALF ? wb0 : 2 * tn + 1;
                at_x = (uint32_t)((row < p.rows ? row : p.rows - 1) * p.ld_xs);
                at_w0 = (uint32_t)(wb0 * p.ld_ws);
                at_w1 = (uint32_t)(min(wb1, p.w_blocks - 1) * p.ld_ws);
                if constexpr (CUT == kParts) {
                    const uint32_t first = (uint32_t)first_block<CUT>(p, item);
                    at_x += first; at_w0 += first; at_w1 += first;
                }
            }
            uint64_t sum[2 * kPer][16];                           // columns 32 j + 2 i, + 1
#pragma unroll
            for (int j = 0; j < 2 * kPer; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[j][i] = 0ull;
            float sx = __ldg(p.xs + at_x), s0 = __ldg(p.ws + at_w0), s1 = __ldg(p.ws + at_w1);
            for (int k = end_block<CUT>(p, item) - first_block<CUT>(p, item); k > 0; --k, ++g) {
                const uint32_t buf = g & 1, taddr = taddr0 + buf * 256 - (HALF ? side * 32 : 0);
                const float f0 = sx * s0, f1 = sx * s1;
                if (k > 1) { sx = __ldg(p.xs + ++at_x); s0 = __ldg(p.ws + ++at_w0); s1 = __ldg(p.ws + ++at_w1); }
                if (!tc::mbar_wait(done0 + 8 * s, parity, abort_flag, &g_fp8_error, 4)) return false;
                if (++s == kStages) { s = 0; parity ^= 1; }
                __syncwarp();
                tc::fence_after();
#pragma unroll
                for (int h = 0; h < kPer; ++h) {                  // 64 columns at once
                    uint32_t r[2][32];
                    tc::ld32(taddr + h * 128, r[0]);
                    tc::ld32(taddr + h * 128 + (HALF ? 64 : 32), r[1]);
                    tc::wait_ld();
                    if (h == kPer - 1) {
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) tc::arrive_relaxed(lead_empty + 8 * buf);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint64_t ff = tc::both((HALF ? j : h) ? f1 : f0);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            sum[2 * h + j][i] = tc::fma2(tc::pair_of(r[j][2 * i], r[j][2 * i + 1]), ff, sum[2 * h + j][i]);
                    }
                }
            }
            int tm, tn;
            int part = 0;
            if constexpr (HALF) part = half_at<CUT>(p, item, tm, tn);
            else tile_at(p, item, tm, tn);
            void *out = p.out;
            if constexpr (CUT == kParts) out = reinterpret_cast<float *>(p.out) + item % p.parts * p.part_step;
            const long long row0 = (long long)tm * 256 + (long long)rank * 128 + quarter * 32;
#pragma unroll
            for (int j = 0; j < 2 * kPer; ++j) {
                if (j >= kPer && p.up_row) break;
                float v[32];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint64_t y = p.up_row ? gated(sum[j][i], sum[(j + kPer) % (2 * kPer)][i]) : sum[j][i];
                    v[2 * i] = tc::low_of(y);
                    v[2 * i + 1] = tc::high_of(y);
                }
                int col;
                if constexpr (HALF) col = p.up_row ? tn * 128 + part * 64 + side * 32 : tn * 256 + part * 128 + j * 64 + side * 32;
                else col = p.up_row ? tn * 128 + side * 64 + j * 32 : tn * 256 + (j >> 1) * 128 + side * 64 + (j & 1) * 32;
                store_32x32<TURNED>(p, out, row0, col, v, turns + (warp - 4) * kTurn);
            }
            return true;
        };
        int item = cluster_id;
        bool ok = true;
        if constexpr (CUT != kParts)
            for (; ok && item < p.whole; item += n_clusters) ok = finish(item, std::false_type());
        if constexpr (CUT != kWhole) {                            // one round at most
            if (ok && item < p.n_items) finish(item, std::true_type());
        }
    }

    __syncwarp();
    if (*abort_flag) tc::drain_after_abort();
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// out = the parts of a reduction, fp32 [parts][rows][ld], added in order; four columns a thread.  They are read past L1:
// the kernel may start before the one that writes them has ended.
__global__ void __launch_bounds__(256)
fp8_join_kernel(const float *partial, int parts, long long part_step, long long ld, long long rows, int n, void *out,
                long long ld_out, int out_dtype) {
    tc::after_previous();
    const long long quads = ld / 4, at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= rows * quads) return;
    const long long row = at / quads;
    const int col = (int)(at - row * quads) * 4;
    const float *src = partial + row * ld + col;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < parts; i0 += 4) {
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __ldcg(reinterpret_cast<const float4 *>(src + min(i0 + i, parts - 1) * part_step));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i0 + i < parts) { s.x += v[i].x; s.y += v[i].y; s.z += v[i].z; s.w += v[i].w; }
    }
    const float r[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (col + i >= n) continue;
        const long long idx = row * ld_out + col + i;
        if (out_dtype == MORTAR_F32) reinterpret_cast<float *>(out)[idx] = r[i];
        else reinterpret_cast<uint16_t *>(out)[idx] = (uint16_t)tc::pack16(r[i], 0.f, out_dtype == MORTAR_F16);
    }
}

// ---- up to 32 rows: the operands change places -------------------------------------------------
//
// With a few tokens most of a 256 x 256 tile's rows do not exist, but its epilogue takes as long.  Here the weights are
// the 256 rows of a tile and 32 tokens its columns: a thread holds 16 sums of one output column, and the tokens'
// scales come from a table in shared memory.  With the gate, a CTA's 128 rows are groups of 16 gate rows and the 16 up rows
// of the same hidden columns, so that lanes l and l + 16 of a warp hold the two sums of an output and exchange them at
// the end.
//
// 32 x 2048 -> 11264 with the gate 13.1 us (L2 flushed 17.3) against 16.6 (21.5) on the tiles above, 32 x 768 -> 4096 9.0
// against 10.4: a block's way from copy to sums.  With 64 or 128 tokens reading the table for
// every block takes longer than the larger tile's epilogue (64 x 2048 -> 11264 14.6 against 16.6, 64 x 5632 -> 2048
// 28.9 against 24.8; 128 rows 20.7 and 38.6 against 16.6 and 25.8); four accumulator sets instead of two changed nothing.
constexpr int kFewRows = 32;
constexpr int kFewStages = 6;
constexpr int kFewB = kFewRows / 2 * 128;                        // this CTA's half of the tokens, one block
constexpr int kFewStage = kStageA + kFewB;
constexpr int kFewFixed = kFewStages * kFewStage + (2 * kFewStages + 2) * 8 + 1024;
constexpr int kFewBlocks = (226 * 1024 - kFewFixed) / (4 * kFewRows);      // that the table has room for
constexpr int few_smem(int k_blocks) { return kFewFixed + 4 * kFewRows * k_blocks; }

__device__ __forceinline__ void store_one(const Fp8Params &p, int m, int col, float v) {
    if (m >= p.rows || col >= p.n) return;
    const long long idx = m * p.ld_out + col;
    if (p.out_dtype == MORTAR_F32) reinterpret_cast<float *>(p.out)[idx] = v;
    else reinterpret_cast<uint16_t *>(p.out)[idx] = (uint16_t)tc::pack16(v, 0.f, p.out_dtype == MORTAR_F16);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
fp8_few_kernel(const __grid_constant__ Fp8Params p) {
    constexpr int kHeld = kFewRows / 2;                             // sums of a thread
    extern __shared__ uint8_t smem_raw[];
    uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(stages + kFewStages * kFewStage), *done = full + kFewStages;
    uint64_t *acc_empty = done + kFewStages;
    float *table = reinterpret_cast<float *>(acc_empty + 2);     // [block][token]
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < kFewStages; ++s) { tc::mbar_init(tc::smem_u32(&full[s]), 1); tc::mbar_init(tc::smem_u32(&done[s]), 1); }
        for (int s = 0; s < 2; ++s) tc::mbar_init(tc::smem_u32(&acc_empty[s]), 2 * kEpiWarps);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                     ::"r"(tc::smem_u32(&tmem_base_s)), "r"(2 * kFewRows) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = tmem_base_s;
    volatile int *abort_flag = &abort_s;

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t full_lead = tc::cluster_addr(tc::smem_u32(full), 0);
            const uint32_t done0 = tc::smem_u32(done), stage0 = tc::smem_u32(stages);
            uint32_t s = 0, parity = 1;
            bool ok = true;
            for (int tile = cluster_id; tile < p.n_items && ok; tile += n_clusters)
                for (int k = 0; k < p.k_blocks; ++k) {
                    if (!tc::mbar_wait(done0 + 8 * s, parity, abort_flag, &g_fp8_error, 1)) { ok = false; break; }
                    const uint32_t bar = full_lead + 8 * s, dst = stage0 + s * kFewStage;
                    if (rank == 0) tc::mbar_arrive_expect_tx(tc::smem_u32(&full[s]), 2 * kFewStage);
                    if (p.up_row) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            tc::load_pair_3d(dst + 4096 * i, &p.map_w, k * 128, tile * 128 + (int)rank * 64 + 16 * i, 0, bar);
                    } else {
                        tc::load_pair(dst, &p.map_w, k * 128, tile * 256 + (int)rank * 128, bar);
                    }
                    tc::load_pair(dst + kStageA, &p.map_x, k * 128, (int)rank * kHeld, bar);
                    if (++s == kFewStages) { s = 0; parity ^= 1; }
                }
        }
    } else if (warp == 1) {
        if (rank == 0 && lane == 0) {
            const uint32_t idesc = (1u << 4) | p.types | ((uint32_t)(kFewRows >> 3) << 17) | ((256u >> 4) << 24);
            const uint32_t full0 = tc::smem_u32(full), done0 = tc::smem_u32(done), acc_empty0 = tc::smem_u32(acc_empty);
            const uint64_t da = tc::make_smem_desc(tc::smem_u32(stages), 16, 1024, 2);
            const uint64_t db = tc::make_smem_desc(tc::smem_u32(stages) + kStageA, 16, 1024, 2);
            uint32_t s = 0, parity = 0, g = 0;
            bool ok = true, ready = tc::mbar_try_wait(full0, 0);
            for (int tile = cluster_id; tile < p.n_items && ok; tile += n_clusters)
                for (int k = 0; k < p.k_blocks; ++k, ++g) {
                    const uint32_t buf = g & 1;
                    if ((!ready && !tc::mbar_wait(full0 + 8 * s, parity, abort_flag, &g_fp8_error, 3)) ||
                        !tc::mbar_wait(acc_empty0 + 8 * buf, ((g >> 1) & 1) ^ 1u, abort_flag, &g_fp8_error, 2)) { ok = false; break; }
                    tc::fence_after();
                    const uint64_t at = (uint64_t)(s * (kFewStage >> 4));
                    const uint32_t bar = done0 + 8 * s;
                    if (++s == kFewStages) { s = 0; parity ^= 1; }
                    ready = tc::poll_mma4_f8(full0 + 8 * s, parity, tmem + buf * kFewRows, da + at, db + at, idesc);
                    tc::commit_both(bar);
                }
        }
    } else if (warp >= 4) {
        // warp w: weight rows 32 (w % 4) .. +31 of the CTA's, tokens kHeld side .. +kHeld - 1
        const int quarter = warp & 3, side = (warp - 4) >> 2, tid = (int)threadIdx.x - 128;
#pragma unroll 4
        for (int i = tid; i < kFewRows * p.k_blocks; i += 32 * kEpiWarps) {
            const int m = i / p.k_blocks, b = i - m * p.k_blocks;
            table[b * kFewRows + m] = m < p.rows ? __ldg(p.xs + m * p.ld_xs + b) : 0.f;
        }
        asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kEpiWarps) : "memory");       // before any of them can give up
        const uint32_t done0 = tc::smem_u32(done), lead_empty = tc::cluster_addr(tc::smem_u32(acc_empty), 0);
        const uint32_t taddr0 = tmem + ((uint32_t)(quarter * 32) << 16) + side * kHeld;
        const bool upper = lane >= 16;
        uint32_t g = 0, s = 0, parity = 0;
        bool ok = true;
        for (int tile = cluster_id; tile < p.n_items && ok; tile += n_clusters) {
            const int block = p.up_row ? tile + (upper ? p.up_row / 128 : 0) : min(2 * tile + (int)rank, p.w_blocks - 1);
            uint32_t at_w = (uint32_t)(block * p.ld_ws);
            float next = __ldg(p.ws + at_w);
            uint64_t sum[kHeld / 2];
#pragma unroll
            for (int i = 0; i < kHeld / 2; ++i) sum[i] = 0ull;
            for (int k = 0; k < p.k_blocks; ++k, ++g) {
                const uint32_t buf = g & 1;
                const uint64_t sw2 = tc::both(next);
                if (k + 1 < p.k_blocks) next = __ldg(p.ws + ++at_w);
                const float4 *sx = reinterpret_cast<const float4 *>(table + k * kFewRows + side * kHeld);
                if (!tc::mbar_wait(done0 + 8 * s, parity, abort_flag, &g_fp8_error, 4)) { ok = false; break; }
                if (++s == kFewStages) { s = 0; parity ^= 1; }
                __syncwarp();
                tc::fence_after();
                uint32_t r[kHeld];
#pragma unroll
                for (int c = 0; c < kHeld; c += 16) tc::ld16_ahead(taddr0 + buf * kFewRows + c, *reinterpret_cast<uint32_t (*)[16]>(r + c));
                tc::wait_ld();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::arrive_relaxed(lead_empty + 8 * buf);
#pragma unroll
                for (int i = 0; i < kHeld / 4; ++i) {
                    const float4 f = sx[i];
                    sum[2 * i] = tc::fma2(tc::pair_of(r[4 * i], r[4 * i + 1]),
                                          tc::mul2(tc::pair_of(__float_as_uint(f.x), __float_as_uint(f.y)), sw2), sum[2 * i]);
                    sum[2 * i + 1] = tc::fma2(tc::pair_of(r[4 * i + 2], r[4 * i + 3]),
                                              tc::mul2(tc::pair_of(__float_as_uint(f.z), __float_as_uint(f.w)), sw2), sum[2 * i + 1]);
                }
            }
            if (!ok) break;
            // with the gate lanes below 16 finish the first half of the tokens, the others the second half
            const int col = p.up_row ? tile * 128 + (int)rank * 64 + quarter * 16 + (lane & 15)
                                     : tile * 256 + (int)rank * 128 + quarter * 32 + lane;
            if (p.up_row) {
#pragma unroll
                for (int i = 0; i < kHeld / 4; ++i) {
                    const uint64_t mine = upper ? sum[kHeld / 4 + i] : sum[i];
                    const uint64_t other = __shfl_xor_sync(0xffffffffu, upper ? sum[i] : sum[kHeld / 4 + i], 16);
                    const uint64_t y = upper ? gated(other, mine) : gated(mine, other);
                    const int m = side * kHeld + (upper ? kHeld / 2 : 0) + 2 * i;
                    store_one(p, m, col, tc::low_of(y));
                    store_one(p, m + 1, col, tc::high_of(y));
                }
            } else {
#pragma unroll
                for (int i = 0; i < kHeld / 2; ++i) {
                    store_one(p, side * kHeld + 2 * i, col, tc::low_of(sum[i]));
                    store_one(p, side * kHeld + 2 * i + 1, col, tc::high_of(sum[i]));
                }
            }
        }
    }

    __syncwarp();
    if (*abort_flag) tc::drain_after_abort();
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(2 * kFewRows) : "memory");
}

bool misaligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

std::mutex g_fp8_mutex;

constexpr int32_t kMaxIn = 1 << 30;              // bytes of a row are counted in 32 bits

template <bool TURNED, int CUT>
int launch(const Fp8Params &p, int sms, cudaStream_t st) {
    static bool ready[64] = {false};
    const int rc = tc::allow_smem(fp8_pair_kernel<TURNED, CUT>, kSmem, ready, g_fp8_mutex, nullptr);
    if (rc != MORTAR_OK) return rc;
    const int clusters = p.n_items < sms / 2 ? p.n_items : sms / 2;
    fp8_pair_kernel<TURNED, CUT><<<(unsigned)(2 * clusters), kThreads, kSmem, st>>>(p);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

// `p` without its maps
int launch_few(Fp8Params &p, const void *x, int64_t ldx, const void *w, int64_t ldw, int in_features, int out_features, int sms,
               cudaStream_t st) {
    static bool ready[64] = {false};
    int rc = tc::allow_smem(fp8_few_kernel, few_smem(kFewBlocks), ready, g_fp8_mutex, nullptr);
    if (rc != MORTAR_OK) return rc;
    rc = tc::encode_u8_2d(&p.map_x, x, in_features, p.rows, ldx, kFewRows / 2);
    if (rc != MORTAR_OK) return rc;
    rc = p.up_row ? tc::encode_u8_3d(&p.map_w, w, in_features, p.up_row, ldw, 16)
                  : tc::encode_u8_2d(&p.map_w, w, in_features, out_features, ldw, 128);
    if (rc != MORTAR_OK) return rc;
    p.n_items = (out_features + 255) / 256;
    const int clusters = p.n_items < sms / 2 ? p.n_items : sms / 2;
    fp8_few_kernel<<<(unsigned)(2 * clusters), kThreads, few_smem(p.k_blocks), st>>>(p);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

// Parts that the reduction of a product without the gate is cut into: where the half tiles fill no more than half of the
// machine and enough blocks are saved to pay for the join (3 to 4 us; a block of a half tile takes 0.3).  64 x 5632 -> 2048
// 25.2 -> 15 us, 333 x 5632 -> 2048 26.7 -> 22, 64 x 2048 -> 768 13.4 -> 10.4, 333 x 2048 -> 768 (13 blocks saved) the
// same 14.5.
// The kernel gives a cluster one part at most, so the clusters are those of the device that it runs on; scratch is asked
// for as if there were kMostClusters (fewer clusters never take more parts).
constexpr int64_t kLeastSaved = 12, kMostClusters = 74;          // blocks; CTA pairs that run at once
int64_t parts_of(int64_t rows, int64_t out_features, int64_t k_blocks, bool gated, int64_t clusters) {
    if (gated || rows <= small::kMaxRows) return 1;
    const int64_t halves = 2 * ((rows + 255) / 256) * ((out_features + 255) / 256);
    const int64_t most = std::min(std::min(clusters, kMostClusters) / halves, k_blocks);
    if (most < 2) return 1;
    const int64_t longest = (k_blocks + most - 1) / most;
    return k_blocks - longest >= kLeastSaved ? (k_blocks + longest - 1) / longest : 1;
}
int64_t padded(int64_t n) { return (n + 31) / 32 * 32; }

}  // namespace

extern "C" int64_t mortar_linear_fp8_parts(int64_t rows, int32_t out_features, int32_t in_features, int32_t flags, int32_t sms) {
    if (rows < 0 || out_features <= 0 || in_features <= 0 || in_features % 16 || sms < 2) return MORTAR_ERR_SHAPE;
    if (flags & ~MORTAR_FLAG_SWIGLU) return MORTAR_ERR_DTYPE;
    if (in_features > kMaxIn) return MORTAR_ERR_CAPACITY;
    return parts_of(rows, out_features, ((int64_t)in_features + 127) / 128, (flags & MORTAR_FLAG_SWIGLU) != 0, sms / 2);
}

extern "C" int64_t mortar_linear_fp8_scratch_floats(int64_t rows, int32_t out_features, int32_t in_features, int32_t flags) {
    const int64_t parts = mortar_linear_fp8_parts(rows, out_features, in_features, flags, 2 * kMostClusters);
    if (parts < 0) return parts;
    return parts > 1 ? parts * rows * padded(out_features) : 0;
}

extern "C" int mortar_linear_fp8(const void *x, int32_t x_type, int64_t ldx, const float *x_scale, int64_t ld_x_scale,
                                 int64_t rows, const void *w, int32_t w_type, int64_t ldw, const float *w_scale,
                                 int64_t ld_w_scale, int32_t out_features, int32_t in_features, int32_t flags, void *out,
                                 int32_t out_dtype, int64_t ld_out, void *stream) {
    return mortar_linear_fp8_cut(x, x_type, ldx, x_scale, ld_x_scale, rows, w, w_type, ldw, w_scale, ld_w_scale, out_features,
                                 in_features, flags, out, out_dtype, ld_out, nullptr, 0, stream);
}

extern "C" int mortar_linear_fp8_cut(const void *x, int32_t x_type, int64_t ldx, const float *x_scale, int64_t ld_x_scale,
                                     int64_t rows, const void *w, int32_t w_type, int64_t ldw, const float *w_scale,
                                     int64_t ld_w_scale, int32_t out_features, int32_t in_features, int32_t flags, void *out,
                                     int32_t out_dtype, int64_t ld_out, float *scratch, int64_t scratch_floats, void *stream) {
    if (!x || !x_scale || !w || !w_scale || !out) return MORTAR_ERR_NULL;
    const bool gated = (flags & MORTAR_FLAG_SWIGLU) != 0;
    const int64_t k_blocks = ((int64_t)in_features + 127) / 128;
    if (rows < 0 || out_features <= 0 || in_features <= 0 || in_features % 16 || ldx < in_features ||
        ldw < in_features || ld_x_scale < k_blocks || ld_w_scale < k_blocks || (gated && out_features % 256) ||
        ld_out < (gated ? out_features / 2 : out_features))
        return MORTAR_ERR_SHAPE;
    if ((x_type != MORTAR_E4M3 && x_type != MORTAR_E5M2) || (w_type != MORTAR_E4M3 && w_type != MORTAR_E5M2) ||
        (out_dtype != MORTAR_F32 && out_dtype != MORTAR_BF16 && out_dtype != MORTAR_F16) || (flags & ~MORTAR_FLAG_SWIGLU))
        return MORTAR_ERR_DTYPE;
    const size_t e = out_dtype == MORTAR_F32 ? 4 : 2;
    if (misaligned(x, 16) || misaligned(w, 16) || ldx % 16 || ldw % 16 || misaligned(out, e) || misaligned(x_scale, 4) ||
        misaligned(w_scale, 4) || misaligned(scratch, 32))
        return MORTAR_ERR_ALIGN;
    if (in_features > kMaxIn || rows > 0x7fffff00LL || out_features > 0x7fffff00 || rows * ld_x_scale > 0xffffffffLL ||
        ((int64_t)out_features + 127) / 128 * ld_w_scale > 0xffffffffLL)
        return MORTAR_ERR_CAPACITY;
    if (rows == 0) return MORTAR_OK;
    cudaStream_t st = (cudaStream_t)stream;

    int sms = 0;
    int rc = tc::sm_count(&sms);
    if (rc != MORTAR_OK) return rc;
    // Up to 16 rows the small kernel wins everywhere, up to 32 where its CTAs share the reduction of few output columns: 32 x
    // 5632 -> 2048 12.9 against 24.8 us below, 32 x 2048 -> 2048 8.3 against 12.6, 32 x 768 -> 2304 7.2 against 9.0,
    // 32 x 4096 -> 4096 16.7 against 20.0; but 32 x 2048 -> 5632 14.4 against 12.9, 32 x 768 -> 4096 10.4 against 9.1
    const int64_t row_tiles = ((int64_t)out_features + 255) / 256;
    if (rows <= 16 || (rows <= small::kMaxRows && row_tiles <= std::max<int64_t>(k_blocks, 12))) {
        small::Params q = {};
        q.x = (const uint8_t *)x; q.ldx = ldx; q.w = (const uint8_t *)w; q.ldw = ldw;
        q.rows = (int)rows; q.n = gated ? out_features / 2 : out_features; q.up_row = gated ? out_features / 2 : 0;
        q.k_bytes = in_features;
        q.xs = x_scale; q.ws = w_scale; q.ld_xs = ld_x_scale; q.ld_ws = ld_w_scale;
        q.out = out; q.ld_out = ld_out; q.out_dtype = out_dtype; q.x_dtype = x_type; q.w_dtype = w_type;
        return small::launch(q, sms, st);
    }
    rc = tc::bind_context();
    if (rc != MORTAR_OK) return rc;
    alignas(64) Fp8Params p = {};
    p.xs = x_scale; p.ws = w_scale; p.ld_xs = ld_x_scale; p.ld_ws = ld_w_scale;
    p.rows = rows;
    p.n = gated ? out_features / 2 : out_features;
    p.up_row = gated ? out_features / 2 : 0;
    p.k_blocks = (int)k_blocks;
    p.w_blocks = (out_features + 127) / 128;
    p.out = out; p.ld_out = ld_out; p.out_dtype = out_dtype;
    if (rows <= kFewRows && k_blocks <= kFewBlocks) {
        p.types = (w_type == MORTAR_E5M2 ? 1u << 7 : 0u) | (x_type == MORTAR_E5M2 ? 1u << 10 : 0u);
        return launch_few(p, x, ldx, w, ldw, in_features, out_features, sms, st);
    }
    p.types = (x_type == MORTAR_E5M2 ? 1u << 7 : 0u) | (w_type == MORTAR_E5M2 ? 1u << 10 : 0u);
    rc = tc::encode_u8_2d(&p.map_x, x, in_features, rows, ldx, 128);
    if (rc != MORTAR_OK) return rc;
    rc = tc::encode_u8_2d(&p.map_w, w, in_features, out_features, ldw, 128);
    if (rc != MORTAR_OK) return rc;
    const int tile_n = gated ? 128 : 256;
    p.tiles_m = (int)((rows + 255) / 256);
    p.tiles_n = (p.n + tile_n - 1) / tile_n;
    if ((int64_t)p.tiles_m * p.tiles_n > 0x3fffffff) return MORTAR_ERR_CAPACITY;
    const int tiles = p.tiles_m * p.tiles_n, clusters = sms / 2, rest = tiles % clusters;
    // The tiles of a round that is at most half full are cut in two.  Behind no, one, two and four full rounds that takes
    // 12.4 -> 10.4, 20.6 -> 18.6, 38.8 -> 37.2 and 60.8 -> 59.8 us; behind six it changes nothing, and behind more the
    // kernel that can do both is the slower one (nineteen: 216.6 -> 220.7).
    p.parts = 1;
    p.whole = 2 * rest <= clusters && tiles < 5 * clusters ? tiles - rest : tiles;
    p.n_items = 2 * tiles - p.whole;
    const int64_t parts = scratch ? parts_of(rows, out_features, k_blocks, gated, clusters) : 1;
    if (p.whole < tiles || parts > 1) {
        rc = tc::encode_u8_2d(&p.map_w_half, w, in_features, out_features, ldw, 64);
        if (rc != MORTAR_OK) return rc;
    }
    if (parts > 1) {
        const int64_t ld = padded(out_features);
        if (scratch_floats < parts * rows * ld) return MORTAR_ERR_CAPACITY;
        const int64_t blocks = (rows * (ld / 4) + 255) / 256;
        if (blocks > 0x7fffffffLL) return MORTAR_ERR_CAPACITY;
        p.parts = (int)parts;
        p.part_step = rows * ld;
        p.n_items = 2 * tiles * p.parts;
        p.out = scratch; p.ld_out = ld; p.out_dtype = MORTAR_F32;
        rc = launch<false, kParts>(p, sms, st);
        if (rc != MORTAR_OK) return rc;
        return tc::launch_after(fp8_join_kernel, (unsigned)blocks, 256u, 0, st, (const float *)scratch, (int)parts, (long long)p.part_step,
                                (long long)ld, (long long)rows, (int)out_features, out, (long long)ld_out, (int)out_dtype);
    }
    const bool turned = misaligned(out, 32) || (ld_out * e) % 32 || p.n % 32;

    if (p.whole < tiles) return turned ? launch<true, kHalves>(p, sms, st) : launch<false, kHalves>(p, sms, st);
    return turned ? launch<true, kWhole>(p, sms, st) : launch<false, kWhole>(p, sms, st);
}

extern "C" int mortar_linear_fp8_error(int32_t *code, int32_t reset) {
    if (!code) return MORTAR_ERR_NULL;
    int v = 0;
    MORTAR_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_fp8_error, sizeof(int)));
    *code = v;
    if (reset && v != 0) {
        const int zero = 0;
        MORTAR_CUDA_CHECK(cudaMemcpyToSymbol(g_fp8_error, &zero, sizeof(int)));
    }
    return MORTAR_OK;
}
