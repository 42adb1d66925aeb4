// Layer norm over the last dimension, forward and backward.
//
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r, y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// (the norm of the reference's router query, morph/model/routing.py:159-284, and of blocks that
// normalise by it).  Sums, statistics and the gradients of weight and bias are fp32; y and dx are
// rounded once, to the rows' type.
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>
#include <type_traits>
#include "common.h"
#include "tc_pair.cuh"

namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

constexpr int kThreads = 256;

// Sum of `v` over the CTA, the same value in every thread.  `red` holds one float per warp.
__device__ __forceinline__ float cta_sum(float v, float *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < kThreads / 32; ++w) s += red[w];
    return s;
}

// ---- rows in registers: up to 16384 columns ---------------------------------------------------
//
// A group of warps owns a row, thread t of its G columns 8 (t + G i) .. + 7 for i < NE: one pass over
// memory, the row stays in registers (packed as it was read) for mean, variance and result, the next
// row is on its way meanwhile, and a thread keeps its columns' weights, and in the backward pass their
// gradients' sums, from row to row.
//
// Rows may start anywhere (odd widths, slices): the 16 bytes at an unaligned address are cut out of
// the two aligned vectors that hold them (the second is the next thread's, so it comes from L1), and a
// result row that starts off 16 bytes is put together from a lane's words and its neighbour's.

constexpr int kUnit = 8;                                 // columns a thread holds side by side
constexpr int kFar = 16384;                              // most columns that stay in registers

struct Span { const char *lo, *hi; };                    // bytes of a tensor, first to last row

// words[0..3] = the 16 bytes at p.  `n` bytes of them are wanted; the rest may hold anything.
__device__ __forceinline__ void load16(const char *p, int n, const Span &span, uint32_t (&w)[4]) {
    const uint32_t sh = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
    if (sh == 0 && n >= 16) {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        return;
    }
    const char *a = p - sh;
    if (a >= span.lo && a + 32 <= span.hi) {
        const uint4 v0 = __ldg(reinterpret_cast<const uint4 *>(a)), v1 = __ldg(reinterpret_cast<const uint4 *>(a) + 1);
        const uint32_t c[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        uint32_t d[6], e[5];
#pragma unroll
        for (int i = 0; i < 6; ++i) d[i] = (sh & 8u) ? c[i + 2] : c[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) e[i] = (sh & 4u) ? d[i + 1] : d[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(e[i], e[i + 1], (sh & 3u) * 8u);
        return;
    }
    // first or last bytes of the tensor: two at a time, nothing outside it
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = 4 * i < n ? *reinterpret_cast<const uint16_t *>(p + 4 * i) : 0u;
        const uint32_t hi = 4 * i + 2 < n ? *reinterpret_cast<const uint16_t *>(p + 4 * i + 2) : 0u;
        w[i] = lo | hi << 16;
    }
}

// Eight columns of a thread as they lie in memory.
template <class T> struct Unit {
    static constexpr int kVecs = sizeof(T) * kUnit / 16;
    uint32_t w[kVecs][4];
    // `n` columns (0..8) exist
    __device__ __forceinline__ void load(const T *p, int n, const Span &span) {
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
            const int left = n * (int)sizeof(T) - 16 * v;
            if (left > 0) load16(reinterpret_cast<const char *>(p) + 16 * v, left, span, w[v]);
            else w[v][0] = w[v][1] = w[v][2] = w[v][3] = 0u;
        }
    }
    __device__ __forceinline__ float get(int j) const;
    __device__ __forceinline__ void put(int j, float even, float odd);           // columns j, j + 1
};
template <> __device__ __forceinline__ float Unit<float>::get(int j) const { return __uint_as_float(w[j >> 2][j & 3]); }
template <> __device__ __forceinline__ void Unit<float>::put(int j, float a, float b) {
    w[j >> 2][j & 3] = __float_as_uint(a);
    w[j >> 2][(j & 3) + 1] = __float_as_uint(b);
}
template <> __device__ __forceinline__ float Unit<__nv_bfloat16>::get(int j) const {
    const uint32_t v = w[0][j >> 1];
    return __uint_as_float((j & 1) ? v & 0xffff0000u : v << 16);
}
template <> __device__ __forceinline__ void Unit<__nv_bfloat16>::put(int j, float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    w[0][j >> 1] = *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ float Unit<__half>::get(int j) const {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[0][j >> 1]));
    return (j & 1) ? f.y : f.x;
}
template <> __device__ __forceinline__ void Unit<__half>::put(int j, float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    w[0][j >> 1] = *reinterpret_cast<const uint32_t *>(&v);
}

// Stores the units of a warp, lane after lane in memory, `n` columns each.  Where the row starts off 16
// bytes, every aligned vector between two full neighbours is put together from both; the ends of the
// warp's stretch go out column by column.
template <class T>
__device__ __forceinline__ void store_unit(T *p, int n, const Unit<T> &u) {
    constexpr int kVecs = Unit<T>::kVecs;
    const uint32_t sh = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;             // the same in all lanes
    if (sh == 0) {
        if (n == kUnit) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v)
                reinterpret_cast<uint4 *>(p)[v] = make_uint4(u.w[v][0], u.w[v][1], u.w[v][2], u.w[v][3]);
        } else {
#pragma unroll
            for (int j = 0; j < kUnit; ++j)
                if (j < n) p[j] = from_f32<T>(u.get(j));
        }
        return;
    }
    const int lane = threadIdx.x & 31;
    const bool full_above = __shfl_down_sync(0xffffffffu, n, 1) == kUnit && lane < 31;
    const bool joined_below = __shfl_up_sync(0xffffffffu, n, 1) == kUnit && lane > 0 && n == kUnit;
    {
        // last 16 bytes of the lane below
        uint32_t below[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) below[i] = __shfl_up_sync(0xffffffffu, u.w[kVecs - 1][i], 1);
        if (n == kUnit) {
            // aligned vector v covers the last `sh` bytes of what precedes vector v and the first 16 - sh of it
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                if (v == 0 && !joined_below) continue;
                const uint32_t c[8] = {v ? u.w[v - (v > 0)][0] : below[0], v ? u.w[v - (v > 0)][1] : below[1],
                                       v ? u.w[v - (v > 0)][2] : below[2], v ? u.w[v - (v > 0)][3] : below[3],
                                       u.w[v][0], u.w[v][1], u.w[v][2], u.w[v][3]};
                const uint32_t k = 16u - sh;                                          // bytes of c that are skipped
                uint32_t d[6], e[5], r[4];
#pragma unroll
                for (int i = 0; i < 6; ++i) d[i] = (k & 8u) ? c[i + 2] : c[i];
#pragma unroll
                for (int i = 0; i < 5; ++i) e[i] = (k & 4u) ? d[i + 1] : d[i];
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(e[i], e[i + 1], (k & 3u) * 8u);
                *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p) - sh + 16 * v) = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
    }
    // what no aligned vector took: the head of a lane that is not joined to the one below, the tail of one that is
    // not joined to the one above
    const int head = n == kUnit ? (joined_below ? 0 : (16 - (int)sh) / (int)sizeof(T)) : n;
    const int tail = n == kUnit && !full_above ? kUnit - (int)sh / (int)sizeof(T) : kUnit;
#pragma unroll
    for (int j = 0; j < kUnit; ++j)
        if (j < n && (j < head || j >= tail)) p[j] = from_f32<T>(u.get(j));
}

// The warps of a CTA form groups of `warps`, one row each at a time.  A group meets at its own named
// barrier, so the groups run apart; two sets of sums take turns, so one barrier a sum is enough.
struct Group {
    int warps, id, warp, thread;
    float2 *red;                                         // [2][16]
    uint32_t turn;
};

__device__ __forceinline__ Group make_group(int warps, float2 (*red)[2][16]) {
    Group g;
    g.warps = warps;
    g.id = (int)(threadIdx.x >> 5) / warps;
    g.warp = (int)(threadIdx.x >> 5) - g.id * warps;
    g.thread = (int)threadIdx.x - g.id * warps * 32;
    g.red = &red[g.id][0][0];
    g.turn = 0;
    return g;
}

// Sums of a and b over the threads of a row, the same in all of them.
__device__ __forceinline__ float2 group_sum(float a, float b, Group &g) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (g.warps == 1) return make_float2(a, b);
    float2 *red = g.red + 16 * (g.turn & 1u);
    ++g.turn;
    if ((threadIdx.x & 31) == 0) red[g.warp] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;\n" ::"r"(g.id + 1), "r"(g.warps * 32) : "memory");
    float2 s = red[0];
    for (int w = 1; w < g.warps; ++w) {
        s.x += red[w].x;
        s.y += red[w].y;
    }
    return s;
}

template <class T>
__device__ __forceinline__ Span span_of(const T *p, long long ld, long long rows, int cols) {
    return Span{reinterpret_cast<const char *>(p), reinterpret_cast<const char *>(p + (rows - 1) * ld + cols)};
}

constexpr int kForwardWarps = 32, kBackwardWarps = 24, kMaxGroups = 15, kWideWarps = 16;
template <int NE> constexpr int kForwardThreads = 32 * (NE == 1 ? kForwardWarps : kWideWarps);
template <int NE> constexpr int kBackwardThreads = 32 * (NE == 1 ? kBackwardWarps : kWideWarps);

template <class T, int NE>
struct Row {
    Unit<T> u[NE];
    __device__ __forceinline__ void load(const T *p, long long row, long long ld, int cols, const Group &g, const Span &span) {
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int c = kUnit * (g.thread + 32 * g.warps * i);
            u[i].load(p + row * ld + c, max(0, min(kUnit, cols - c)), span);
        }
    }
};

template <class T, int NE>
__global__ void __launch_bounds__(kForwardThreads<NE>, 1)
layer_norm_kernel(const T *__restrict__ x, long long ldx, long long rows, int cols, const float *__restrict__ w,
                  const float *__restrict__ b, float eps, T *__restrict__ y, long long ldy, float *__restrict__ stats,
                  int warps) {
    __shared__ float2 red[kForwardWarps][2][16];
    Group g = make_group(warps, red);
    const int groups = (int)(blockDim.x >> 5) / warps;
    const Span span = span_of(x, ldx, rows, cols);
    const float inv = 1.f / cols;
    const long long stride = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + g.id;
    float wv[NE][kUnit], bv[NE][kUnit];
#pragma unroll
    for (int i = 0; i < NE; ++i)
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
            const int c = kUnit * (g.thread + 32 * warps * i) + j;
            wv[i][j] = w && c < cols ? __ldg(w + c) : 1.f;
            bv[i][j] = b && c < cols ? __ldg(b + c) : 0.f;
        }
    Row<T, NE> next;
    if (row < rows) next.load(x, row, ldx, cols, g, span);
    for (; row < rows; row += stride) {
        const Row<T, NE> cur = next;
        if (row + stride < rows) next.load(x, row + stride, ldx, cols, g, span);      // under this row's sums
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int j = 0; j < kUnit; ++j)
                s += kUnit * (g.thread + 32 * warps * i) + j < cols ? cur.u[i].get(j) : 0.f;
        const float mean = group_sum(s, 0.f, g).x * inv;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int j = 0; j < kUnit; ++j) {
                const float d = kUnit * (g.thread + 32 * warps * i) + j < cols ? cur.u[i].get(j) - mean : 0.f;
                v = fmaf(d, d, v);
            }
        const float rstd = rsqrtf(group_sum(v, 0.f, g).x * inv + eps);
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int c = kUnit * (g.thread + 32 * warps * i);
            Unit<T> r;
#pragma unroll
            for (int j = 0; j < kUnit; j += 2)
                r.put(j, fmaf((cur.u[i].get(j) - mean) * rstd, wv[i][j], bv[i][j]),
                      fmaf((cur.u[i].get(j + 1) - mean) * rstd, wv[i][j + 1], bv[i][j + 1]));
            store_unit(y + row * ldy + c, max(0, min(kUnit, cols - c)), r);
        }
        if (stats && g.thread == 0) {
            stats[row] = mean;
            stats[rows + row] = rstd;
        }
    }
}

// dx, and partial[cta][0 / 1][col] = the sums of dy xh and dy over the CTA's rows.
template <class T, int NE>
__global__ void __launch_bounds__(kBackwardThreads<NE>, 1)
layer_norm_backward_kernel(const T *__restrict__ dy, long long lddy, const T *__restrict__ x, long long ldx, long long rows,
                           int cols, const float *__restrict__ w, const float *__restrict__ stats, T *__restrict__ dx,
                           long long lddx, float *__restrict__ partial, int warps) {
    tc::let_next();
    __shared__ float2 red[kBackwardWarps][2][16];
    extern __shared__ float fold[];                      // [groups][columns, rounded up to the group's]
    Group g = make_group(warps, red);
    const int groups = (int)(blockDim.x >> 5) / warps;
    const Span sx = span_of(x, ldx, rows, cols), sd = span_of(dy, lddy, rows, cols);
    const float inv = 1.f / cols;
    const long long stride = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + g.id;
    float dw[NE][kUnit], db[NE][kUnit], wv[NE][kUnit];
#pragma unroll
    for (int i = 0; i < NE; ++i)
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
            const int c = kUnit * (g.thread + 32 * warps * i) + j;
            dw[i][j] = db[i][j] = 0.f;
            wv[i][j] = w && c < cols ? __ldg(w + c) : 1.f;
        }
    Row<T, NE> nx, nd;
    float next_mean = 0.f, next_rstd = 0.f;
    if (row < rows) {
        nx.load(x, row, ldx, cols, g, sx);
        nd.load(dy, row, lddy, cols, g, sd);
        next_mean = __ldg(stats + row);
        next_rstd = __ldg(stats + rows + row);
    }
    for (; row < rows; row += stride) {
        const Row<T, NE> cx = nx, cd = nd;
        const float mean = next_mean, rstd = next_rstd;
        if (row + stride < rows) {                                                    // under this row's sums
            nx.load(x, row + stride, ldx, cols, g, sx);
            nd.load(dy, row + stride, lddy, cols, g, sd);
            next_mean = __ldg(stats + row + stride);
            next_rstd = __ldg(stats + rows + row + stride);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int j = 0; j < kUnit; ++j) {
                const bool in = kUnit * (g.thread + 32 * warps * i) + j < cols;
                const float d = in ? cd.u[i].get(j) : 0.f, xh = in ? (cx.u[i].get(j) - mean) * rstd : 0.f, t = d * wv[i][j];
                s1 += t;
                s2 = fmaf(t, xh, s2);
                dw[i][j] = fmaf(d, xh, dw[i][j]);
                db[i][j] += d;
            }
        if (dx) {
            const float2 c = group_sum(s1, s2, g);
            const float c1 = c.x * inv, c2 = c.y * inv;
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const int col = kUnit * (g.thread + 32 * warps * i);
                Unit<T> r;
#pragma unroll
                for (int j = 0; j < kUnit; j += 2) {
                    float o[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float xh = (cx.u[i].get(j + k) - mean) * rstd;
                        o[k] = (cd.u[i].get(j + k) * wv[i][j + k] - c1 - xh * c2) * rstd;
                    }
                    r.put(j, o[0], o[1]);
                }
                store_unit(dx + row * lddx + col, max(0, min(kUnit, cols - col)), r);
            }
        }
    }
    if (!partial) return;
    float *dst = partial + (long long)blockIdx.x * 2 * cols;
    if (groups == 1) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int j = 0; j < kUnit; ++j) {
                const int c = kUnit * (g.thread + 32 * warps * i) + j;
                if (c < cols) {
                    dst[c] = dw[i][j];
                    dst[cols + c] = db[i][j];
                }
            }
        return;
    }
    // several groups: add their sums in group order, dw first, then db
    const int width = 32 * kUnit * NE * warps;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            float4 *f = reinterpret_cast<float4 *>(fold + g.id * width + kUnit * (g.thread + 32 * warps * i));
            const float (&v)[kUnit] = which ? db[i] : dw[i];
            f[0] = make_float4(v[0], v[1], v[2], v[3]);
            f[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += blockDim.x) {
            float s = 0.f;
            for (int r = 0; r < groups; ++r) s += fold[r * width + c];
            dst[which * cols + c] = s;
        }
    }
}

// ---- the same for rows that are whole vectors ---------------------------------------------------
//
// Where every row starts on 16 bytes (fp32: 32) and has a multiple of 8 columns, a unit is there or not, loads
// and stores are single vectors of a unit's size, and the arithmetic runs on pairs of columns (fma.rn.f32x2 and its
// like): 16 to 18 instructions a column forward and 29 backward, against 20 and 34 above.  A thread takes NE units
// of its row.  The next row is on its way meanwhile, forward in registers, backward two or three rows in shared
// memory (forward too that takes longer: bf16 39 instead of 35 us).  [16384][2048] fp32: forward 48 us = 5.5 TB/s (57
// with a unit in two 16-byte vectors), backward 73 us = 5.5 TB/s (a copy reaches 5.9 here); [65536][2048] bf16: 115 us =
// 4.7 TB/s and 140 us = 5.7 TB/s (the kernels above: 180 and 207 us); [8192][5632] fp32 backward 131 us (192 without rows
// on their way, which fp32 rows of two units have no registers for).  What is left forward is the two sums that a row
// waits for.

constexpr int kWholeWarps = 16;                          // of a CTA, one CTA an SM: 128 registers a thread

template <class T> constexpr int kVecs = sizeof(T) * kUnit / 16;                     // 16-byte vectors of a unit
template <class T> struct Packed { uint4 v[kVecs<T>]; };
template <class T> __device__ __forceinline__ void load_packed(Packed<T> &u, const T *p) {
    if constexpr (sizeof(T) == 4) {
        uint32_t r[8];
        tc::load_v8(reinterpret_cast<const float *>(p), r);
        u.v[0] = make_uint4(r[0], r[1], r[2], r[3]);
        u.v[1] = make_uint4(r[4], r[5], r[6], r[7]);
    } else {
        u.v[0] = __ldg(reinterpret_cast<const uint4 *>(p));
    }
}
// four pairs of columns as fp32
__device__ __forceinline__ void unpack(const Packed<float> &u, uint64_t (&p)[4]) {
    p[0] = tc::pair_of(u.v[0].x, u.v[0].y); p[1] = tc::pair_of(u.v[0].z, u.v[0].w);
    p[2] = tc::pair_of(u.v[1].x, u.v[1].y); p[3] = tc::pair_of(u.v[1].z, u.v[1].w);
}
__device__ __forceinline__ void unpack(const Packed<__nv_bfloat16> &u, uint64_t (&p)[4]) {
    const uint32_t w[4] = {u.v[0].x, u.v[0].y, u.v[0].z, u.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = tc::pair_of(w[i] << 16, w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const Packed<__half> &u, uint64_t (&p)[4]) {
    const uint32_t w[4] = {u.v[0].x, u.v[0].y, u.v[0].z, u.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        p[i] = tc::pair_of(__float_as_uint(f.x), __float_as_uint(f.y));
    }
}
template <class T> __device__ __forceinline__ void store_pairs(T *dst, const uint64_t (&p)[4]) {
    if constexpr (sizeof(T) == 4) {
        uint32_t r[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) { r[2 * i] = __float_as_uint(tc::low_of(p[i])); r[2 * i + 1] = __float_as_uint(tc::high_of(p[i])); }
        tc::store_v8(dst, r);
    } else {
        constexpr bool kHalf = std::is_same<T, __half>::value;
        *reinterpret_cast<uint4 *>(dst) =
            make_uint4(tc::pack16(tc::low_of(p[0]), tc::high_of(p[0]), kHalf), tc::pack16(tc::low_of(p[1]), tc::high_of(p[1]), kHalf),
                       tc::pack16(tc::low_of(p[2]), tc::high_of(p[2]), kHalf), tc::pack16(tc::low_of(p[3]), tc::high_of(p[3]), kHalf));
    }
}
__device__ __forceinline__ void load_pairs(const float *p, int c, bool in, float fill, uint64_t (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = p && in ? tc::pair_of(__float_as_uint(__ldg(p + c + 2 * i)), __float_as_uint(__ldg(p + c + 2 * i + 1))) : tc::both(fill);
}

template <class T, int NE>
__global__ void __launch_bounds__(32 * kWholeWarps, 1)
layer_norm_whole_kernel(const T *__restrict__ x, long long ldx, long long rows, int cols, const float *__restrict__ w,
                        const float *__restrict__ b, float eps, T *__restrict__ y, long long ldy, float *__restrict__ stats,
                        int warps) {
    __shared__ float2 red[kWholeWarps][2][16];
    Group g = make_group(warps, red);
    const int groups = (int)(blockDim.x >> 5) / warps;
    const float inv = 1.f / cols;
    const long long stride = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + g.id;
    uint64_t wv[NE][4], bv[NE][4];
    bool in[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int c = kUnit * (g.thread + 32 * warps * i);
        in[i] = c < cols;
        load_pairs(w, c, in[i], 1.f, wv[i]);
        load_pairs(b, c, in[i], 0.f, bv[i]);
    }
    const T *xp = x + row * ldx + kUnit * g.thread;
    T *yp = y + row * ldy + kUnit * g.thread;
    Packed<T> next[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i)
        if (row < rows && in[i]) load_packed(next[i], xp + 32 * kUnit * warps * i);
    for (; row < rows; row += stride, yp += stride * ldy) {
        uint64_t v[NE][4];
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            unpack(next[i], v[i]);
            if (!in[i]) v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0ull;
        }
        xp += stride * ldx;
#pragma unroll
        for (int i = 0; i < NE; ++i)                                                // under this row's sums
            if (row + stride < rows && in[i]) load_packed(next[i], xp + 32 * kUnit * warps * i);
        uint64_t s = 0ull;
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s = tc::add2(s, v[i][j]);
        const float mean = group_sum(tc::low_of(s) + tc::high_of(s), 0.f, g).x * inv;
        const uint64_t minus = tc::both(-mean);
        s = 0ull;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (in[i]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[i][j] = tc::add2(v[i][j], minus);
                    s = tc::fma2(v[i][j], v[i][j], s);
                }
            }
        const float rstd = rsqrtf(group_sum(tc::low_of(s) + tc::high_of(s), 0.f, g).x * inv + eps);
        const uint64_t r2 = tc::both(rstd);
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (in[i]) {
                uint64_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = tc::fma2(tc::mul2(v[i][j], r2), wv[i][j], bv[i][j]);
                store_pairs(yp + 32 * kUnit * warps * i, o);
            }
        if (stats && g.thread == 0) {
            stats[row] = mean;
            stats[rows + row] = rstd;
        }
    }
}

// Rows on their way in shared memory, so that they hold no registers: a thread copies the vectors of its own units
// where a unit is one vector, and of fp32 units, two vectors, a warp's lanes copy vectors that lie side by side (each its
// own they would ask for half a sector at a time: 111 instead of 78 us at [16384][2048]).  `kSlots` rows of R operands, one
// of them at work; a slot is filled again a row after it was read.
template <class T, int NE, int R> struct Ring {
    static constexpr int kV = kVecs<T>, kRow = R * NE * kV;                           // vectors of a thread and a row
    static constexpr int kSlots = 4 * kRow * 16 * 32 * kWholeWarps <= 200 * 1024 ? 4 : 3;
    static constexpr int kBytes = kSlots * kRow * 16;                                 // of a thread
    uint4 *mine;
    bool there[NE][kV];
    int get_slot = 0, put_slot = 0;
    // `col`: the first column of this thread's unit 0, `step`: columns from unit to unit
    __device__ __forceinline__ Ring(uint4 *shared, int col, int step, int cols)
        : mine(shared + (threadIdx.x >> 5) * kSlots * kRow * 32 + (threadIdx.x & 31)) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int v = 0; v < kV; ++v) there[i][v] = first(col) + 128 * v + step * i < cols;
    }
    static __device__ __forceinline__ int first(int col) { return kV == 1 ? col : col - 4 * (int)(threadIdx.x & 31); }
    __device__ __forceinline__ uint4 *at(int slot, int r, int i) { return mine + ((slot * R + r) * NE + i) * kV * 32; }
    // `row`: column `first(col)` of the row
    __device__ __forceinline__ void put(int r, const T *row, int step) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
#pragma unroll
            for (int v = 0; v < kV; ++v)
                if (there[i][v])
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(tc::smem_u32(at(put_slot, r, i) + 32 * v)),
                                 "l"(row + step * i + 128 * v) : "memory");
    }
    __device__ __forceinline__ void end_row() {                                       // also where no row is left
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        if (++put_slot == kSlots) put_slot = 0;
    }
    __device__ __forceinline__ void wait_row() {
        asm volatile("cp.async.wait_group %0;\n" ::"n"(kSlots - 2) : "memory");
        if (kV > 1) __syncwarp();
    }
    __device__ __forceinline__ void get(int r, int i, Packed<T> &u) {
#pragma unroll
        for (int v = 0; v < kV; ++v) u.v[v] = at(get_slot, r, i)[(int)(threadIdx.x & 31) * (kV - 1) + v];
    }
    __device__ __forceinline__ void end_read() {
        if (kV > 1) __syncwarp();
        if (++get_slot == kSlots) get_slot = 0;
    }
};

template <class T, int NE>
__global__ void __launch_bounds__(32 * kWholeWarps, 1)
layer_norm_whole_backward_kernel(const T *__restrict__ dy, long long lddy, const T *__restrict__ x, long long ldx,
                                 long long rows, int cols, const float *__restrict__ w, const float *__restrict__ stats,
                                 T *__restrict__ dx, long long lddx, float *__restrict__ partial, int warps) {
    tc::let_next();
    __shared__ float2 red[kWholeWarps][2][16];
    extern __shared__ uint4 ring_s[];
    float *fold = reinterpret_cast<float *>(ring_s);     // at the end: [groups][columns, rounded up to the group's]
    Group g = make_group(warps, red);
    const int groups = (int)(blockDim.x >> 5) / warps;
    const float inv = 1.f / cols;
    const long long stride = (long long)gridDim.x * groups;
    long long row = (long long)blockIdx.x * groups + g.id;
    const int step = 32 * kUnit * warps;
    Ring<T, NE, 2> ring(ring_s, kUnit * g.thread, step, cols);
    const T *xp = x + row * ldx + ring.first(kUnit * g.thread), *dp = dy + row * lddy + ring.first(kUnit * g.thread);
    bool in[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) in[i] = kUnit * (g.thread + 32 * warps * i) < cols;
    long long ahead = row;
    auto fetch = [&] {
        if (ahead < rows) {
            ring.put(0, xp, step);
            ring.put(1, dp, step);
        }
        ring.end_row();
        ahead += stride;
        xp += stride * ldx;
        dp += stride * lddy;
    };
#pragma unroll
    for (int k = 1; k < ring.kSlots; ++k) fetch();
    uint64_t dw[NE][4], db[NE][4], wv[NE][4];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        load_pairs(w, kUnit * (g.thread + 32 * warps * i), in[i], 1.f, wv[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) dw[i][j] = db[i][j] = 0ull;
    }
    float next_mean = row < rows ? __ldg(stats + row) : 0.f, next_rstd = row < rows ? __ldg(stats + rows + row) : 0.f;
    for (; row < rows; row += stride) {
        uint64_t xv[NE][4], dv[NE][4];
        const float mean = next_mean, rstd = next_rstd;
        const uint64_t minus = tc::both(-mean), r2 = tc::both(rstd);
        ring.wait_row();
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (in[i]) {
                Packed<T> ux, ud;
                ring.get(0, i, ux);
                ring.get(1, i, ud);
                unpack(ux, xv[i]);
                unpack(ud, dv[i]);
            }
        ring.end_read();
        fetch();
        if (row + stride < rows) {
            next_mean = __ldg(stats + row + stride);
            next_rstd = __ldg(stats + rows + row + stride);
        }
        uint64_t s1 = 0ull, s2 = 0ull;
#pragma unroll
        for (int i = 0; i < NE; ++i)
            if (in[i]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    xv[i][j] = tc::mul2(tc::add2(xv[i][j], minus), r2);
                    dw[i][j] = tc::fma2(dv[i][j], xv[i][j], dw[i][j]);
                    db[i][j] = tc::add2(db[i][j], dv[i][j]);
                    dv[i][j] = tc::mul2(dv[i][j], wv[i][j]);
                    s1 = tc::add2(s1, dv[i][j]);
                    s2 = tc::fma2(dv[i][j], xv[i][j], s2);
                }
            }
        if (dx) {
            const float2 c = group_sum(tc::low_of(s1) + tc::high_of(s1), tc::low_of(s2) + tc::high_of(s2), g);
            const uint64_t c1 = tc::both(-c.x * inv), c2 = tc::both(-c.y * inv);
            T *op = dx + row * lddx + kUnit * g.thread;
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (in[i]) {
                    uint64_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = tc::mul2(tc::fma2(xv[i][j], c2, tc::add2(dv[i][j], c1)), r2);
                    store_pairs(op + step * i, o);
                }
        }
    }
    if (!partial) return;
    float *dst = partial + (long long)blockIdx.x * 2 * cols;
    const int width = step * NE;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (groups > 1) __syncthreads();
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            const int c = kUnit * (g.thread + 32 * warps * i);
            const uint64_t (&v)[4] = which ? db[i] : dw[i];
            if (groups > 1) {
                float4 *f = reinterpret_cast<float4 *>(fold + g.id * width + c);
                f[0] = make_float4(tc::low_of(v[0]), tc::high_of(v[0]), tc::low_of(v[1]), tc::high_of(v[1]));
                f[1] = make_float4(tc::low_of(v[2]), tc::high_of(v[2]), tc::low_of(v[3]), tc::high_of(v[3]));
            }
            else if (in[i])
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    dst[which * cols + c + 2 * j] = tc::low_of(v[j]);
                    dst[which * cols + c + 2 * j + 1] = tc::high_of(v[j]);
                }
        }
        if (groups == 1) continue;
        __syncthreads();
        for (int c = threadIdx.x; c < cols; c += blockDim.x) {       // the groups' sums, in group order
            float s = 0.f;
            for (int r = 0; r < groups; ++r) s += fold[r * width + c];
            dst[which * cols + c] = s;
        }
    }
}

// ---- any number of columns: the row is read again for each step -------------------------------

template <class T>
__global__ void __launch_bounds__(kThreads)
layer_norm_far_kernel(const T *x, long long ldx, long long rows, int cols, const float *w, const float *b, float eps,
                  T *y, long long ldy, float *stats) {
    __shared__ float red[kThreads / 32];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx;
        T *yr = y + row * ldy;
        float s = 0.f;
        for (int i = threadIdx.x; i < cols; i += kThreads) s += to_f32(xr[i]);
        const float mean = cta_sum(s, red) / cols;
        float v = 0.f;
        for (int i = threadIdx.x; i < cols; i += kThreads) {
            const float d = to_f32(xr[i]) - mean;
            v = fmaf(d, d, v);
        }
        const float rstd = rsqrtf(cta_sum(v, red) / cols + eps);
        for (int i = threadIdx.x; i < cols; i += kThreads) {
            const float xh = (to_f32(xr[i]) - mean) * rstd;
            yr[i] = from_f32<T>(fmaf(xh, w ? w[i] : 1.f, b ? b[i] : 0.f));
        }
        if (stats && threadIdx.x == 0) {
            stats[row] = mean;
            stats[rows + row] = rstd;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
layer_norm_far_dx_kernel(const T *dy, long long lddy, const T *x, long long ldx, long long rows, int cols, const float *w,
                     const float *stats, T *dx, long long lddx) {
    __shared__ float red[kThreads / 32];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * ldx, *dr = dy + row * lddy;
        const float mean = stats[row], rstd = stats[rows + row];
        float s1 = 0.f, s2 = 0.f;
        for (int i = threadIdx.x; i < cols; i += kThreads) {
            const float g = to_f32(dr[i]) * (w ? w[i] : 1.f);
            s1 += g;
            s2 = fmaf(g, (to_f32(xr[i]) - mean) * rstd, s2);
        }
        const float c1 = cta_sum(s1, red) / cols, c2 = cta_sum(s2, red) / cols;
        for (int i = threadIdx.x; i < cols; i += kThreads) {
            const float g = to_f32(dr[i]) * (w ? w[i] : 1.f), xh = (to_f32(xr[i]) - mean) * rstd;
            dx[row * lddx + i] = from_f32<T>((g - c1 - xh * c2) * rstd);
        }
    }
}

// partial[split][0][col] = sum over the split's rows of dy xh, partial[split][1][col] = sum of dy
template <class T>
__global__ void __launch_bounds__(kThreads)
layer_norm_far_dw_kernel(const T *dy, long long lddy, const T *x, long long ldx, long long rows, int cols,
                     const float *stats, float *partial, long long rows_per_split) {
    tc::let_next();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    const long long r0 = blockIdx.y * rows_per_split, r1 = min(rows, r0 + rows_per_split);
    float dw = 0.f, db = 0.f;
    for (long long r = r0; r < r1; ++r) {
        const float d = to_f32(dy[r * lddy + c]);
        dw = fmaf(d, (to_f32(x[r * ldx + c]) - stats[r]) * stats[rows + r], dw);
        db += d;
    }
    partial[(long long)blockIdx.y * 2 * cols + c] = dw;
    partial[(long long)blockIdx.y * 2 * cols + cols + c] = db;
}

// dw / db [col] = sum of the partials: eight interleaved chains a column, added in a fixed order; the loads of
// a chain's next ten parts are in flight together (one at a time it took 10 us, all of it waiting).
__global__ void __launch_bounds__(kThreads)
layer_norm_reduce_kernel(const float *__restrict__ partial, int splits, int cols, float *dw, float *db) {
    __shared__ float part[8][33];
    tc::after_previous();
    const int lane = threadIdx.x & 31, chain = threadIdx.x >> 5;
    const long long c = (long long)blockIdx.x * 32 + lane;
    float s = 0.f;
    const float *src = partial + min(c, 2LL * cols - 1);
    for (int i0 = chain; i0 < splits; i0 += 80) {
        float v[10];
#pragma unroll
        for (int i = 0; i < 10; ++i) v[i] = __ldcg(src + (long long)min(i0 + 8 * i, splits - 1) * 2 * cols);
#pragma unroll
        for (int i = 0; i < 10; ++i) s += i0 + 8 * i < splits ? v[i] : 0.f;
    }
    part[chain][lane] = s;
    __syncthreads();
    if (chain == 0 && c < 2LL * cols) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += part[k][lane];
        float *dst = c < cols ? dw : db;
        if (dst) dst[c < cols ? c : c - cols] = s;
    }
}

bool misaligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

size_t elem_bytes(int dtype) { return dtype == MORTAR_F32 ? 4 : 2; }

// How a row of `cols` columns is laid over a CTA: units of 8 columns a thread, warps a row, and rows at a time (at most
// `most` warps; fewer rows at a time when there are too few rows for every SM).
struct Layout { int units, warps, groups; };

Layout layout_of(int64_t rows, int32_t cols, int most) {
    Layout l;
    l.units = cols <= 4096 ? 1 : cols <= 8192 ? 2 : 4;
    l.warps = (cols + 32 * kUnit * l.units - 1) / (32 * kUnit * l.units);
    int g = l.units > 1 ? 1 : most / l.warps;
    if (l.warps > 1 && g > kMaxGroups) g = kMaxGroups;
    const int64_t share = (rows + 147) / 148;
    l.groups = g < 1 ? 1 : (share < g ? (int)(share < 1 ? 1 : share) : g);
    return l;
}

// CTAs of the backward pass, one partial sum each: one per SM at most, whatever kernel runs
int64_t splits_for(int64_t rows, int32_t) { return rows < 1 ? 1 : (rows < 148 ? rows : 148); }

// The same for rows of whole vectors, 16 warps a CTA: of the units a thread may take, the number that leaves the fewest
// lanes and warps idle (the larger on a tie: less to do per row).
Layout whole_layout(int64_t rows, int32_t cols, int most_units) {
    const int units = cols / kUnit;
    Layout best = {0, 0, 0};
    float best_use = 0.f;
    for (int ne = most_units; ne >= 1; --ne) {
        const int warps = (units + 32 * ne - 1) / (32 * ne);
        if (warps > kWholeWarps) continue;
        int g = kWholeWarps / warps;
        if (warps > 1 && g > kMaxGroups) g = kMaxGroups;
        const float use = (float)units * g / (32.f * ne * kWholeWarps);
        if (use > best_use * 1.0001f) {
            best = {ne, warps, g};
            best_use = use;
        }
    }
    const int64_t share = (rows + 147) / 148;
    if (best.groups > share) best.groups = (int)(share < 1 ? 1 : share);
    return best;                                         // units 0: the row does not fit
}

// the rows' types leave registers for so many units
template <class T> constexpr int kWholeForward = sizeof(T) == 4 ? 2 : 3;
template <class T> constexpr int kWholeBackward = sizeof(T) == 4 ? 1 : 2;             // fp32 rows of more than 4096 columns take 2
                                                                                      // (with the join, 16384 x 2048: 82 instead of
                                                                                      // 77 us, 8192 x 4096: 89 instead of 85)

std::mutex g_norm_mutex;

bool whole_rows(const void *p, int64_t ld, size_t elem) {
    return reinterpret_cast<uintptr_t>(p) % (kUnit * elem) == 0 && ld % kUnit == 0;
}

template <class T, int NE>
int run_whole_forward(const Layout &l, const void *x, int64_t ldx, int64_t rows, int32_t cols, const float *w, const float *b,
                      float eps, void *y, int64_t ldy, float *stats, cudaStream_t st) {
    const int64_t need = (rows + l.groups - 1) / l.groups;
    layer_norm_whole_kernel<T, NE><<<(unsigned)(need < 148 ? need : 148), 32 * l.warps * l.groups, 0, st>>>(
        (const T *)x, ldx, rows, cols, w, b, eps, (T *)y, ldy, stats, l.warps);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T, int NE>
int run_whole_backward(const Layout &l, const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int32_t cols,
                       const float *w, const float *stats, void *dx, int64_t lddx, float *partial, int64_t splits,
                       cudaStream_t st) {
    static bool ready[64] = {false};
    const int threads = 32 * l.warps * l.groups;
    static_assert(Ring<T, NE, 2>::kBytes >= kUnit * NE * (int)sizeof(float), "the groups' sums fit where the rows were");
    const int rc = tc::allow_smem(layer_norm_whole_backward_kernel<T, NE>, Ring<T, NE, 2>::kBytes * 32 * kWholeWarps, ready,
                                  g_norm_mutex, nullptr);
    if (rc != MORTAR_OK) return rc;
    layer_norm_whole_backward_kernel<T, NE><<<(unsigned)splits, threads, Ring<T, NE, 2>::kBytes * threads, st>>>(
        (const T *)dy, lddy, (const T *)x, ldx, rows, cols, w, stats, (T *)dx, lddx, partial, l.warps);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T, int NE>
int run_forward(const Layout &l, const void *x, int64_t ldx, int64_t rows, int32_t cols, const float *w, const float *b,
                float eps, void *y, int64_t ldy, float *stats, cudaStream_t st) {
    const int64_t need = (rows + l.groups - 1) / l.groups;
    layer_norm_kernel<T, NE><<<(unsigned)(need < 148 ? need : 148), 32 * l.warps * l.groups, 0, st>>>(
        (const T *)x, ldx, rows, cols, w, b, eps, (T *)y, ldy, stats, l.warps);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T, int NE>
int run_backward(const Layout &l, const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int32_t cols,
                 const float *w, const float *stats, void *dx, int64_t lddx, float *partial, cudaStream_t st) {
    // at most 24 warps' columns: 24 KB
    const int smem = partial && l.groups > 1 ? l.groups * l.warps * 32 * kUnit * NE * (int)sizeof(float) : 0;
    layer_norm_backward_kernel<T, NE><<<(unsigned)splits_for(rows, cols), 32 * l.warps * l.groups, smem, st>>>(
        (const T *)dy, lddy, (const T *)x, ldx, rows, cols, w, stats, (T *)dx, lddx, partial, l.warps);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T>
int forward(const void *x, int64_t ldx, int64_t rows, int32_t cols, const float *w, const float *b, float eps, void *y,
            int64_t ldy, float *stats, cudaStream_t st) {
    if (cols % kUnit == 0 && whole_rows(x, ldx, sizeof(T)) && whole_rows(y, ldy, sizeof(T))) {
        const Layout l = whole_layout(rows, cols, kWholeForward<T>);
        if (l.units == 1) return run_whole_forward<T, 1>(l, x, ldx, rows, cols, w, b, eps, y, ldy, stats, st);
        if (l.units == 2) return run_whole_forward<T, 2>(l, x, ldx, rows, cols, w, b, eps, y, ldy, stats, st);
        if constexpr (kWholeForward<T> > 2)
            if (l.units == 3) return run_whole_forward<T, 3>(l, x, ldx, rows, cols, w, b, eps, y, ldy, stats, st);
    }
    if (cols <= kFar) {
        const Layout l = layout_of(rows, cols, kForwardWarps);
        if (l.units == 1) return run_forward<T, 1>(l, x, ldx, rows, cols, w, b, eps, y, ldy, stats, st);
        if (l.units == 2) return run_forward<T, 2>(l, x, ldx, rows, cols, w, b, eps, y, ldy, stats, st);
        return run_forward<T, 4>(l, x, ldx, rows, cols, w, b, eps, y, ldy, stats, st);
    }
    const unsigned grid = (unsigned)(rows < 1184 ? rows : 1184);
    layer_norm_far_kernel<T><<<grid, kThreads, 0, st>>>((const T *)x, ldx, rows, cols, w, b, eps, (T *)y, ldy, stats);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T>
int backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int32_t cols, const float *w,
             const float *stats, void *dx, int64_t lddx, float *dw, float *db, float *scratch, cudaStream_t st) {
    const int64_t splits = splits_for(rows, cols);
    float *partial = dw || db ? scratch : nullptr;
    Layout wl = {0, 0, 0};
    if (cols % kUnit == 0 && whole_rows(x, ldx, sizeof(T)) && whole_rows(dy, lddy, sizeof(T)) &&
        (!dx || whole_rows(dx, lddx, sizeof(T))))
        wl = whole_layout(rows, cols, cols <= 4096 ? kWholeBackward<T> : 2);
    if (wl.units) {
        const int rc = wl.units == 1 ? run_whole_backward<T, 1>(wl, dy, lddy, x, ldx, rows, cols, w, stats, dx, lddx, partial, splits, st)
                                     : run_whole_backward<T, 2>(wl, dy, lddy, x, ldx, rows, cols, w, stats, dx, lddx, partial, splits, st);
        if (rc != MORTAR_OK) return rc;
    } else if (cols <= kFar) {
        const Layout l = layout_of(rows, cols, kBackwardWarps);
        const int rc = l.units == 1   ? run_backward<T, 1>(l, dy, lddy, x, ldx, rows, cols, w, stats, dx, lddx, partial, st)
                       : l.units == 2 ? run_backward<T, 2>(l, dy, lddy, x, ldx, rows, cols, w, stats, dx, lddx, partial, st)
                                      : run_backward<T, 4>(l, dy, lddy, x, ldx, rows, cols, w, stats, dx, lddx, partial, st);
        if (rc != MORTAR_OK) return rc;
    } else {
        if (dx) {
            const unsigned grid = (unsigned)(rows < 1184 ? rows : 1184);
            layer_norm_far_dx_kernel<T><<<grid, kThreads, 0, st>>>((const T *)dy, lddy, (const T *)x, ldx, rows, cols, w,
                                                                  stats, (T *)dx, lddx);
            MORTAR_CUDA_CHECK(cudaGetLastError());
        }
        if (partial) {
            const unsigned cb = (unsigned)((cols + kThreads - 1) / kThreads);
            layer_norm_far_dw_kernel<T><<<dim3(cb, (unsigned)splits), kThreads, 0, st>>>(
                (const T *)dy, lddy, (const T *)x, ldx, rows, cols, stats, partial, (rows + splits - 1) / splits);
            MORTAR_CUDA_CHECK(cudaGetLastError());
        }
    }
    if (partial) {
        return tc::launch_after(layer_norm_reduce_kernel, (unsigned)((2LL * cols + 31) / 32), (unsigned)kThreads, 0, st,
                                (const float *)partial, (int)splits, (int)cols, dw, db);
    }
    return MORTAR_OK;
}

constexpr int32_t kMaxCols = 1 << 20;

}  // namespace

extern "C" int mortar_layer_norm(const void *x, int32_t dtype, int64_t ldx, int64_t rows, int32_t cols,
                                 const float *weight, const float *bias, float eps, void *y, int64_t ldy, float *stats,
                                 void *stream) {
    if (!x || !y) return MORTAR_ERR_NULL;
    if (rows < 0 || cols <= 0 || ldx < cols || ldy < cols) return MORTAR_ERR_SHAPE;
    if (dtype != MORTAR_F32 && dtype != MORTAR_BF16 && dtype != MORTAR_F16) return MORTAR_ERR_DTYPE;
    if (cols > kMaxCols) return MORTAR_ERR_CAPACITY;
    if (misaligned(x, elem_bytes(dtype)) || misaligned(y, elem_bytes(dtype)) || misaligned(weight, 4) ||
        misaligned(bias, 4) || misaligned(stats, 4))
        return MORTAR_ERR_ALIGN;
    if (rows == 0) return MORTAR_OK;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MORTAR_F32) return forward<float>(x, ldx, rows, cols, weight, bias, eps, y, ldy, stats, st);
    if (dtype == MORTAR_BF16) return forward<__nv_bfloat16>(x, ldx, rows, cols, weight, bias, eps, y, ldy, stats, st);
    return forward<__half>(x, ldx, rows, cols, weight, bias, eps, y, ldy, stats, st);
}

extern "C" int64_t mortar_layer_norm_scratch_floats(int64_t rows, int32_t cols) {
    if (rows < 0 || cols <= 0) return MORTAR_ERR_SHAPE;
    return splits_for(rows, cols) * 2 * cols;
}

extern "C" int mortar_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int32_t dtype,
                                          int64_t rows, int32_t cols, const float *weight, const float *stats,
                                          void *dx, int64_t lddx, float *dweight, float *dbias, float *scratch,
                                          int64_t scratch_floats, void *stream) {
    if (!dy || !x || !stats) return MORTAR_ERR_NULL;
    if (rows < 0 || cols <= 0 || lddy < cols || ldx < cols || (dx && lddx < cols)) return MORTAR_ERR_SHAPE;
    if (dtype != MORTAR_F32 && dtype != MORTAR_BF16 && dtype != MORTAR_F16) return MORTAR_ERR_DTYPE;
    if (cols > kMaxCols) return MORTAR_ERR_CAPACITY;
    if (misaligned(x, elem_bytes(dtype)) || misaligned(dy, elem_bytes(dtype)) || misaligned(dx, elem_bytes(dtype)) ||
        misaligned(weight, 4) || misaligned(stats, 4) || misaligned(dweight, 4) || misaligned(dbias, 4) ||
        misaligned(scratch, 4))
        return MORTAR_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {
        if (dweight) MORTAR_CUDA_CHECK(cudaMemsetAsync(dweight, 0, (size_t)cols * 4, st));
        if (dbias) MORTAR_CUDA_CHECK(cudaMemsetAsync(dbias, 0, (size_t)cols * 4, st));
        return MORTAR_OK;
    }
    if ((dweight || dbias) && (!scratch || scratch_floats < splits_for(rows, cols) * 2 * cols)) return MORTAR_ERR_CAPACITY;
    if (dtype == MORTAR_F32)
        return backward<float>(dy, lddy, x, ldx, rows, cols, weight, stats, dx, lddx, dweight, dbias, scratch, st);
    if (dtype == MORTAR_BF16)
        return backward<__nv_bfloat16>(dy, lddy, x, ldx, rows, cols, weight, stats, dx, lddx, dweight, dbias, scratch, st);
    return backward<__half>(dy, lddy, x, ldx, rows, cols, weight, stats, dx, lddx, dweight, dbias, scratch, st);
}
