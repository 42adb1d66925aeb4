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
#include "common.h"

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

template <class T>
__global__ void __launch_bounds__(kThreads)
layer_norm_kernel(const T *x, long long ldx, long long rows, int cols, const float *w, const float *b, float eps,
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
layer_norm_dx_kernel(const T *dy, long long lddy, const T *x, long long ldx, long long rows, int cols, const float *w,
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
layer_norm_dw_kernel(const T *dy, long long lddy, const T *x, long long ldx, long long rows, int cols,
                     const float *stats, float *partial, long long rows_per_split) {
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

// dw / db [col] = sum of the partials in split order
__global__ void __launch_bounds__(kThreads)
layer_norm_reduce_kernel(const float *partial, int splits, int cols, float *dw, float *db) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= 2 * cols) return;
    float s = 0.f;
    for (int i = 0; i < splits; ++i) s += partial[(long long)i * 2 * cols + c];
    float *dst = c < cols ? dw : db;
    if (dst) dst[c < cols ? c : c - cols] = s;
}

bool misaligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

size_t elem_bytes(int dtype) { return dtype == MORTAR_F32 ? 4 : 2; }

constexpr int64_t kMaxSplits = 296;

int64_t splits_for(int64_t rows) { return rows < 1 ? 1 : (rows < kMaxSplits * 4 ? (rows + 3) / 4 : kMaxSplits); }

template <class T>
int forward(const void *x, int64_t ldx, int64_t rows, int32_t cols, const float *w, const float *b, float eps, void *y,
            int64_t ldy, float *stats, cudaStream_t st) {
    const unsigned grid = (unsigned)(rows < 1184 ? rows : 1184);
    layer_norm_kernel<T><<<grid, kThreads, 0, st>>>((const T *)x, ldx, rows, cols, w, b, eps, (T *)y, ldy, stats);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T>
int backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int64_t rows, int32_t cols, const float *w,
             const float *stats, void *dx, int64_t lddx, float *dw, float *db, float *scratch, cudaStream_t st) {
    const unsigned grid = (unsigned)(rows < 1184 ? rows : 1184);
    if (dx) {
        layer_norm_dx_kernel<T><<<grid, kThreads, 0, st>>>((const T *)dy, lddy, (const T *)x, ldx, rows, cols, w, stats,
                                                          (T *)dx, lddx);
        MORTAR_CUDA_CHECK(cudaGetLastError());
    }
    if (dw || db) {
        const int64_t splits = splits_for(rows), rps = (rows + splits - 1) / splits;
        const unsigned cb = (unsigned)((cols + kThreads - 1) / kThreads);
        layer_norm_dw_kernel<T><<<dim3(cb, (unsigned)splits), kThreads, 0, st>>>((const T *)dy, lddy, (const T *)x, ldx,
                                                                                 rows, cols, stats, scratch, rps);
        MORTAR_CUDA_CHECK(cudaGetLastError());
        layer_norm_reduce_kernel<<<(unsigned)((2LL * cols + kThreads - 1) / kThreads), kThreads, 0, st>>>(
            scratch, (int)splits, cols, dw, db);
        MORTAR_CUDA_CHECK(cudaGetLastError());
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
    return splits_for(rows) * 2 * cols;
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
    if ((dweight || dbias) && (!scratch || scratch_floats < splits_for(rows) * 2 * cols)) return MORTAR_ERR_CAPACITY;
    if (dtype == MORTAR_F32)
        return backward<float>(dy, lddy, x, ldx, rows, cols, weight, stats, dx, lddx, dweight, dbias, scratch, st);
    if (dtype == MORTAR_BF16)
        return backward<__nv_bfloat16>(dy, lddy, x, ldx, rows, cols, weight, stats, dx, lddx, dweight, dbias, scratch, st);
    return backward<__half>(dy, lddy, x, ldx, rows, cols, weight, stats, dx, lddx, dweight, dbias, scratch, st);
}
