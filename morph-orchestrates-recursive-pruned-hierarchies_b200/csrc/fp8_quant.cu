// 8-bit floating point with one fp32 scale per block: 1 x 128 blocks for activations, 128 x 128 for
// weights.  Written (mortar_quantize_fp8) and read back (mortar_dequantize_fp8).
//
//   scale = the smallest power of two with max|block| / scale <= top,  top = 448 (e4m3) or 57344 (e5m2)
//   q = round_to_nearest_even(x / scale)
//
// A power of two costs a floating-point type no precision, only the top binade of its range, and
// keeps x / scale exact, so q is THE nearest value for every input type, ties included; a quotient by
// max|block| / top would round twice.  A block of zeros has scale 1, one below 2^-126 * top scale
// 2^-126; a block that holds an infinity or a NaN has scale NaN, and so reads back as NaN throughout.
//
// Both passes are bound by memory: 8192 x 5632 bf16 quantised in 32 us = 4.3 TB/s and read back in 26 us = 5.4;
// 65536 x 2048 in 78 us = 5.2 TB/s and 76 us (a copy reaches 5.9 here).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "common.h"

namespace {

constexpr int kThreads = 256;

template <class T> struct Chunk8;                    // 8 neighbouring values of a row
template <> struct Chunk8<float> {
    static __device__ __forceinline__ void load(const float *p, float (&v)[8]) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(float *p, const float (&v)[8]) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};
template <> struct Chunk8<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&v)[8]) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&ws[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[8]) {
        __nv_bfloat162 r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(r);
    }
};
template <> struct Chunk8<__half> {
    static __device__ __forceinline__ void load(const __half *p, float (&v)[8]) {
        const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&ws[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(__half *p, const float (&v)[8]) {
        __half2 r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(r);
    }
};

// Largest magnitude of 8 values as a bit pattern: patterns of non-negative floats order like the
// floats, and a NaN's lies above infinity's, so a NaN is not lost as it is in fmaxf.
__device__ __forceinline__ uint32_t magnitude8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// scale and its reciprocal from a block's largest magnitude; `top` = exponent of the type's largest value 1.75 * 2^top
__device__ __forceinline__ void block_scale(uint32_t amax, int top, float &scale, float &inv) {
    if (amax >= 0x7f800000u) {
        scale = inv = __uint_as_float(0x7fc00000u);
        return;
    }
    int e = (int)(amax >> 23) - 127 - top + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (amax == 0) e = 0;
    e = max(e, -126);
    scale = __uint_as_float((uint32_t)(127 + e) << 23);
    inv = __uint_as_float((uint32_t)(127 - e) << 23);
}

__device__ __forceinline__ uint2 to_fp8(const float (&v)[8], float inv, bool e5m2) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 a = make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), b = make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv);
        const __nv_fp8_interpretation_t kind = e5m2 ? __NV_E5M2 : __NV_E4M3;
        w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, kind) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, kind) << 16;
    }
    return make_uint2(w[0], w[1]);
}

// a / b with 32-bit arithmetic where it fits (a 64-bit division costs more than the rest of a block)
__device__ __forceinline__ long long quotient(long long a, int b) {
    return a <= 0xffffffffLL ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// A warp takes 8 blocks of a row: 16 lanes a block, 8 values a lane, four pairs of blocks in flight together.
// With one pair at a time and a division for each the kernel reached 3.4 TB/s of the card's 6.6.
template <class T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T *x, long long ldx, long long rows, int cols, uint8_t *q, long long ldq, float *scale,
                     int e5m2) {
    constexpr int kAtOnce = 4;
    const int n_blocks = (cols + 127) >> 7, parts = (n_blocks + 2 * kAtOnce - 1) / (2 * kAtOnce);
    const int lane = threadIdx.x & 31, sub = lane & 15, side = lane >> 4;
    const long long units = rows * parts, stride = (long long)gridDim.x * (kThreads / 32);
    for (long long unit = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); unit < units; unit += stride) {
        const long long row = quotient(unit, parts);
        const int blk0 = (int)(unit - row * parts) * 2 * kAtOnce + side;
        const T *xr = x + row * ldx + blk0 * 128 + sub * 8;
        float v[kAtOnce][8];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[u][j] = 0.f;
            if ((blk0 + 2 * u) * 128 + sub * 8 < cols) Chunk8<T>::load(xr + u * 256, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int blk = blk0 + 2 * u;
            uint32_t m = magnitude8(v[u]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            float s, inv;
            block_scale(m, e5m2 ? 15 : 8, s, inv);
            if (blk * 128 + sub * 8 < cols) *reinterpret_cast<uint2 *>(q + row * ldq + blk * 128 + sub * 8) = to_fp8(v[u], inv, e5m2 != 0);
            if (blk < n_blocks && sub == 0) scale[row * n_blocks + blk] = s;
        }
    }
}

// One 128 x 128 block per CTA: 16 lanes a row, 16 rows at a time.
template <class T>
__global__ void __launch_bounds__(kThreads)
quantize_tiles_kernel(const T *x, long long ldx, long long rows, int cols, uint8_t *q, long long ldq, float *scale,
                      int e5m2) {
    __shared__ uint32_t red[kThreads / 32];
    const int n_blocks = (cols + 127) >> 7, sub = threadIdx.x & 15;
    const long long rb = blockIdx.x / n_blocks;
    const int blk = (int)(blockIdx.x - rb * n_blocks), col = blk * 128 + sub * 8;
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long row = rb * 128 + i * 16 + (threadIdx.x >> 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (row < rows && col < cols) Chunk8<T>::load(x + row * ldx + col, v[i]);
        m = max(m, magnitude8(v[i]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = max(m, red[w]);
    float s, inv;
    block_scale(m, e5m2 ? 15 : 8, s, inv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long row = rb * 128 + i * 16 + (threadIdx.x >> 4);
        if (row < rows && col < cols) *reinterpret_cast<uint2 *>(q + row * ldq + col) = to_fp8(v[i], inv, e5m2 != 0);
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

// out = q * scale, 8 values a thread, four such chunks in flight together.
template <class T>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t *q, long long ldq, const float *scale, long long rows, int cols, int row_shift, T *out,
                  long long ld_out, int e5m2) {
    constexpr int kAtOnce = 4;
    const int chunks = cols >> 3, n_blocks = (cols + 127) >> 7;
    const long long total = rows * chunks, stride = (long long)gridDim.x * kThreads * kAtOnce;
    for (long long i0 = (long long)blockIdx.x * kThreads * kAtOnce + threadIdx.x; i0 < total; i0 += stride) {
        uint2 w[kAtOnce];
        float s[kAtOnce];
        long long row[kAtOnce];
        int col[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const long long i = i0 + u * kThreads;
            if (i >= total) continue;
            row[u] = quotient(i, chunks);
            col[u] = (int)(i - row[u] * chunks) * 8;
            w[u] = __ldg(reinterpret_cast<const uint2 *>(q + row[u] * ldq + col[u]));
            s[u] = __ldg(scale + (row[u] >> row_shift) * n_blocks + (col[u] >> 7));
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            if (i0 + u * kThreads >= total) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)((j < 2 ? w[u].x : w[u].y) >> (16 * (j & 1)));
                const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, e5m2 ? __NV_E5M2 : __NV_E4M3)));
                v[2 * j] = f.x * s[u];
                v[2 * j + 1] = f.y * s[u];
            }
            Chunk8<T>::store(out + row[u] * ld_out + col[u], v);
        }
    }
}

bool misaligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

int check(const void *x, int64_t ldx, int x_dtype, int64_t rows, int32_t cols, int32_t block_rows, const void *q,
          int32_t q_dtype, int64_t ldq, const float *scale) {
    if (!x || !q || !scale) return MORTAR_ERR_NULL;
    if (rows < 0 || cols <= 0 || cols % 16 || ldx < cols || ldq < cols || (block_rows != 1 && block_rows != 128))
        return MORTAR_ERR_SHAPE;
    if ((x_dtype != MORTAR_F32 && x_dtype != MORTAR_BF16 && x_dtype != MORTAR_F16) ||
        (q_dtype != MORTAR_E4M3 && q_dtype != MORTAR_E5M2))
        return MORTAR_ERR_DTYPE;
    const size_t e = x_dtype == MORTAR_F32 ? 4 : 2;
    if (misaligned(x, 16) || (ldx * e) % 16 || misaligned(q, 16) || ldq % 16 || misaligned(scale, 4))
        return MORTAR_ERR_ALIGN;
    return MORTAR_OK;
}

template <class T>
int quantize(const void *x, int64_t ldx, int64_t rows, int32_t cols, int32_t block_rows, void *q, int e5m2, int64_t ldq,
             float *scale, cudaStream_t st) {
    const int64_t n_blocks = (cols + 127) / 128;
    if (block_rows == 1) {
        const int64_t need = (rows * ((n_blocks + 7) / 8) + kThreads / 32 - 1) / (kThreads / 32);
        quantize_rows_kernel<T><<<(unsigned)(need < 1184 ? need : 1184), kThreads, 0, st>>>(
            (const T *)x, ldx, rows, cols, (uint8_t *)q, ldq, scale, e5m2);
    } else {
        const int64_t need = (rows + 127) / 128 * n_blocks;
        if (need > 0x7fffffffLL) return MORTAR_ERR_CAPACITY;
        quantize_tiles_kernel<T><<<(unsigned)need, kThreads, 0, st>>>((const T *)x, ldx, rows, cols, (uint8_t *)q, ldq,
                                                                      scale, e5m2);
    }
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T>
int dequantize(const void *q, int e5m2, int64_t ldq, const float *scale, int64_t rows, int32_t cols, int32_t block_rows,
               void *out, int64_t ld_out, cudaStream_t st) {
    const int64_t need = (rows * (cols / 8) + 4 * kThreads - 1) / (4 * kThreads);
    dequantize_kernel<T><<<(unsigned)(need < 1184 ? need : 1184), kThreads, 0, st>>>(
        (const uint8_t *)q, ldq, scale, rows, cols, block_rows == 1 ? 0 : 7, (T *)out, ld_out, e5m2);
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

}  // namespace

extern "C" int mortar_quantize_fp8(const void *x, int32_t dtype, int64_t ldx, int64_t rows, int32_t cols,
                                   int32_t block_rows, void *q, int32_t q_dtype, int64_t ldq, float *scale,
                                   void *stream) {
    const int rc = check(x, ldx, dtype, rows, cols, block_rows, q, q_dtype, ldq, scale);
    if (rc != MORTAR_OK || rows == 0) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const int e5m2 = q_dtype == MORTAR_E5M2;
    if (dtype == MORTAR_F32) return quantize<float>(x, ldx, rows, cols, block_rows, q, e5m2, ldq, scale, st);
    if (dtype == MORTAR_BF16) return quantize<__nv_bfloat16>(x, ldx, rows, cols, block_rows, q, e5m2, ldq, scale, st);
    return quantize<__half>(x, ldx, rows, cols, block_rows, q, e5m2, ldq, scale, st);
}

extern "C" int mortar_dequantize_fp8(const void *q, int32_t q_dtype, int64_t ldq, const float *scale, int64_t rows,
                                     int32_t cols, int32_t block_rows, void *out, int32_t out_dtype, int64_t ld_out,
                                     void *stream) {
    const int rc = check(out, ld_out, out_dtype, rows, cols, block_rows, q, q_dtype, ldq, scale);
    if (rc != MORTAR_OK || rows == 0) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const int e5m2 = q_dtype == MORTAR_E5M2;
    if (out_dtype == MORTAR_F32) return dequantize<float>(q, e5m2, ldq, scale, rows, cols, block_rows, out, ld_out, st);
    if (out_dtype == MORTAR_BF16) return dequantize<__nv_bfloat16>(q, e5m2, ldq, scale, rows, cols, block_rows, out, ld_out, st);
    return dequantize<__half>(q, e5m2, ldq, scale, rows, cols, block_rows, out, ld_out, st);
}
