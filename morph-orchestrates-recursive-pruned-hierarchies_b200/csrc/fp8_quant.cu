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
// Both passes are bound by memory: 8192 x 5632 bf16 quantised in 29 us = 4.8 TB/s and read back in 27 us = 5.1 TB/s, fp32 in
// 43 us = 5.4 TB/s each way; 65536 x 2048 in 70 us = 5.8 TB/s and 76 us (a copy reaches 5.9 here).  A thread takes 16
// values: with 8, in 16-byte accesses, bf16 blocks of 128 x 128 took 43 instead of 29 us and fp32 read back 61.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "common.h"
#include "tc_pair.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int32_t kMaxCols = 1 << 30;                    // columns are counted in 32 bits

// 16 neighbouring values of a row as 32-bit words.  WIDE: the row's pieces of 32 bytes start on 32 bytes and are
// moved whole (in two halves, lanes that lie 32 bytes apart ask for half a sector at a time).
template <bool WIDE, int WORDS>
__device__ __forceinline__ void load_words(const void *p, uint32_t (&w)[WORDS]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8) tc::load_v8(reinterpret_cast<const uint32_t *>(p) + i, w + i);
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i / 4);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    }
}
template <bool WIDE, int WORDS>
__device__ __forceinline__ void store_words(void *p, const uint32_t (&w)[WORDS]) {
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 8) {
            uint32_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = w[i + j];
            tc::store_v8(reinterpret_cast<uint32_t *>(p) + i, v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
            reinterpret_cast<uint4 *>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
}
template <class T> constexpr int kWords = 4 * sizeof(T);

__device__ __forceinline__ void to_floats(const uint32_t (&w)[16], float (&v)[16], float) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void to_floats(const uint32_t (&w)[8], float (&v)[16], __nv_bfloat16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void to_floats(const uint32_t (&w)[8], float (&v)[16], __half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void from_floats(const float (&v)[16], uint32_t (&w)[16], float) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
}
__device__ __forceinline__ void from_floats(const float (&v)[16], uint32_t (&w)[8], __nv_bfloat16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = tc::pack16(v[2 * i], v[2 * i + 1], false);
}
__device__ __forceinline__ void from_floats(const float (&v)[16], uint32_t (&w)[8], __half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = tc::pack16(v[2 * i], v[2 * i + 1], true);
}

// Largest magnitude of 16 values as a bit pattern: patterns of non-negative floats order like the
// floats, and a NaN's lies above infinity's, so a NaN is not lost as it is in fmaxf. 
__device__ __forceinline__ uint32_t magnitude(const float (&v)[16]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
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

__device__ __forceinline__ uint4 to_fp8(const float (&v)[16], float inv, bool e5m2) {
    const __nv_fp8_interpretation_t kind = e5m2 ? __NV_E5M2 : __NV_E4M3;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), b = make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv);
        w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, kind) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, kind) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// a / b with 32-bit arithmetic where it fits (a 64-bit division costs more than the rest of a block)
__device__ __forceinline__ long long quotient(long long a, int b) {
    return a <= 0xffffffffLL ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// A warp takes 4 blocks of a row at once: 8 lanes a block, 16 values a lane, and two such groups in flight together (four:
// 16384 x 768 16.4 instead of 14.3 us).  A 64-bit division for each unit held the kernel at 3.4 TB/s.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T *x, long long ldx, long long rows, int cols, uint8_t *q, long long ldq, float *scale,
                     int e5m2) {
    constexpr int kAtOnce = 2;
    const int n_blocks = (cols + 127) >> 7, parts = (n_blocks + 4 * kAtOnce - 1) / (4 * kAtOnce);
    const int lane = threadIdx.x & 31, sub = lane & 7, side = lane >> 3;
    const long long units = rows * parts, stride = (long long)gridDim.x * (kThreads / 32);
    for (long long unit = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); unit < units; unit += stride) {
        const long long row = quotient(unit, parts);
        const int blk0 = (int)(unit - row * parts) * 4 * kAtOnce + side;
        const T *xr = x + row * ldx + blk0 * 128 + sub * 16;
        uint32_t w[kAtOnce][kWords<T>];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
#pragma unroll
            for (int j = 0; j < kWords<T>; ++j) w[u][j] = 0;
            if ((blk0 + 4 * u) * 128 + sub * 16 < cols) load_words<WIDE>(xr + u * 512, w[u]);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int blk = blk0 + 4 * u;
            float v[16];
            to_floats(w[u], v, T());
            uint32_t m = magnitude(v);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            float s, inv;
            block_scale(m, e5m2 ? 15 : 8, s, inv);
            if (blk * 128 + sub * 16 < cols) *reinterpret_cast<uint4 *>(q + row * ldq + blk * 128 + sub * 16) = to_fp8(v, inv, e5m2 != 0);
            if (blk < n_blocks && sub == 0) scale[row * n_blocks + blk] = s;
        }
    }
}

// One 128 x 128 block per CTA: 8 lanes a row, 32 rows at a time.
template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
quantize_tiles_kernel(const T *x, long long ldx, long long rows, int cols, uint8_t *q, long long ldq, float *scale,
                      int e5m2) {
    __shared__ uint32_t red[kThreads / 32];
    const int n_blocks = (cols + 127) >> 7, sub = threadIdx.x & 7;
    const long long rb = blockIdx.x / n_blocks;
    const int blk = (int)(blockIdx.x - rb * n_blocks), col = blk * 128 + sub * 16;
    uint32_t w[4][kWords<T>];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long row = rb * 128 + i * 32 + (threadIdx.x >> 3);
#pragma unroll
        for (int j = 0; j < kWords<T>; ++j) w[i][j] = 0;
        if (row < rows && col < cols) load_words<WIDE>(x + row * ldx + col, w[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[16];
        to_floats(w[i], v, T());
        m = max(m, magnitude(v));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kThreads / 32; ++j) m = max(m, red[j]);
    float s, inv;
    block_scale(m, e5m2 ? 15 : 8, s, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long row = rb * 128 + i * 32 + (threadIdx.x >> 3);
        float v[16];
        to_floats(w[i], v, T());
        if (row < rows && col < cols) *reinterpret_cast<uint4 *>(q + row * ldq + col) = to_fp8(v, inv, e5m2 != 0);
    }
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

// out = q * scale, 16 values a thread, two such chunks in flight together (four: 65536 x 2048 72 instead of 76 us, but
// 300 x 768 8 instead of 6).
constexpr int kReadAtOnce = 2;
template <class T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t *q, long long ldq, const float *scale, long long rows, int cols, int row_shift, T *out,
                  long long ld_out, int e5m2) {
    const int chunks = cols >> 4, n_blocks = (cols + 127) >> 7;
    const long long total = rows * chunks, stride = (long long)gridDim.x * kThreads * kReadAtOnce;
    for (long long i0 = (long long)blockIdx.x * kThreads * kReadAtOnce + threadIdx.x; i0 < total; i0 += stride) {
        uint4 w[kReadAtOnce];
        float s[kReadAtOnce];
        T *dst[kReadAtOnce];
#pragma unroll
        for (int u = 0; u < kReadAtOnce; ++u) {
            const long long i = i0 + u * kThreads;
            if (i >= total) continue;
            const long long row = quotient(i, chunks);
            const int col = (int)(i - row * chunks) * 16;
            w[u] = __ldg(reinterpret_cast<const uint4 *>(q + row * ldq + col));
            s[u] = __ldg(scale + (row >> row_shift) * n_blocks + (col >> 7));
            dst[u] = out + row * ld_out + col;
        }
#pragma unroll
        for (int u = 0; u < kReadAtOnce; ++u) {
            if (i0 + u * kThreads >= total) continue;
            const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            float v[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const __nv_fp8x2_storage_t two = (__nv_fp8x2_storage_t)(words[j / 2] >> (16 * (j & 1)));
                const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, e5m2 ? __NV_E5M2 : __NV_E4M3)));
                v[2 * j] = f.x * s[u];
                v[2 * j + 1] = f.y * s[u];
            }
            uint32_t r[kWords<T>];
            from_floats(v, r, T());
            store_words<WIDE>(dst[u], r);
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
    if (cols > kMaxCols) return MORTAR_ERR_CAPACITY;
    const size_t e = x_dtype == MORTAR_F32 ? 4 : 2;
    if (misaligned(x, 16) || (ldx * e) % 16 || misaligned(q, 16) || ldq % 16 || misaligned(scale, 4))
        return MORTAR_ERR_ALIGN;
    return MORTAR_OK;
}

// the pieces of 32 bytes that rows of whole 16 values are made of start on 32 bytes
template <class T> bool wide_rows(const void *p, int64_t ld) { return !misaligned(p, 32) && ld * (int64_t)sizeof(T) % 32 == 0; }

template <class T, bool WIDE>
int quantize_as(const void *x, int64_t ldx, int64_t rows, int32_t cols, int32_t block_rows, void *q, int e5m2, int64_t ldq,
                float *scale, cudaStream_t st) {
    const int64_t n_blocks = (cols + 127) / 128;
    if (block_rows == 1) {
        const int64_t need = (rows * ((n_blocks + 7) / 8) + kThreads / 32 - 1) / (kThreads / 32);
        quantize_rows_kernel<T, WIDE><<<(unsigned)(need < 1184 ? need : 1184), kThreads, 0, st>>>(
            (const T *)x, ldx, rows, cols, (uint8_t *)q, ldq, scale, e5m2);
    } else {
        const int64_t need = (rows + 127) / 128 * n_blocks;
        if (need > 0x7fffffffLL) return MORTAR_ERR_CAPACITY;
        quantize_tiles_kernel<T, WIDE><<<(unsigned)need, kThreads, 0, st>>>((const T *)x, ldx, rows, cols, (uint8_t *)q, ldq,
                                                                            scale, e5m2);
    }
    MORTAR_CUDA_CHECK(cudaGetLastError());
    return MORTAR_OK;
}

template <class T>
int quantize(const void *x, int64_t ldx, int64_t rows, int32_t cols, int32_t block_rows, void *q, int e5m2, int64_t ldq,
             float *scale, cudaStream_t st) {
    return wide_rows<T>(x, ldx) ? quantize_as<T, true>(x, ldx, rows, cols, block_rows, q, e5m2, ldq, scale, st)
                                : quantize_as<T, false>(x, ldx, rows, cols, block_rows, q, e5m2, ldq, scale, st);
}

template <class T>
int dequantize(const void *q, int e5m2, int64_t ldq, const float *scale, int64_t rows, int32_t cols, int32_t block_rows,
               void *out, int64_t ld_out, cudaStream_t st) {
    const int64_t need = (rows * (cols / 16) + kReadAtOnce * kThreads - 1) / (kReadAtOnce * kThreads);
    const unsigned grid = (unsigned)(need < 1184 ? need : 1184);
    const int shift = block_rows == 1 ? 0 : 7;
    if (wide_rows<T>(out, ld_out))
        dequantize_kernel<T, true><<<grid, kThreads, 0, st>>>((const uint8_t *)q, ldq, scale, rows, cols, shift, (T *)out, ld_out, e5m2);
    else
        dequantize_kernel<T, false><<<grid, kThreads, 0, st>>>((const uint8_t *)q, ldq, scale, rows, cols, shift, (T *)out, ld_out, e5m2);
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
