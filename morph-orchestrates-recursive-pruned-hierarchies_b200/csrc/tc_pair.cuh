// Device helpers of the kernels that run one tcgen05 product on two CTAs (cta_group::2): cluster
// addressing, loads and commits that complete on a barrier of either CTA, paired MMAs of both operand
// kinds, wide tensor-memory reads, and the reduced-precision conversions of their epilogues.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "tc_common.cuh"

namespace tc {

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
    return r;
}
// shared::cluster address of the same shared-memory offset in CTA `rank` of this cluster
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }

// TMA tile load into this CTA's shared memory that completes on a barrier of either CTA of the pair
__device__ __forceinline__ void load_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];\n"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void load_pair_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];\n"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(cluster_bar) : "memory");
}
// Whether the phase has completed, without waiting for it (try_wait may hold the thread for a while)
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// one arrival, when the MMAs issued so far have ended, at the barrier of this offset in both CTAs of the pair
__device__ __forceinline__ void commit_both(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// Arrival that orders nothing but execution: what has to be over before it are tensor-memory reads,
// which `wait_ld` and `fence_before` order.  A release at cluster scope would also wait for the
// thread's stores to global memory, a microsecond or more.
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
}
// a pair of fp32 multiply-adds
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ uint64_t both(float v) { return pair_of(__float_as_uint(v), __float_as_uint(v)); }
__device__ __forceinline__ float low_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
// 32 bytes to a 32-byte aligned address
__device__ __forceinline__ void store_v8(void *p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ void load_v8(const void *p, uint32_t *w) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}
template <int REGS> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REGS)); }
// A poll of the barrier that the issuing thread needs next, and the eight (or four) MMAs of a stage as
// one instruction sequence: the poll's result is read after the MMAs have been issued, so its latency
// runs under them.  Descriptors advance by step_a / step_b from MMA to MMA, and from the fourth to the
// fifth so that the fifth starts half_a / half_b after the first.  `acc`: whether the first MMA adds
// to what the accumulator holds.  Returns whether the polled phase had completed.
__device__ __forceinline__ bool poll_mma8_f16(uint32_t bar, uint32_t parity, uint32_t d, uint64_t a, uint64_t b,
                                              uint64_t step_a, uint64_t step_b, uint64_t half_a, uint64_t half_b,
                                              uint32_t idesc, uint32_t acc) {
    uint32_t ready;
    asm volatile(
        "{\n.reg .pred q, p0, p1;\n.reg .b64 x, y, x2, y2;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%1], %2;\n"
        "setp.ne.b32 p0, %11, 0;\nsetp.eq.u32 p1, 1, 1;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], %4, %5, %10, p0;\n"
        "add.s64 x, %4, %6;\nadd.s64 y, %5, %7;\nadd.s64 x2, %4, %8;\nadd.s64 y2, %5, %9;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x, y, %10, p1;\n"
        "add.s64 x, x, %6;\nadd.s64 y, y, %7;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x, y, %10, p1;\n"
        "add.s64 x, x, %6;\nadd.s64 y, y, %7;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x, y, %10, p1;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x2, y2, %10, p1;\n"
        "add.s64 x2, x2, %6;\nadd.s64 y2, y2, %7;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x2, y2, %10, p1;\n"
        "add.s64 x2, x2, %6;\nadd.s64 y2, y2, %7;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x2, y2, %10, p1;\n"
        "add.s64 x2, x2, %6;\nadd.s64 y2, y2, %7;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%3], x2, y2, %10, p1;\n"
        "selp.b32 %0, 1, 0, q;\n}\n"
        : "=r"(ready)
        : "r"(bar), "r"(parity), "r"(d), "l"(a), "l"(b), "l"(step_a), "l"(step_b), "l"(half_a), "l"(half_b), "r"(idesc),
          "r"(acc)
        : "memory");
    return ready != 0;
}
// Four 8-bit MMAs (K = 32 each, 32 bytes apart) into a fresh accumulator.
__device__ __forceinline__ bool poll_mma4_f8(uint32_t bar, uint32_t parity, uint32_t d, uint64_t a, uint64_t b,
                                             uint32_t idesc) {
    uint32_t ready;
    asm volatile(
        "{\n.reg .pred q, p0, p1;\n.reg .b64 x, y;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%1], %2;\n"
        "setp.ne.u32 p0, 1, 1;\nsetp.eq.u32 p1, 1, 1;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%3], %4, %5, %6, p0;\n"
        "add.s64 x, %4, 2;\nadd.s64 y, %5, 2;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%3], x, y, %6, p1;\n"
        "add.s64 x, x, 2;\nadd.s64 y, y, 2;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%3], x, y, %6, p1;\n"
        "add.s64 x, x, 2;\nadd.s64 y, y, 2;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%3], x, y, %6, p1;\n"
        "selp.b32 %0, 1, 0, q;\n}\n"
        : "=r"(ready)
        : "r"(bar), "r"(parity), "r"(d), "l"(a), "l"(b), "r"(idesc)
        : "memory");
    return ready != 0;
}

// 32 accumulator columns of this thread's tensor-memory lane; `wait_ld` before the registers are read
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
// 16 columns, likewise
__device__ __forceinline__ void ld16_ahead(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// two fp32 values as one word of bf16 (or fp16) values, `lo` in the low half, round to nearest even
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool half) {
    if (half) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ float2 unpack16(uint32_t w, bool half) {
    if (half) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}

// A role that gave up leaves copies and MMAs of its CTA in flight; they end within microseconds of
// the last issue, so an aborted CTA waits about a millisecond before it frees anything.
__device__ __forceinline__ void drain_after_abort() {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

// A kernel launched with `launch_after` may start while the one before it in the stream still runs; it
// calls `after_previous` before it touches that kernel's results.  `let_next` in the earlier kernel
// lets the next one start (its blocks take their places as this one's leave).
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;\n"); }

template <class Kernel, class... Args>
inline int launch_after(Kernel kernel, unsigned grid, unsigned block, int smem, cudaStream_t st, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    MORTAR_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
    return MORTAR_OK;
}

// [rows][cols] 8-bit row-major with row stride ld as a 2-D map with a [box_rows][128] box and the
// 128-byte swizzle.
inline int encode_u8_2d(CUtensorMap *map, const void *base, int64_t cols, int64_t rows, int64_t ld,
                        uint32_t box_rows) {
    EncodeTiledFn encode;
    const int rc = get_encode_fn(&encode);
    if (rc != MORTAR_OK) return rc;
    const cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, box_rows};
    const cuuint32_t estride[2] = {1, 1};
    const CUresult cr = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), gdim, gstride, box,
                               estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) {
        mortar_set_cuda_error("cuTensorMapEncodeTiled", "failed to encode a tensor map");
        return MORTAR_ERR_CUDA;
    }
    return MORTAR_OK;
}

// The same matrix seen as its two halves of `rows` rows each: a box is the same [box_rows] rows of both.
inline int encode_u8_3d(CUtensorMap *map, const void *base, int64_t cols, int64_t rows, int64_t ld, uint32_t box_rows) {
    EncodeTiledFn encode;
    const int rc = get_encode_fn(&encode);
    if (rc != MORTAR_OK) return rc;
    const cuuint64_t gdim[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 2};
    const cuuint64_t gstride[2] = {(cuuint64_t)ld, (cuuint64_t)ld * (cuuint64_t)rows};
    const cuuint32_t box[3] = {128, box_rows, 2};
    const cuuint32_t estride[3] = {1, 1, 1};
    const CUresult cr = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), gdim, gstride, box,
                               estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) {
        mortar_set_cuda_error("cuTensorMapEncodeTiled", "failed to encode a tensor map");
        return MORTAR_ERR_CUDA;
    }
    return MORTAR_OK;
}

// Makes the current device's context current to the calling thread.  Encoding a tensor map is a driver
// call and fails in a thread that has made no runtime call that needs a context yet, as an autograd
// thread whose allocations all come from a cache.
inline int bind_context() {
    int dev = 0;
    MORTAR_CUDA_CHECK(cudaGetDevice(&dev));
    MORTAR_CUDA_CHECK(cudaSetDevice(dev));
    return MORTAR_OK;
}

// First use of a kernel on the current device: its dynamic shared memory limit.  `done` holds one
// flag per device.
template <class Kernel>
inline int allow_smem(Kernel kernel, int bytes, bool (&done)[64], std::mutex &m, int *device) {
    int dev = 0;
    MORTAR_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return MORTAR_ERR_CAPACITY;
    std::lock_guard<std::mutex> lock(m);
    if (!done[dev]) {
        MORTAR_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done[dev] = true;
    }
    if (device) *device = dev;
    return MORTAR_OK;
}

// SMs of the current device (queried once per device)
inline int sm_count(int *out) {
    static int cached[64] = {0};
    static std::mutex m;
    int dev = 0;
    MORTAR_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return MORTAR_ERR_CAPACITY;
    std::lock_guard<std::mutex> lock(m);
    if (!cached[dev])
        MORTAR_CUDA_CHECK(cudaDeviceGetAttribute(&cached[dev], cudaDevAttrMultiProcessorCount, dev));
    *out = cached[dev];
    return MORTAR_OK;
}

}  // namespace tc
