// Entry of the kernels for a few tokens (dense_small.cu): C[m][n] = sum_k A[m][k] W[n][k], plain or with the
// gate of the two halves of n applied, for 16-bit operands and for 8-bit ones with block scales.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace small {

// Most rows that these kernels take.  Against the tensor-memory kernels (us, L2 flushed): 16-bit block 2048/5632 of 32 rows
// 39 here, 45 in dense_tc.cu with its 256-row tiles; 8-bit operands of 17 to 32 rows only where the weight is narrow, as
// fp8_tc.cu says.
constexpr int kMaxRows = 32;

struct Params {
    const uint8_t *x, *w;            // rows of bytes
    long long ldx, ldw;              // bytes
    int rows;
    int n;                           // output columns (hidden columns with the gate)
    int up_row;                      // 0, or the first up row of w
    int k_bytes;
    const float *xs, *ws;            // 8-bit: block scales
    long long ld_xs, ld_ws;
    void *out;
    long long ld_out;                // elements
    int out_dtype;
    int after_previous;              // x comes from the kernel before in the stream: weights are fetched first
    int x_dtype, w_dtype;
};

// Enqueues one product; `sms` = SMs of the device.
int launch(const Params &p, int sms, cudaStream_t st);

}  // namespace small
