// Y[m][n] = act(x_scale[m] * w_scale[n] * sum_k X[m][k] W[n][k] + bias[n]) for 8-bit integer X [M][K] and W [N][K]
// with 32-bit integer sums, which are exact: |sum| < 2^31 for K up to kI8MaxK.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

namespace mkb {

constexpr int kI8MaxK = 131071;  // 128 * 128 * K < 2^31

struct GemmI8Args {
    const int8_t* x;
    long ldx;
    const float* x_scale;  // [M]
    const int8_t* w;
    long ldw;
    const float* w_scale;  // [N]
    const float* bias;     // [N] or null
    void* y;               // fp32 (out_f32) or bf16
    long ldy;
    int M, N, K;
    int act;  // Act of gemm.cuh
    int out_f32;
    uint32_t* status;
    // Failure-path testing only (mkb_selftest_stalled_proj_i8): the pair kernel's CTA 0 withholds its first stage's load.
    int test_stall = 0;
};
cudaError_t gemm_i8(const GemmI8Args& a, const char** err, cudaStream_t st);

}  // namespace mkb
