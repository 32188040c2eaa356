// The 8-bit integer projection (see gemm_i8.cuh).
#include "gemm_i8.cuh"
#include "common.cuh"
#include "gemm.cuh"
#include "launch.cuh"

#include <cuda_bf16.h>

namespace mkb {

namespace {

__device__ __forceinline__ float act_of(float v, int act)
{
    switch (act) {
    case kActGeluTanh:
        return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
    case kActSilu:
        return v / (1.0f + __expf(-v));
    case kActQuickGelu:
        return v / (1.0f + __expf(-1.702f * v));
    case kActGeluErf:
        return 0.5f * v * (1.0f + erff(v * 0.7071067811865476f));
    }
    return v;
}

// 64 x 64 outputs a block, 4 x 4 a thread, 64 bytes of K at a time in shared memory.
__global__ void __launch_bounds__(256) k_gemm_i8_simple(const GemmI8Args a)
{
    __shared__ int sx[64][17], sw[64][17];
    grid_dep_wait();
    grid_dep_launch();
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 16; i += 256) {
            const int r = i / 16, c = i % 16;
            uint32_t xv = 0, wv = 0;
            for (int b = 0; b < 4; ++b) {
                const int k = k0 + 4 * c + b;
                if (k < a.K) {
                    if (m0 + r < a.M)
                        xv |= uint32_t(uint8_t(a.x[(m0 + r) * a.ldx + k])) << (8 * b);
                    if (n0 + r < a.N)
                        wv |= uint32_t(uint8_t(a.w[(n0 + r) * a.ldw + k])) << (8 * b);
                }
            }
            sx[r][c] = int(xv);
            sw[r][c] = int(wv);
        }
        __syncthreads();
        for (int c = 0; c < 16; ++c)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __dp4a(sx[ty * 4 + i][c], sw[tx + 16 * j][c], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long m = m0 + ty * 4 + i;
            const int n = n0 + tx + 16 * j;
            if (m >= a.M || n >= a.N)
                continue;
            const float v = act_of(float(acc[i][j]) * a.x_scale[m] * a.w_scale[n] + (a.bias ? a.bias[n] : 0.0f), a.act);
            if (a.out_f32)
                static_cast<float*>(a.y)[m * a.ldy + n] = v;
            else
                static_cast<__nv_bfloat16*>(a.y)[m * a.ldy + n] = __float2bfloat16(v);
        }
}

}  // namespace

cudaError_t gemm_i8(const GemmI8Args& a, const char** err, cudaStream_t st)
{
    (void)err;
    const cudaError_t e = launch_k(k_gemm_i8_simple, dim3((a.N + 63) / 64, (a.M + 63) / 64), 256, 0, st, a);
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace mkb
