// Attention to another stream's keys (see cross_attention.cuh).
#include "cross_attention.cuh"
#include "common.cuh"
#include "launch.cuh"

#include <algorithm>

namespace mkb {

namespace {

// A warp a query row, D / 32 values a lane, one key after another.
template <int D>
__global__ void __launch_bounds__(256) k_cross_simple(const CrossArgs a)
{
    constexpr int E = D / 32;
    grid_dep_wait();
    grid_dep_launch();
    const long w = (long(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (w >= long(a.B) * a.H * a.Lq)
        return;
    const int row = int(w % a.Lq), h = int(w / a.Lq % a.H), b = int(w / a.Lq / a.H), hk = h / (a.H / a.Hkv);
    float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
    const __nv_bfloat16* qr = a.q + b * a.sq.sample + h * a.sq.head + row * a.sq.row;
    for (int i = 0; i < E; ++i)
        q[i] = __bfloat162float(qr[lane + 32 * i]);
    const int n = a.key_len ? min(max(a.key_len[b], 0), a.Lk) : a.Lk;
    for (int j = 0; j < n; ++j) {
        if (a.key_mask && !a.key_mask[b * a.mask_stride + j])
            continue;
        const __nv_bfloat16* kr = a.k + b * a.sk.sample + hk * a.sk.head + j * a.sk.row;
        const __nv_bfloat16* vr = a.v + b * a.sv.sample + hk * a.sv.head + j * a.sv.row;
        float s = 0.0f;
        for (int i = 0; i < E; ++i)
            s = fmaf(q[i], __bfloat162float(kr[lane + 32 * i]), s);
        for (int t = 16; t > 0; t >>= 1)
            s += __shfl_xor_sync(0xffffffffu, s, t);
        s *= a.scale_log2;
        const float mn = fmaxf(m, s), f = exp2f(m - mn), p = exp2f(s - mn);
        l = l * f + p;
        for (int i = 0; i < E; ++i)
            o[i] = fmaf(o[i], f, p * __bfloat162float(vr[lane + 32 * i]));
        m = mn;
    }
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    __nv_bfloat16* dst = a.out + b * a.so.sample + h * a.so.head + row * a.so.row;
    for (int i = 0; i < E; ++i)
        dst[lane + 32 * i] = __float2bfloat16(o[i] * inv);
}

}  // namespace

cudaError_t cross_attention(const CrossArgs& a, const char** err, cudaStream_t st)
{
    (void)err;
    const long warps = long(a.B) * a.H * a.Lq;
    const dim3 grid(unsigned((warps + 7) / 8));
    const cudaError_t e = a.d == 64 ? launch_k(k_cross_simple<64>, grid, 256, 0, st, a)
                                    : launch_k(k_cross_simple<128>, grid, 256, 0, st, a);
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace mkb
