// Row kernels of a quantised block (see gate_norm.cuh). A row belongs to one block, a thread holds up to 24 (32 for
// plain quantising) of its values in registers between the passes over it, so each byte crosses HBM once.
#include "gate_norm.cuh"
#include "common.cuh"
#include "launch.cuh"
#include "quant.cuh"

namespace mkb {

namespace {

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the block's threads, in the same order in every thread and call. `s`: a float for each warp, not used by
// another reduction of the block (so no barrier has to guard its reuse).
__device__ __forceinline__ float block_sum(float v, float* s)
{
    v = warp_sum(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1)
        return v;
    if ((threadIdx.x & 31) == 0)
        s[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < warps; ++i)
        t += s[i];
    return t;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s)
{
    v = __reduce_max_sync(0xffffffffu, v);
    const int warps = blockDim.x >> 5;
    if (warps == 1)
        return v;
    if ((threadIdx.x & 31) == 0)
        s[threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t t = 0;
    for (int i = 0; i < warps; ++i)
        t = max(t, s[i]);
    return t;
}

// VEC consecutive values as fp32.
template <int VEC>
__device__ __forceinline__ void load_f32(const float* p, float* v)
{
    if constexpr (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x;
        v[1] = t.y;
        v[2] = t.z;
        v[3] = t.w;
    } else {
        v[0] = *p;
    }
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t u)
{
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

template <int VEC>
__device__ __forceinline__ void load_bf16(const __nv_bfloat16* p, float* v)
{
    if constexpr (VEC == 8) {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_bf16(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else if constexpr (VEC == 4) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        const float2 a = unpack_bf16(t.x), b = unpack_bf16(t.y);
        v[0] = a.x;
        v[1] = a.y;
        v[2] = b.x;
        v[3] = b.y;
    } else {
        v[0] = __bfloat162float(*p);
    }
}

template <int VEC>
__device__ __forceinline__ void store_f32(float* p, const float* v)
{
    if constexpr (VEC == 4)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
        *p = v[0];
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Standardises the row held in v (NC chunks of VEC values a thread; values past the row are 0 on entry).
template <int VEC, int NC>
__device__ __forceinline__ void normalise(float (&v)[NC][VEC], int kind, int n, float eps, float (*red)[32])
{
    const int tid = threadIdx.x, T = blockDim.x;
    float mean = 0.0f;
    if (kind == kNormLayer) {  // mean first, then the squares about it: no cancellation where the mean is large
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                s += v[i][k];
        mean = block_sum(s, red[0]) / float(n);
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if ((i * T + tid) * VEC < n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[i][k] -= mean;
                s = fmaf(v[i][k], v[i][k], s);
            }
    const float r = rsqrtf(block_sum(s, red[1]) / float(n) + eps);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            v[i][k] *= r;
}

// One block a row: VEC values at a time, NC chunks a thread. n is a multiple of VEC.
template <int VEC, int NC>
__global__ void __launch_bounds__(512) k_gate_norm(const GateNormArgs a)
{
    __shared__ float red[5][32];
    grid_dep_wait();
    grid_dep_launch();
    const long row = blockIdx.x;
    const int tid = threadIdx.x, T = blockDim.x, n = a.n;
    const long sample = row / a.rows_per_sample;
    float x[NC][VEC], y[NC][VEC];
    const float* xr = a.x + row * a.ldx;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * T + tid) * VEC;
        if (c < n) {
            load_f32<VEC>(xr + c, x[i]);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                x[i][k] = 0.0f;
        }
    }
    if (a.y) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (i * T + tid) * VEC;
            if (c >= n) {
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    y[i][k] = 0.0f;
            } else if (a.y_f32) {
                load_f32<VEC>(static_cast<const float*>(a.y) + row * a.ldy + c, y[i]);
            } else {
                load_bf16<VEC>(static_cast<const __nv_bfloat16*>(a.y) + row * a.ldy + c, y[i]);
            }
        }
        if (a.y_norm != kNormNone)
            normalise<VEC, NC>(y, a.y_norm, n, a.eps, red);
        const float* gate = a.gate ? a.gate + sample * a.gate_stride : nullptr;
        float* xo = a.x_out + row * a.ldxo;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = (i * T + tid) * VEC;
            if (c < n) {
                float g[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    g[k] = 1.0f;
                if (gate) {
                    load_f32<VEC>(gate + c, g);
                    if (a.tanh_gate) {
#pragma unroll
                        for (int k = 0; k < VEC; ++k)
                            g[k] = tanhf(g[k]);
                    }
                }
                if (a.y_weight) {
                    float w[VEC];
                    load_f32<VEC>(a.y_weight + c, w);
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        y[i][k] *= w[k];
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    x[i][k] = fmaf(g[k], y[i][k], x[i][k]);
                store_f32<VEC>(xo + c, x[i]);
            }
        }
    }
    if (a.out_type == kOutNone)
        return;
    if (a.x_norm != kNormNone)
        normalise<VEC, NC>(x, a.x_norm, n, a.eps, red + 2);
    const float* scale = a.scale ? a.scale + sample * a.mod_stride : nullptr;
    const float* shift = a.shift ? a.shift + sample * a.mod_stride : nullptr;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * T + tid) * VEC;
        if (c < n) {
            float t[VEC];
            if (a.x_weight) {
                load_f32<VEC>(a.x_weight + c, t);
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    x[i][k] *= t[k];
            }
            if (scale) {
                load_f32<VEC>(scale + c, t);
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    x[i][k] = fmaf(x[i][k], t[k], x[i][k]);
            }
            if (shift) {
                load_f32<VEC>(shift + c, t);
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    x[i][k] += t[k];
            }
            if (a.out_type == kOutBf16) {
                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + row * a.ldo + c;
                if constexpr (VEC == 4)
                    *reinterpret_cast<uint2*>(o) =
                        make_uint2(pack_bf16(x[i][0], x[i][1]), pack_bf16(x[i][2], x[i][3]));
                else
                    *o = __float2bfloat16(x[i][0]);
            } else if (a.out_type == kOutF32) {
                store_f32<VEC>(static_cast<float*>(a.out) + row * a.ldo + c, x[i]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    top = max(top, abs_bits(x[i][k]));
            }
        }
    }
    if (a.out_type != kOutI8)
        return;
    const RowStep step(block_max(top, reinterpret_cast<uint32_t*>(red[4])));
    if (tid == 0)
        a.out_scale[row] = step.step;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * T + tid) * VEC;
        if (c < n) {
            int8_t* o = static_cast<int8_t*>(a.out) + row * a.ldo + c;
            if constexpr (VEC == 4)
                *reinterpret_cast<uint32_t*>(o) = pack4_i8(step(x[i][0]), step(x[i][1]), step(x[i][2]), step(x[i][3]));
            else
                *o = int8_t(step(x[i][0]));
        }
    }
}

// One block a row; rows up to blockDim * NC * VEC values stay in registers.
template <typename XT, int VEC, int NC>
__global__ void __launch_bounds__(512) k_quant_rows(const QuantRowsArgs a)
{
    __shared__ uint32_t red[32];
    grid_dep_wait();
    grid_dep_launch();
    const long row = blockIdx.x;
    const int tid = threadIdx.x, T = blockDim.x, n = a.n;
    const XT* xr = static_cast<const XT*>(a.x) + row * a.ldx;
    int8_t* qr = a.q + row * a.ldq;
    float x[NC][VEC];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * T + tid) * VEC;
        if (c < n) {
            if constexpr (sizeof(XT) == 4)
                load_f32<VEC>(xr + c, x[i]);
            else
                load_bf16<VEC>(xr + c, x[i]);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                x[i][k] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            top = max(top, abs_bits(x[i][k]));
    const RowStep step(block_max(top, red));
    if (tid == 0)
        a.scale[row] = step.step;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = (i * T + tid) * VEC;
        if (c < n) {
            if constexpr (VEC == 1) {
                qr[c] = int8_t(step(x[i][0]));
            } else {
                uint32_t p[VEC / 4];
#pragma unroll
                for (int k = 0; k < VEC / 4; ++k)
                    p[k] = pack4_i8(step(x[i][4 * k]), step(x[i][4 * k + 1]), step(x[i][4 * k + 2]),
                                    step(x[i][4 * k + 3]));
                if constexpr (VEC == 8)
                    *reinterpret_cast<uint2*>(qr + c) = make_uint2(p[0], p[1]);
                else
                    *reinterpret_cast<uint32_t*>(qr + c) = p[0];
            }
        }
    }
}

// Rows too long for a block's registers: a pass for the step, a second one (out of L2) for the values.
template <typename XT>
__global__ void __launch_bounds__(512) k_quant_long(const QuantRowsArgs a)
{
    __shared__ uint32_t red[32];
    grid_dep_wait();
    grid_dep_launch();
    const long row = blockIdx.x;
    const XT* xr = static_cast<const XT*>(a.x) + row * a.ldx;
    int8_t* qr = a.q + row * a.ldq;
    uint32_t top = 0;
    for (int c = threadIdx.x; c < a.n; c += blockDim.x)
        top = max(top, abs_bits(float(xr[c])));
    const RowStep step(block_max(top, red));
    if (threadIdx.x == 0)
        a.scale[row] = step.step;
    for (int c = threadIdx.x; c < a.n; c += blockDim.x)
        qr[c] = int8_t(step(float(xr[c])));
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <int VEC, int NC>
cudaError_t launch_gate_norm(const GateNormArgs& a, int threads, cudaStream_t st)
{
    return launch_k(k_gate_norm<VEC, NC>, dim3(unsigned(a.rows)), threads, 0, st, a);
}

template <typename XT, int VEC, int NC>
cudaError_t launch_quant(const QuantRowsArgs& a, int threads, cudaStream_t st)
{
    return launch_k(k_quant_rows<XT, VEC, NC>, dim3(unsigned(a.rows)), threads, 0, st, a);
}

}  // namespace

cudaError_t gate_norm(const GateNormArgs& a, cudaStream_t st)
{
    if (a.rows == 0)
        return cudaSuccess;
    // 16-byte accesses where every row and vector allows them, single values otherwise.
    const size_t yb = a.y_f32 ? 16 : 8, ob = a.out_type == kOutBf16 ? 8 : a.out_type == kOutF32 ? 16 : 4;
    const bool vec = a.n % 4 == 0 && aligned(a.x, 16) && a.ldx % 4 == 0 &&
                     (!a.y || (aligned(a.y, yb) && a.ldy % 4 == 0 && aligned(a.x_out, 16) && a.ldxo % 4 == 0)) &&
                     aligned(a.y_weight, 16) && aligned(a.gate, 16) && a.gate_stride % 4 == 0 &&
                     aligned(a.x_weight, 16) && aligned(a.scale, 16) && aligned(a.shift, 16) &&
                     a.mod_stride % 4 == 0 && (a.out_type == kOutNone || (aligned(a.out, ob) && a.ldo % 4 == 0));
    // Up to 24 values a thread (both rows' values stay in registers), so as many warps as that takes.
    int warps = 1;
    while (warps * 32 * 24 < a.n && warps < 16)
        warps *= 2;
    const int per = (a.n + warps * 32 - 1) / (warps * 32), t = warps * 32;
    cudaError_t e;
    if (vec) {
        const int nc = (a.n / 4 + t - 1) / t;
        e = nc <= 1   ? launch_gate_norm<4, 1>(a, t, st)
            : nc <= 2 ? launch_gate_norm<4, 2>(a, t, st)
            : nc <= 4 ? launch_gate_norm<4, 4>(a, t, st)
                      : launch_gate_norm<4, 6>(a, t, st);
    } else {
        e = per <= 8    ? launch_gate_norm<1, 8>(a, t, st)
            : per <= 16 ? launch_gate_norm<1, 16>(a, t, st)
                        : launch_gate_norm<1, 24>(a, t, st);
    }
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

cudaError_t quantize_rows(const QuantRowsArgs& a, cudaStream_t st)
{
    if (a.rows == 0)
        return cudaSuccess;
    int warps = 1;
    while (warps * 32 * 32 < a.n && warps < 16)
        warps *= 2;
    const int t = warps * 32, v = a.x_f32 ? 4 : 8;
    const bool vec = a.n % v == 0 && aligned(a.x, 16) && a.ldx % v == 0 && aligned(a.q, v) && a.ldq % v == 0;
    const int per = (a.n + t - 1) / t;
    cudaError_t e;
    if (per > 32) {
        e = a.x_f32 ? launch_k(k_quant_long<float>, dim3(unsigned(a.rows)), 512, 0, st, a)
                    : launch_k(k_quant_long<__nv_bfloat16>, dim3(unsigned(a.rows)), 512, 0, st, a);
    } else if (!vec) {
        if (a.x_f32)
            e = per <= 8 ? launch_quant<float, 1, 8>(a, t, st) : launch_quant<float, 1, 32>(a, t, st);
        else
            e = per <= 8 ? launch_quant<__nv_bfloat16, 1, 8>(a, t, st) : launch_quant<__nv_bfloat16, 1, 32>(a, t, st);
    } else if (a.x_f32) {
        const int nc = (a.n / 4 + t - 1) / t;
        e = nc <= 2 ? launch_quant<float, 4, 2>(a, t, st)
            : nc <= 4 ? launch_quant<float, 4, 4>(a, t, st)
            : nc <= 6 ? launch_quant<float, 4, 6>(a, t, st)
                      : launch_quant<float, 4, 8>(a, t, st);
    } else {
        const int nc = (a.n / 8 + t - 1) / t;
        e = nc <= 1 ? launch_quant<__nv_bfloat16, 8, 1>(a, t, st)
            : nc <= 2 ? launch_quant<__nv_bfloat16, 8, 2>(a, t, st)
            : nc <= 3 ? launch_quant<__nv_bfloat16, 8, 3>(a, t, st)
                      : launch_quant<__nv_bfloat16, 8, 4>(a, t, st);
    }
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace mkb
