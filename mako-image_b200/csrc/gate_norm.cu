// Row kernels of a quantised block (see gate_norm.cuh). Bounded by HBM: a row's values stay in its block's registers between
// the passes over them, so each byte crosses HBM once. Where there are rows enough a block walks a run of one sample's rows
// with the vectors (weights, gate, modulation: five values for each of a row's elements, out of L2, and the gate's tanh)
// folded into three in shared memory.
#include "gate_norm.cuh"
#include "common.cuh"
#include "gemm.cuh"
#include "launch.cuh"
#include "quant.cuh"

#include <algorithm>

namespace mkb {

namespace {

// Sum (or largest magnitude) over the block's threads, in the same order in every thread and call. `s`: a float for each of up
// to 16 warps; a caller that comes back to the same ones has passed another reduction's barrier in between.
__device__ __forceinline__ float block_sum(float v, float* s)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1)
        return v;
    if (lane == 0)
        s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (lane & 15) < warps ? s[lane & 15] : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float block_max_abs(float v, float* s)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v = max_abs(v, __shfl_xor_sync(0xffffffffu, v, o));
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1)
        return v;
    if (lane == 0)
        s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (lane & 15) < warps ? s[lane & 15] : 0.0f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
        v = max_abs(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// VEC consecutive values as fp32. Rows pass once (streaming loads); the vectors, read by every block, stay cached.
template <int VEC>
__device__ __forceinline__ void load_vec(const float* p, float (&v)[VEC])
{
    if constexpr (VEC == 4) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(p));
        v[0] = t.x;
        v[1] = t.y;
        v[2] = t.z;
        v[3] = t.w;
    } else {
        v[0] = __ldg(p);
    }
}

// Columns c .. c + VEC - 1 of n, 0 outside them.
template <int VEC, bool ODD>
__device__ __forceinline__ void load_cols(const float* p, int c, int n, float (&v)[VEC])
{
    if constexpr (ODD) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            v[k] = unsigned(c + k) < unsigned(n) ? __ldg(p + c + k) : 0.0f;
    } else {
        load_vec(p + c, v);
    }
}

template <int VEC>
__device__ __forceinline__ void load_shared(const float* p, float (&v)[VEC])
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

// VEC values of a row as they lie in memory, so that a load's registers are not touched before its data is wanted.
template <int VEC>
struct Raw {
    uint32_t u[VEC];  // fp32: a word each; bf16: two to a word, VEC / 2 words (VEC = 1: its low half)
    __device__ __forceinline__ void load(const float* p)
    {
        if constexpr (VEC == 4) {
            const uint4 t = __ldcs(reinterpret_cast<const uint4*>(p));
            u[0] = t.x;
            u[1] = t.y;
            u[2] = t.z;
            u[3] = t.w;
        } else {
            u[0] = __ldcs(reinterpret_cast<const uint32_t*>(p));
        }
    }
    __device__ __forceinline__ void load(const __nv_bfloat16* p)
    {
        if constexpr (VEC == 8) {
            const uint4 t = __ldcs(reinterpret_cast<const uint4*>(p));
            u[0] = t.x;
            u[1] = t.y;
            u[2] = t.z;
            u[3] = t.w;
        } else if constexpr (VEC == 4) {
            const uint2 t = __ldcs(reinterpret_cast<const uint2*>(p));
            u[0] = t.x;
            u[1] = t.y;
        } else {
            u[0] = __ldcs(reinterpret_cast<const unsigned short*>(p));
        }
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            u[k] = 0;
    }
    // Value k alone, into words that were zero.
    __device__ __forceinline__ void load_one(const float* p, int k) { u[k] = __ldcs(reinterpret_cast<const uint32_t*>(p) + k); }
    __device__ __forceinline__ void load_one(const __nv_bfloat16* p, int k)
    {
        u[k >> 1] |= uint32_t(__ldcs(reinterpret_cast<const unsigned short*>(p) + k)) << (16 * (k & 1));
    }
    __device__ __forceinline__ void values(bool f32, float (&v)[VEC]) const
    {
        if constexpr (VEC == 8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = unpack_bf16(u[k]);
                v[2 * k] = f.x;
                v[2 * k + 1] = f.y;
            }
        } else if (f32) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                v[k] = __uint_as_float(u[k]);
        } else if constexpr (VEC == 4) {
            const float2 a = unpack_bf16(u[0]), b = unpack_bf16(u[1]);
            v[0] = a.x;
            v[1] = a.y;
            v[2] = b.x;
            v[3] = b.y;
        } else {
            v[0] = __uint_as_float(u[0] << 16);
        }
    }
};

template <int VEC>
__device__ __forceinline__ void store_row(float* p, const float (&v)[VEC])
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

template <int VEC>
__device__ __forceinline__ void store_row(__nv_bfloat16* p, const float (&v)[VEC])
{
    if constexpr (VEC == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    else
        *p = __float2bfloat16(v[0]);
}

// A row's chunks of 32 * VEC values: NC to a warp, one after another, so that a thread's places in the row are constants apart.
// ODD: the row starts `skip` values after a vector's border, so the first and the last vector may be cut; `first` then counts
// from the row's start and may be negative.
template <int VEC, int NC, bool ODD = false>
struct Place {
    int first;  // the thread's first value
    __device__ __forceinline__ explicit Place(int skip = 0)
        : first(int(threadIdx.x >> 5) * NC * 32 * VEC + int(threadIdx.x & 31) * VEC - skip)
    {
    }
    __device__ __forceinline__ int at(int i) const { return first + i * 32 * VEC; }
    // Any of vector i in the row; all of it; value k of it.
    __device__ __forceinline__ bool in(int i, int n) const { return at(i) < n; }
    __device__ __forceinline__ bool all(int i, int n) const { return !ODD || (at(i) >= 0 && at(i) + VEC <= n); }
    __device__ __forceinline__ bool has(int i, int k, int n) const { return !ODD || unsigned(at(i) + k) < unsigned(n); }
};

// Standardises the row held in v (values past the row are 0 on entry and stay so).
template <int VEC, int NC, bool ODD>
__device__ __forceinline__ void normalise(float (&v)[NC][VEC], const Place<VEC, NC, ODD>& at, int kind, int n, float inv_n,
                                          float eps, float* red)
{
    if (kind == kNormLayer) {  // mean first, then the squares about it: no cancellation where the mean is large
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                s += v[i][k];
        const float mean = block_sum(s, red) * inv_n;
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (at.in(i, n))
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (at.has(i, k, n))
                        v[i][k] -= mean;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            s = fmaf(v[i][k], v[i][k], s);
    const float r = rsqrtf(fmaf(block_sum(s, red + 16), inv_n, eps));
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            v[i][k] *= r;
}

template <int VEC, int NC, bool ODD, typename T>
__device__ __forceinline__ void load_row_at(Raw<VEC> (&v)[NC], const T* p, const Place<VEC, NC, ODD>& at, int n)
{
    p += at.first;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if (at.in(i, n) && at.all(i, n)) {
            v[i].load(p + i * 32 * VEC);
        } else {
            v[i].zero();
            if constexpr (ODD) {
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (at.has(i, k, n))
                        v[i].load_one(p + i * 32 * VEC, k);
            }
        }
    }
}

template <int VEC, int NC>
__device__ __forceinline__ void values(const Raw<VEC> (&r)[NC], bool f32, float (&v)[NC][VEC])
{
#pragma unroll
    for (int i = 0; i < NC; ++i)
        r[i].values(f32, v[i]);
}

__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

// `whole`: the row lies on the vectors' borders as the loaded rows do (always, unless ODD).
template <int VEC, int NC, bool ODD, typename T>
__device__ __forceinline__ void store_row_at(const float (&v)[NC][VEC], T* p, const Place<VEC, NC, ODD>& at, int n,
                                             bool whole = true)
{
    p += at.first;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if (at.in(i, n) && at.all(i, n) && (!ODD || whole)) {
            store_row(p + i * 32 * VEC, v[i]);
        } else if constexpr (ODD) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (at.has(i, k, n))
                    store_one(p + i * 32 * VEC + k, v[i][k]);
        }
    }
}

// The row as 8-bit integers with their step.
template <int VEC, int NC, bool ODD>
__device__ __forceinline__ void quant_row_at(const float (&v)[NC][VEC], int8_t* q, float* scale,
                                             const Place<VEC, NC, ODD>& at, int n, float* red, bool whole = true)
{
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            top = max_abs(top, v[i][k]);
    const RowStep step(block_max_abs(top, red));
    if (threadIdx.x == 0)
        *scale = step.step;
    q += at.first;
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (at.in(i, n)) {
            int8_t* o = q + i * 32 * VEC;
            if constexpr (VEC == 1) {
                *o = step.one(v[i][0]);
            } else {
                uint32_t p[VEC / 4];
#pragma unroll
                for (int k = 0; k < VEC / 4; ++k) {
                    const float u[4] = {v[i][4 * k], v[i][4 * k + 1], v[i][4 * k + 2], v[i][4 * k + 3]};
                    p[k] = step.pack4(u);
                }
                if (ODD && !(whole && at.all(i, n))) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        if (at.has(i, k, n))
                            o[k] = int8_t(p[k / 4] >> (8 * (k & 3)));
                } else if constexpr (VEC == 8) {
                    *reinterpret_cast<uint2*>(o) = make_uint2(p[0], p[1]);
                } else {
                    *reinterpret_cast<uint32_t*>(o) = p[0];
                }
            }
        }
}

// tanh(x) to a few units of 2^-24 of itself: below 0.4 its Taylor series to x^13 (what is left is under 2^-27 of x there), to
// 1.5 units, else 1 - 2 / (e^2|x| + 1) with x's sign, where the difference makes up to 14 of the exponential's and the division's.
__device__ __forceinline__ float tanh_near(float x)
{
    const float s = x * x, a = fabsf(x);
    float p = fmaf(s, 3.5921280e-3f, -8.8632355e-3f);
    p = fmaf(s, p, 2.1869488e-2f);
    p = fmaf(s, p, -5.3968254e-2f);
    p = fmaf(s, p, 1.3333333e-1f);
    p = fmaf(s, p, -3.3333333e-1f);
    const float small = fmaf(x * s, p, x);
    const float big = copysignf(1.0f - __fdividef(2.0f, __expf(2.0f * fminf(a, 20.0f)) + 1.0f), x);
    return a < 0.4f ? small : a >= 0.4f ? big : x;  // a NaN comes back
}

// The vectors over a row's places, as far as one chunk of one thread goes: y's factor g(gate) * y_weight, and x's
// h * factor + shift with factor = x_weight * (1 + scale).
template <int VEC, bool ODD>
struct Vectors {
    float gate[VEC], factor[VEC], shift[VEC];
    __device__ __forceinline__ void branch(const GateNormArgs& a, long sample, int c)
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            gate[k] = 1.0f;
        if (a.gate) {
            load_cols<VEC, ODD>(a.gate + sample * a.gate_stride, c, a.n, gate);
            if (a.tanh_gate)
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    gate[k] = tanh_near(gate[k]);
        }
        if (a.y_weight) {
            float w[VEC];
            load_cols<VEC, ODD>(a.y_weight, c, a.n, w);
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                gate[k] *= w[k];
        }
    }
    __device__ __forceinline__ void stream(const GateNormArgs& a, long sample, int c)
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            factor[k] = 1.0f;
            shift[k] = 0.0f;
        }
        if (a.x_weight)
            load_cols<VEC, ODD>(a.x_weight, c, a.n, factor);
        if (a.scale) {
            float s[VEC];
            load_cols<VEC, ODD>(a.scale + sample * a.mod_stride, c, a.n, s);
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                factor[k] = fmaf(factor[k], s[k], factor[k]);
        }
        if (a.shift)
            load_cols<VEC, ODD>(a.shift + sample * a.mod_stride, c, a.n, shift);
    }
};

// A launch's arguments: a sample's blocks, the rows that runs start at (ODD: the first four of a sample, or as many as it has);
// out_whole: out's rows lie on the vectors' borders as x's do.
struct GateNormOf : GateNormArgs {
    unsigned blocks, starts;
    bool out_whole;
};

// A block a run of `run` rows of one sample, NC chunks of 32 * VEC values a warp and row. The vectors stay in shared memory from
// row to row and each row is loaded while the one before is worked on.
// ODD: rows that do not all begin on a vector's border, but x, y and x_out alike. Rows four apart begin alike, so a run takes
// every fourth row and all of it has one place in the vectors; the cut vectors at a row's ends go value by value.
// T: threads at most; up to 256 leave 85 registers each for three blocks an SM, the widest rows take an SM's for one block.
template <int VEC, int NC, bool ODD, int T>
__global__ void __launch_bounds__(T, NC * VEC <= 12 ? (T == 256 ? 3 : 2) : 1) k_gate_norm(const GateNormOf a, int run)
{
    __shared__ float red[2][5][16];
    grid_dep_wait();
    grid_dep_launch();
    constexpr int kApart = ODD ? 4 : 1;
    const unsigned part = blockIdx.x % a.blocks;
    const long sample = blockIdx.x / a.blocks;
    const long lo = sample * a.rows_per_sample + long(part / a.starts) * run * kApart + part % a.starts;
    const long hi = min(min(a.rows, (sample + 1) * a.rows_per_sample), lo + long(run) * kApart);
    const int n = a.n;
    const float inv_n = 1.0f / float(n);
    const Place<VEC, NC, ODD> at(ODD ? int((reinterpret_cast<uintptr_t>(a.x) / 4 + lo * a.ldx) & 3) : 0);
    extern __shared__ __align__(16) float kept[];  // [gate, factor, shift][ns], each thread its own places
    const int ns = ODD ? (n + 6) & ~3 : n;
    float* mine = kept + Place<VEC, NC>().first;
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (at.in(i, n)) {
            Vectors<VEC, ODD> v;
            v.branch(a, sample, at.at(i));
            v.stream(a, sample, at.at(i));
            store_row(mine + i * 32 * VEC, v.gate);
            store_row(mine + ns + i * 32 * VEC, v.factor);
            store_row(mine + 2 * ns + i * 32 * VEC, v.shift);
        }
    Raw<VEC> rx[NC], ry[NC];
    const auto load = [&](long row) {
        load_row_at(rx, a.x + row * a.ldx, at, n);
        if (a.y && a.y_f32)
            load_row_at(ry, static_cast<const float*>(a.y) + row * a.ldy, at, n);
        else if (a.y)
            load_row_at(ry, static_cast<const __nv_bfloat16*>(a.y) + row * a.ldy, at, n);
    };
    if (lo < hi)
        load(lo);
    int turn = 0;
    for (long row = lo; row < hi; row += kApart, turn ^= 1) {
        float x[NC][VEC], y[NC][VEC];
        values(rx, true, x);
        if (a.y)
            values(ry, a.y_f32, y);
        if (row + kApart < hi)
            load(row + kApart);
        if (a.y) {
            if (a.y_norm != kNormNone)
                normalise(y, at, a.y_norm, n, inv_n, a.eps, red[turn][0]);
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (at.in(i, n)) {
                    Vectors<VEC, ODD> v;
                    load_shared(mine + i * 32 * VEC, v.gate);
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        x[i][k] = fmaf(y[i][k], v.gate[k], x[i][k]);
                }
            store_row_at(x, a.x_out + row * a.ldxo, at, n);
        }
        if (a.out_type == kOutNone)
            continue;
        if (a.x_norm != kNormNone)
            normalise(x, at, a.x_norm, n, inv_n, a.eps, red[turn][2]);
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (at.in(i, n)) {
                Vectors<VEC, ODD> v;
                load_shared(mine + ns + i * 32 * VEC, v.factor);
                load_shared(mine + 2 * ns + i * 32 * VEC, v.shift);
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    x[i][k] = fmaf(x[i][k], v.factor[k], v.shift[k]);
            }
        if (a.out_type == kOutBf16)
            store_row_at(x, static_cast<__nv_bfloat16*>(a.out) + row * a.ldo, at, n, a.out_whole);
        else if (a.out_type == kOutF32)
            store_row_at(x, static_cast<float*>(a.out) + row * a.ldo, at, n, a.out_whole);
        else
            quant_row_at(x, static_cast<int8_t*>(a.out) + row * a.ldo, a.out_scale + row, at, n, red[turn][4], a.out_whole);
    }
}

// A block a row, NC chunks of 32 * VEC values a warp; WALK: every gridDim.x-th row, each loaded while the one before is worked
// on.
template <typename XT, int VEC, int NC, bool WALK>
__global__ void __launch_bounds__(512) k_quant_rows(const QuantRowsArgs a)
{
    __shared__ float red[2][16];
    grid_dep_wait();
    grid_dep_launch();
    const Place<VEC, NC> at;
    const XT* from = static_cast<const XT*>(a.x);
    Raw<VEC> r[NC];
    long row = blockIdx.x;
    load_row_at(r, from + row * a.ldx, at, a.n);
    for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
        float x[NC][VEC];
        values(r, sizeof(XT) == 4, x);
        if (WALK && row + gridDim.x < a.rows)
            load_row_at(r, from + (row + gridDim.x) * a.ldx, at, a.n);
        quant_row_at(x, a.q + row * a.ldq, a.scale + row, at, a.n, red[turn]);
        if (!WALK)
            return;
    }
}

// Rows too long for a block's registers: a pass for the step, a second one (out of L2) for the values.
template <typename XT>
__global__ void __launch_bounds__(512) k_quant_long(const QuantRowsArgs a)
{
    __shared__ float red[16];
    grid_dep_wait();
    grid_dep_launch();
    const long row = blockIdx.x;
    const XT* xr = static_cast<const XT*>(a.x) + row * a.ldx;
    int8_t* qr = a.q + row * a.ldq;
    float top = 0.0f;
    for (int c = threadIdx.x; c < a.n; c += blockDim.x)
        top = max_abs(top, float(xr[c]));
    const RowStep step(block_max_abs(top, red));
    if (threadIdx.x == 0)
        a.scale[row] = step.step;
    for (int c = threadIdx.x; c < a.n; c += blockDim.x)
        qr[c] = step.one(float(xr[c]));
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// How a row of `chunks` chunks is dealt out: NC chunks a warp (at most `most`) on up to 16 warps, with few idle chunk places.
// Among equals fewer warps where there are many rows (8704 x 3072 to int8: 60 us on 8 warps a row, 63 on 12; plain quantising
// 8192 x 3072: 15.5 us on 3 warps a row, 21 on 6 or 12), more where there are few, as that shortens a block's way from its
// loads to its stores (154 x 1280: 2.6 us on 10 warps a row, 3.2 on 5).
struct Deal {
    int nc, warps;
};
Deal deal(int chunks, int most, bool few_warps, int least = 1)
{
    Deal best{0, 0};
    for (int nc = least; nc <= most; ++nc) {
        const int warps = (chunks + nc - 1) / nc;
        const int more = best.nc ? warps * nc - best.warps * best.nc : -1;
        if (warps <= 16 && (more < 0 || (more == 0 && few_warps)))
            best = Deal{nc, warps};
    }
    return best;
}

template <int VEC, int NC, bool ODD, int T>
cudaError_t launch_gate_norm_of(GateNormOf& a, int warps, cudaStream_t st)
{
    constexpr int kApart = ODD ? 4 : 1;
    const long samples = (a.rows + a.rows_per_sample - 1) / a.rows_per_sample;
    const size_t smem = size_t(3) * (ODD ? (a.n + 6) & ~3 : a.n) * sizeof(float);
    if (smem > 47 * 1024) {  // with the reductions' places more than the 48 KB that need no leave
        static std::atomic<uint64_t> devs{0};
        const cudaError_t e =
            smem_limit_once(devs, k_gate_norm<VEC, NC, ODD, T>, 3 * kGateNormMaxWidth * int(sizeof(float)));
        if (e != cudaSuccess)
            return e;
    }
    // Runs as long as still leave one wave of resident blocks (two waves: 65 against 63 us at 8704 x 3072, three 69).
    const long apart = (a.rows_per_sample + kApart - 1) / kApart;
    int run = 1;
    if (a.rows > 2L * num_sms()) {
        int resident = 1;
        const cudaError_t e =
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, k_gate_norm<VEC, NC, ODD, T>, 32 * warps, smem);
        if (e != cudaSuccess)
            return e;
        const long wave = long(num_sms()) * std::max(1, resident);
        run = int(std::min(apart, std::max(1L, (a.rows + wave - 1) / wave)));
    }
    a.starts = unsigned(std::min(a.rows_per_sample, long(kApart)));
    a.blocks = unsigned((apart + run - 1) / run) * a.starts;
    return launch_k(k_gate_norm<VEC, NC, ODD, T>, dim3(unsigned(samples * a.blocks)), 32 * warps, smem, st, a, run);
}

template <int VEC, int NC, bool ODD = false>
cudaError_t launch_gate_norm(GateNormOf& a, int warps, cudaStream_t st)
{
    if constexpr (NC * VEC <= 12)
        if (warps <= 8)
            return launch_gate_norm_of<VEC, NC, ODD, 256>(a, warps, st);
    return launch_gate_norm_of<VEC, NC, ODD, 512>(a, warps, st);
}

template <bool ODD>
cudaError_t launch_gate_norm_by_four(GateNormOf& a, int chunks, cudaStream_t st)
{
    const bool many = a.rows > 2L * num_sms();
    // Rows with cut vectors: two chunks a warp at least where there are many (the warps with an end hold the others up at each
    // reduction: 4099 x 1283 20.8 us on 4 warps, 24.3 on 11).
    const Deal d = deal(chunks, chunks <= 48 ? 3 : 6, many, ODD && many ? 2 : 1);
    return d.nc == 1   ? launch_gate_norm<4, 1, ODD>(a, d.warps, st)
           : d.nc == 2 ? launch_gate_norm<4, 2, ODD>(a, d.warps, st)
           : d.nc == 3 ? launch_gate_norm<4, 3, ODD>(a, d.warps, st)
           : d.nc == 4 ? launch_gate_norm<4, 4, ODD>(a, d.warps, st)
           : d.nc == 5 ? launch_gate_norm<4, 5, ODD>(a, d.warps, st)
                       : launch_gate_norm<4, 6, ODD>(a, d.warps, st);
}

template <typename XT, int VEC, int NC>
cudaError_t walk_quant(const QuantRowsArgs& a, int warps, cudaStream_t st)
{
    long blocks = a.rows;
    if (blocks > num_sms()) {
        int resident = 1;
        const cudaError_t e =
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, k_quant_rows<XT, VEC, NC, true>, 32 * warps, 0);
        if (e != cudaSuccess)
            return e;
        blocks = std::min(blocks, long(num_sms()) * std::max(1, resident));
    }
    return launch_k(k_quant_rows<XT, VEC, NC, true>, dim3(unsigned(blocks)), 32 * warps, 0, st, a);
}

template <typename XT, int VEC, int NC>
cudaError_t launch_quant(const QuantRowsArgs& a, int warps, cudaStream_t st)
{
    // Blocks of one warp come too fast for the launch hardware, about one a ns (20000 x 640 bf16: a block a row 21.4 us, a wave
    // of walking blocks 9.8); wide blocks and single values gain from the next row's loads (8192 x 12288 bf16 60 against 57,
    // 4000 x 5001 37 against 29). In between a block a row evens out better (8192 x 3072 bf16 15.3 against 16.9).
    if constexpr (VEC == 1)
        return walk_quant<XT, VEC, NC>(a, warps, st);
    if (warps == 1 || warps >= 8)
        return walk_quant<XT, VEC, NC>(a, warps, st);
    return launch_k(k_quant_rows<XT, VEC, NC, false>, dim3(unsigned(a.rows)), 32 * warps, 0, st, a);
}

}  // namespace

cudaError_t gate_norm(const GateNormArgs& args, cudaStream_t st)
{
    if (args.rows == 0)
        return cudaSuccess;
    GateNormOf a{args, 0, 1, true};
    a.rows_per_sample = std::min(a.rows_per_sample, a.rows);
    // Vectors of four where every row and vector allows them; rows that begin off a border, but alike, cut their end vectors
    // (1916 x 2719 to int8 21 us, value by value 31; 4803 x 5111 90 against 100); rows that begin differently go by value.
    const size_t yb = a.y_f32 ? 16 : 8, ob = a.out_type == kOutBf16 ? 8 : a.out_type == kOutF32 ? 16 : 4;
    const bool vec = a.n % 4 == 0 && aligned(a.x, 16) && a.ldx % 4 == 0 &&
                     (!a.y || (aligned(a.y, yb) && a.ldy % 4 == 0 && aligned(a.x_out, 16) && a.ldxo % 4 == 0)) &&
                     aligned(a.y_weight, 16) && aligned(a.gate, 16) && a.gate_stride % 4 == 0 &&
                     aligned(a.x_weight, 16) && aligned(a.scale, 16) && aligned(a.shift, 16) &&
                     a.mod_stride % 4 == 0 && (a.out_type == kOutNone || (aligned(a.out, ob) && a.ldo % 4 == 0));
    const auto as_x = [&](const void* p, size_t bytes, long ld) {
        return ((reinterpret_cast<uintptr_t>(p) / bytes ^ reinterpret_cast<uintptr_t>(a.x) / 4) & 3) == 0 && (ld - a.ldx) % 4 == 0;
    };
    a.out_whole = a.out_type == kOutNone || as_x(a.out, ob / 4, a.ldo);
    cudaError_t e;
    if (vec)
        e = launch_gate_norm_by_four<false>(a, (a.n + 127) / 128, st);
    else if (a.n + 3 <= kGateNormMaxWidth && (!a.y || (as_x(a.y, yb / 4, a.ldy) && as_x(a.x_out, 4, a.ldxo))))
        e = launch_gate_norm_by_four<true>(a, (a.n + 3 + 127) / 128, st);
    else if (a.n <= 4096)
        e = launch_gate_norm<1, 8>(a, (a.n + 255) / 256, st);
    else
        e = launch_gate_norm<1, 24>(a, (a.n + 767) / 768, st);
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

cudaError_t quantize_rows(const QuantRowsArgs& a, cudaStream_t st)
{
    if (a.rows == 0)
        return cudaSuccess;
    const int v = a.x_f32 ? 4 : 8;
    const bool vec = a.n % v == 0 && aligned(a.x, 16) && a.ldx % v == 0 && aligned(a.q, v) && a.ldq % v == 0;
    const int chunks = (a.n + 32 * (vec ? v : 1) - 1) / (32 * (vec ? v : 1));
    cudaError_t e;
    if (a.n > 16384 || (!vec && chunks > 16 * 32)) {
        e = a.x_f32 ? launch_k(k_quant_long<float>, dim3(unsigned(a.rows)), 512, 0, st, a)
                    : launch_k(k_quant_long<__nv_bfloat16>, dim3(unsigned(a.rows)), 512, 0, st, a);
    } else if (!vec) {
        if (a.x_f32)
            e = chunks <= 128 ? launch_quant<float, 1, 8>(a, (chunks + 7) / 8, st)
                              : launch_quant<float, 1, 32>(a, (chunks + 31) / 32, st);
        else
            e = chunks <= 128 ? launch_quant<__nv_bfloat16, 1, 8>(a, (chunks + 7) / 8, st)
                              : launch_quant<__nv_bfloat16, 1, 32>(a, (chunks + 31) / 32, st);
    } else if (a.x_f32) {
        const Deal d = deal(chunks, chunks <= 64 ? 4 : 8, true);
        e = d.nc == 1   ? launch_quant<float, 4, 1>(a, d.warps, st)
            : d.nc == 2 ? launch_quant<float, 4, 2>(a, d.warps, st)
            : d.nc == 3 ? launch_quant<float, 4, 3>(a, d.warps, st)
            : d.nc == 4 ? launch_quant<float, 4, 4>(a, d.warps, st)
            : d.nc <= 6 ? launch_quant<float, 4, 6>(a, (chunks + 5) / 6, st)
                        : launch_quant<float, 4, 8>(a, (chunks + 7) / 8, st);
    } else {
        const Deal d = deal(chunks, 4, true);
        e = d.nc == 1   ? launch_quant<__nv_bfloat16, 8, 1>(a, d.warps, st)
            : d.nc == 2 ? launch_quant<__nv_bfloat16, 8, 2>(a, d.warps, st)
            : d.nc == 3 ? launch_quant<__nv_bfloat16, 8, 3>(a, d.warps, st)
                        : launch_quant<__nv_bfloat16, 8, 4>(a, d.warps, st);
    }
    if (e != cudaSuccess)
        return e;
    count_launch();
    return cudaGetLastError();
}

}  // namespace mkb
