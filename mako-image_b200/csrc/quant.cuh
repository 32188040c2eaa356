// Symmetric 8-bit rows: a row's step is amax / 127 (one IEEE fp32 division) and its values are x / step rounded to the
// nearest whole number, ties to even, decided exactly.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

namespace mkb {

// Row steps below the smallest normal number are taken as 0 (the row's values all become 0): 1 / step stays finite.
constexpr float kMinStep = 1.17549435e-38f;

// |x| as an ordered integer: a maximum over these bits keeps infinities and NaN, which fmaxf would drop.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct RowStep {
    float step, inv, half;
    __device__ __forceinline__ explicit RowStep(uint32_t amax_bits)
    {
        const float amax = __uint_as_float(amax_bits);
        step = amax_bits >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __fdiv_rn(amax, 127.0f);
        if (step < kMinStep)
            step = 0.0f;
        // A row of zeros, or one with an infinity or a NaN in it (step NaN), has only zeros.
        inv = step > 0.0f ? 1.0f / step : 0.0f;
        half = 0.5f * step;
    }
    // x / step to the nearest whole number, ties to even. rint(x * inv) may be one off next to a border of two whole
    // numbers; the remainder x - q step decides. It is a multiple of the smaller of the two numbers' last places and no
    // larger than about step / 2, so the fused multiply-add gives it without rounding.
    __device__ __forceinline__ int operator()(float x) const
    {
        if (inv == 0.0f)
            return 0;
        float q = rintf(x * inv);
        const float r = fmaf(-q, step, x), d = fabsf(r) - half;
        if (d > 0.0f || (d == 0.0f && (int(q) & 1)))
            q += copysignf(1.0f, r);
        return int(q);
    }
};

__device__ __forceinline__ uint32_t pack4_i8(int a, int b, int c, int d)
{
    return (uint32_t(a) & 0xff) | (uint32_t(b) & 0xff) << 8 | (uint32_t(c) & 0xff) << 16 | uint32_t(d) << 24;
}

}  // namespace mkb
