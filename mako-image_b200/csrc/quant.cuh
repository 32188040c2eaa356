// Symmetric 8-bit rows: a row's step is amax / 127 (one IEEE fp32 division) and its values are x / step rounded to the
// nearest whole number, ties to even, decided exactly.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

namespace mkb {

// Row steps below the smallest normal number are taken as 0 (the row's values all become 0): 1 / step stays finite.
constexpr float kMinStep = 1.17549435e-38f;

// The larger magnitude, or NaN where there is one.
__device__ __forceinline__ float max_abs(float m, float x)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}

struct RowStep {
    static constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, ties to even
    float step, inv;
    __device__ __forceinline__ explicit RowStep(float amax)
    {
        step = amax <= 3.4028235e38f ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fffffffu);
        if (step < kMinStep)
            step = 0.0f;
        // A row of zeros, or one with an infinity or a NaN in it (step NaN), has only zeros.
        inv = step > 0.0f ? 1.0f / step : 0.0f;
    }
    // x / step to the nearest whole number, ties to even, as the low byte of each result's bits. x * inv is off by a few
    // roundings, so its nearest whole number may be one off next to a border of two; the remainder x - q step decides. It is
    // a multiple of the smaller of the two numbers' last places and no larger than about step / 2, so the fused
    // multiply-add gives it without rounding. Twice the remainder is set against the step: below 2^-125 half a step may be no
    // fp32 number.
    template <int N>
    __device__ __forceinline__ void whole(const float (&x)[N], float (&t)[N]) const
    {
        float far = -1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            t[i] = fmaf(x[i], inv, kRound);
            far = fmaxf(far, fmaf(2.0f, fabsf(fmaf(kRound - t[i], step, x[i])), -step));
        }
        if (far >= 0.0f) {  // on or beyond a border: rare
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float r = fmaf(kRound - t[i], step, x[i]), over = fmaf(2.0f, fabsf(r), -step);
                if (over > 0.0f || (over == 0.0f && (__float_as_int(t[i]) & 1)))
                    t[i] += copysignf(1.0f, r);
            }
        }
    }
    __device__ __forceinline__ uint32_t pack4(const float (&x)[4]) const
    {
        if (!(inv > 0.0f))
            return 0;
        float t[4];
        whole(x, t);
        const uint32_t lo = __byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040);
        return __byte_perm(lo, hi, 0x5410);
    }
    __device__ __forceinline__ int8_t one(float x) const
    {
        if (!(inv > 0.0f))
            return 0;
        const float v[1] = {x};
        float t[1];
        whole(v, t);
        return int8_t(__float_as_uint(t[0]) & 0xff);
    }
};

}  // namespace mkb
