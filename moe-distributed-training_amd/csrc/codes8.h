// Values in 8 bits, as rows (int8_rows.hip) and blocks (swiglu8.hip) of them are coded: codes rne(127 v / a), a the largest magnitude that shares the scale a / 127.
#pragma once
#include "common.h"

namespace {

// Magnitudes are compared as bits: those of an infinity lie above every number's, and NaN's above those.
constexpr uint32_t NOT_FINITE = 0x7f800000u;
__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// What turns values of a row into its codes.  f: what the values are multiplied by first, so that 127 v and 127 / a stay inside fp32's range (a value that the
// factor makes subnormal is far below half a step).
struct RowCoder {
    float f, a, a_lo, inv, scale;
    __device__ __forceinline__ RowCoder(uint32_t top, float top_lo = 0.f)
    {
        const float amax = __uint_as_float(top);
        const bool fine = top < NOT_FINITE;
        f = amax > 0x1p64f ? 0x1p-64f : amax < 0x1p-64f ? 0x1p64f : 1.f;
        a = fine ? amax * f : 0.f;
        a_lo = fine ? top_lo * f : 0.f;
        inv = a > 0.f ? 127.f / a : 0.f;
        if (inv == 0.f) f = 0.f;   // every code 0
        scale = fine ? amax / 127.f : __uint_as_float(0x7fc00000u);
    }
    // The code of v + lo, lo the rounding error of v.  v times 127 / a is off by five roundings, 127 * 5 * 2^-24 < 4e-5 of a step: only beside a border does more matter.
    __device__ __forceinline__ float code(float v, float lo) const
    {
        const float t = f == 0.f ? 0.f : v * f * inv, q = rintf(t);
        return fabsf(t - q) > 0.49995f ? exact(v, lo) : q;
    }
    __device__ __forceinline__ float exact(float v, float lo) const
    {
        v = f == 0.f ? 0.f : v * f;
        lo = f == 0.f ? 0.f : lo * f;
        float q = rintf(v * inv);
        const float t = 127.f * v, te = fmaf(127.f, v, -t) + 127.f * lo - q * a_lo, r = fmaf(-q, a, t);
        const float side = copysignf(1.f, r), d = fmaf(2.f, fabsf(r), -a) + (2.f * side * te - a_lo);   // twice the distance to q, minus a step
        if (d > 0.f || (d == 0.f && a > 0.f && ((int)q & 1))) q += side;
        return q;
    }
    // ... of a value that carries fp32 rounding anyway
    __device__ __forceinline__ float nearest(float v) const { return f == 0.f ? 0.f : rintf(v * f * inv); }
};

// four whole numbers of magnitude 127 at most as bytes: 1.5 * 2^23 more, and they stand in the lowest bits
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d)
{
    constexpr float M = 12582912.f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + M), __float_as_uint(a + M), 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d + M), __float_as_uint(c + M), 0x04000c0cu);
    return ab | cd;
}

}  // namespace
