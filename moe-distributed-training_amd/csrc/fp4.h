// Weights in 4 bits: codes of one sign, two exponent and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even input in the lower half, times a power
// of two for each 32 consecutive inputs of an output column, held as its biased exponent (255: NaN).  The hardware turns a byte of codes and a scale into a pair of 16-bit
// or 32-bit numbers in one instruction.  A code has two significant bits, so the 16-bit weight is exact wherever its exponent fits: in bf16 always (subnormals included), in fp16
// for scales from 2^-23 to 2^13; beyond them fp16 rounds, or overflows to infinity, as the conversion of the weight itself would.
#pragma once
#include "common.h"

constexpr int FP4_GROUP = 32;         // inputs that share a scale
constexpr int FP4_GROUP_BYTES = 16;   // their codes

typedef uint32_t fp4_u32x4_t __attribute__((ext_vector_type(4)));

// a scale byte as the fp32 number whose exponent the conversions read (0 stands for 2^-127, 255 for NaN)
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// byte SEL of src -> its pair of weights, the lower code first
template <class Num, int SEL> __device__ __forceinline__ uint32_t fp4_pair(uint32_t src, float scale)
{
    if constexpr (Num::dtype == MOE_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(src, scale, SEL));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(src, scale, SEL));
}
// eight codes of one scale -> a lane's 16 bytes of a matrix operand
template <class Num> __device__ __forceinline__ bf16x8_t fp4_expand8(uint32_t src, float scale)
{
    const fp4_u32x4_t v = {fp4_pair<Num, 0>(src, scale), fp4_pair<Num, 1>(src, scale), fp4_pair<Num, 2>(src, scale), fp4_pair<Num, 3>(src, scale)};
    return __builtin_bit_cast(bf16x8_t, v);
}
template <int SEL> __device__ __forceinline__ float2 fp4_pair_f32(uint32_t src, float scale)
{
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(src, scale, SEL);
    return make_float2(v[0], v[1]);
}
