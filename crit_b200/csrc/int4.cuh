// The 4-bit page format ("int4"): a row of one kv head is dim codes, two a byte (element 2 i in the low half of byte i),
// and a byte of scale for each group of 32 elements.
//
// The byte is an unsigned float of 5 exponent and 3 mantissa bits, the bits 14..7 of an FP16 number, so `byte << 7` IS the
// scale as FP16: up to 61,440, steps of 2^-17 below 2^-14, a NaN at 0xff.  With s the float nearest to max |x| / 7 (half to
// even, 61,440 at most), code = 8 + clamp(rint(x / s), -7, 7), 8 where s is 0; a group that holds a NaN has scale 0xff and
// codes of 8.  A code stands for (code - 8) * s.  From 2^-14 up s is at most 1/16 below max |x| / 7 and 7 * 17 / 16 < 7.5, so
// below the saturation no element is further than s / 2 from its code's value (below 2^-14: than s / 2 or 7 * 2^-18).
//
// Why such scales: the product of a code of 4 bits and a scale of 4 significant bits has at most 8 of them, so bf16 and
// FP16 hold every value as it is (FP16 up to its range) and 16-bit tensor-core tiles can read it with no second rounding;
// and a row of 128 is 68 bytes, where an FP16 scale a group would make it 72.
#pragma once

#include "common.cuh"

namespace crit_b200 {

constexpr int INT4_GROUP = 32;

// max |x| of a group -> the byte of its scale.
__device__ __forceinline__ uint32_t int4_scale_byte(float amax, bool nan) {
    if (nan) return 0xffu;
    const float s = __fdiv_rn(amax, 7.f);
    if (s < 0x1p-14f) return (uint32_t)__float2int_rn(s * 0x1p17f);                // subnormal: steps of 2^-17 (8 is 2^-14)
    const uint32_t u = __float_as_uint(s);
    const uint32_t byte = ((u + 0x7ffffu + ((u >> 20) & 1u)) >> 20) - ((127u - 15u) << 3);
    return byte < 0xf7u ? byte : 0xf7u;
}

__device__ __forceinline__ float int4_scale(uint32_t byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }

// Eight elements of one group -> eight codes, element i in bits 4 i: rint(x / s), ties to even.  x is brought within 7 s first
// (exact: s has 4 significant bits).  The quotient is Markstein's: with r the reciprocal of s rounded to nearest, q = x r is
// corrected once by its remainder x - q s, exact in one FMA, and q + (x - q s) r is then x / s rounded to nearest, so that
// quotients half way between two codes, common where x has few bits, come out half way.  Adding 3 * 2^22 + 8 rounds to a
// whole number and leaves the code in the low bits.
__device__ __forceinline__ uint32_t int4_codes(const float (&x)[8], float s) {
    if (!(s > 0.f)) return 0x88888888u;                    // 0, or a NaN
    const float r = __frcp_rn(s), top = 7.f * s;
    uint32_t w = 0u;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float y = fminf(fmaxf(x[i], -top), top);
        const float q = __fmul_rn(y, r);
        const float n = __fmaf_rn(__fmaf_rn(-q, s, y), r, q);
        w = (w << 4) | (__float_as_uint(__fadd_rn(n, 12582920.f)) & 15u);
    }
    return w;
}

// The four lanes that hold a group (8 elements each, lanes 4 k .. 4 k + 3) agree on its scale byte; the lane's code word.
__device__ __forceinline__ uint32_t int4_quantise(const float (&x)[8], uint32_t& byte) {
    float amax = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        nan |= x[i] != x[i];
        amax = fmaxf(amax, fabsf(x[i]));
    }
    if (nan) amax = __int_as_float(0x7fffffff);        // passed on by the integer maximum below: a NaN is above infinity
    int bits = __float_as_int(amax);                    // (not negative: their order as integers is the floats')
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
    byte = int4_scale_byte(__int_as_float(bits), bits > 0x7f800000);
    return int4_codes(x, int4_scale(byte));
}

}  // namespace crit_b200
