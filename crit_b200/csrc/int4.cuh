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
    const float q = __fmul_rn(amax, 1.f / 7.f);
    const float s = amax > 0x1p-100f && amax < 0x1p100f ? __fmaf_rn(__fmaf_rn(-q, 7.f, amax), 1.f / 7.f, q) : q;      // amax / 7 to nearest (Markstein)
    if (s < 0x1p-14f) return (uint32_t)__float2int_rn(s * 0x1p17f);                // subnormal: steps of 2^-17 (8 is 2^-14)
    const uint32_t u = __float_as_uint(s);
    const uint32_t byte = ((u + 0x7ffffu + ((u >> 20) & 1u)) >> 20) - ((127u - 15u) << 3);
    return byte < 0xf7u ? byte : 0xf7u;
}

__device__ __forceinline__ float int4_scale(uint32_t byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }

// Two FP32 numbers in a register pair, worked on together.
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void one_each(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// The reciprocal of a scale, to nearest: the hardware's approximation corrected once by its error 1 - s r, exact in one FMA
// (Markstein; s has 4 significant bits, none of the mantissas the step fails for).
__device__ __forceinline__ float int4_reciprocal(float s) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return __fmaf_rn(__fmaf_rn(-s, r, 1.f), r, r);
}

// Eight elements of one group -> eight codes, element i in bits 4 i: rint(x / s), ties to even.  x is brought within 7 s first
// (exact: s has 4 significant bits) where the scale is one that max |x| / 7 may be far above.  The quotient is Markstein's:
// with r the reciprocal of s rounded to nearest, q = x r is corrected once by its remainder x - q s, exact in one FMA, and
// q + (x - q s) r is then x / s rounded to nearest, so that quotients half way between two codes, common where x has few
// bits, come out half way.  Adding 3 * 2^22 + 8 rounds to a whole number, whose bits are 0x4b400000 + the code; the word is
// their sum in base 16 less the constants'.
__device__ __forceinline__ uint32_t int4_codes(float (&x)[8], float s, uint32_t byte) {
    if (!(s > 0.f)) return 0x88888888u;                    // 0, or a NaN
    const float r = int4_reciprocal(s);
    if (byte < 8u || byte == 0xf7u) {                       // (else |x| / s is below 7.5)
        const float top = 7.f * s;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -top), top);
    }
    const uint64_t r2 = two(r, r), s2 = two(-s, -s), magic = two(12582920.f, 12582920.f);
    uint32_t bits[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t y = two(x[i], x[i + 1]), q = mul2(y, r2);
        float a, b;
        one_each(add2(fma2(fma2(q, s2, y), r2, q), magic), a, b);
        bits[i] = __float_as_uint(a), bits[i + 1] = __float_as_uint(b);
    }
    uint32_t w = bits[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) w = w * 16u + bits[i];
    return w - 0x4b400000u * 0x11111111u;
}

// Eight codes -> what they stand for (exact in FP32): a code in the low bits of 2^23 is 2^23 + code as a float.
__device__ __forceinline__ void int4_values(uint32_t codes, float s, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(__fadd_rn(__uint_as_float(0x4b000000u | ((codes >> (4 * i)) & 15u)), -8388616.f), s);
}

// max |x| of eight elements, its bits: their order as integers is the floats', a NaN above infinity.
__device__ __forceinline__ int int4_top(const float (&x)[8]) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(fabsf(x[i])));
    return __float_as_int(amax) & 0x7fffffff;
}

// The four lanes that hold a group (8 elements each, lanes 4 k .. 4 k + 3) agree on its scale byte; the lane's code word.
__device__ __forceinline__ uint32_t int4_quantise(float (&x)[8], uint32_t& byte) {
    int bits = int4_top(x);
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
    byte = int4_scale_byte(__int_as_float(bits), bits > 0x7f800000);
    return int4_codes(x, int4_scale(byte), byte);
}

}  // namespace crit_b200
