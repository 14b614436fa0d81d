// The 8-bit cache: e4m3 codes in pages, one power-of-two scale for each page and kv head.
//
// value = code * scale.  A power of two as the scale means that x / scale is exact, so a
// value is rounded once, by the conversion, and that a code moves to a greater scale without
// a further rounding unless it becomes subnormal there.  The greatest code of a page lies
// in (224, 448] and the least normal one is 2^-6: values down to between 2^-13.8 and 2^-14.8
// of the page's greatest keep 3 bits behind the leading one (off by at most 2^-4 of themselves),
// smaller ones are off by at most 2^-10 * scale.  Against a scale that takes the greatest to 448 itself
// a power of two costs nothing above and at most one binade there.
#pragma once
#include "common.cuh"

// The smallest 2^e, e >= -126, with 448 * 2^e >= amax (finite, >= 0): amax = 1.m * 2^E fits
// 448 = 1.75 * 2^8 at e = E - 8 if 1.m <= 1.75, else at E - 7.
__device__ __forceinline__ float e4m3_scale(float amax) {
    const unsigned b = __float_as_uint(amax);
    const int E = (int)(b >> 23) - 127;
    const int e = max(E - ((b & 0x7fffffu) <= 0x600000u ? 8 : 7), -126);
    return __uint_as_float((unsigned)(e + 127) << 23);
}
// 1 / scale of a power of two 2^e, -126 <= e <= 126
__device__ __forceinline__ float e4m3_inverse(float scale) {
    return __uint_as_float((254u << 23) - __float_as_uint(scale));
}
// |x| as it counts for a scale: 0 where x is not finite
__device__ __forceinline__ float e4m3_magnitude(float x) {
    const unsigned b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? __uint_as_float(b) : 0.f;
}
// Two codes, a in the low byte: nearest, ties to even; what is not finite becomes NaN (the
// conversion alone would saturate an infinity).
__device__ __forceinline__ unsigned e4m3_pair(float a, float b) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    unsigned v = r;
    if ((__float_as_uint(a) & 0x7fffffffu) >= 0x7f800000u) v |= 0x007fu;
    if ((__float_as_uint(b) & 0x7fffffffu) >= 0x7f800000u) v |= 0x7f00u;
    return v;
}
// Two codes (the low 16 bits) as two half floats: exact, NaN stays NaN.
__device__ __forceinline__ unsigned e4m3_to_half2(unsigned codes) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)codes));
    return r;
}
__device__ __forceinline__ float2 e4m3_to_float2(unsigned codes) {
    const unsigned h = e4m3_to_half2(codes);
    float lo, hi;
    asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.f32.f16 %0, a;\n cvt.f32.f16 %1, b;}"
        : "=f"(lo), "=f"(hi) : "r"(h));
    return make_float2(lo, hi);
}
// Four codes as two pairs of half floats.
__device__ __forceinline__ void e4m3_word(unsigned codes, unsigned& lo, unsigned& hi) {
    asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;}"
        : "=r"(lo), "=r"(hi) : "r"(codes));
}
