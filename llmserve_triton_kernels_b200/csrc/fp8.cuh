// Numbers in 8 bits (e4m3: sign, 4 bits of exponent, 3 of mantissa, largest 448, no infinities) with a power of two for a
// block of them.
//
// The scale of a block is 2^e for the smallest e with max|x| <= 448 * 2^e, so that the largest value lies in (224, 448] and
// dividing by the scale is exact: the rounding to e4m3 is the only rounding there is.  Scales that fill the range to its last
// bit (max|x| / 448) would be rounded themselves, and so would the quotient; e4m3 being a floating format, they buy no
// precision but for values some 2^-15 below the block's largest.
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace fp8 {

// Bits of |v|, 0 for infinities and NaN: they do not enter a block's scale.
__device__ __forceinline__ unsigned finite_bits(float v) {
    const unsigned b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// The scale's biased exponent e + 127 from the bits of the block's largest |x| (0: a block of zeros, scale 1).  448 is
// 1.75 * 2^8: a mantissa above 1.75 needs the next power.  e >= -126, so that scales are normal numbers.
__device__ __forceinline__ unsigned scale_exponent(unsigned bits) {
    if (bits == 0u) return 127u;
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (unsigned)max(e, 1);
}
__device__ __forceinline__ float power(unsigned biased) { return __uint_as_float(biased << 23); }
__device__ __forceinline__ float inverse(unsigned biased) { return __uint_as_float((254u - biased) << 23); }

// Two values times the scale's inverse, rounded to e4m3 (the first in the low byte).  v * 0 + v is v, and NaN for an infinity:
// what was not finite is NaN in 8 bits too.
__device__ __forceinline__ unsigned short pack2(float a, float b, float inv) {
    return __nv_cvt_float2_to_fp8x2(make_float2(fmaf(a, 0.f, a) * inv, fmaf(b, 0.f, b) * inv), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d, float inv) {
    return (unsigned)pack2(a, b, inv) | ((unsigned)pack2(c, d, inv) << 16);
}

}  // namespace fp8
