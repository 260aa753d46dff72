// Numbers in 8 bits (e4m3: sign, 4 bits of exponent, 3 of mantissa, largest 448, no infinities) with a power of two for a
// block of them.
//
// The scale of a block is 2^e for the smallest e with max|x| <= 448 * 2^e, so that the largest value lies in (224, 448] and
// dividing by the scale is exact: the rounding to e4m3 is the only rounding there is.  Scales that fill the range to its last
// bit (max|x| / 448) would be rounded themselves, and so would the quotient; e4m3 being a floating format, they buy no
// precision but for values some 2^-15 below the block's largest.
#pragma once

#include "common.cuh"

#include <cuda_fp16.h>
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

// The two numbers of a pair (the first in the low byte); by way of half precision, which holds every e4m3 number.
__device__ __forceinline__ float2 unpack2(unsigned short v) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(v, __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Eight consecutive values, 16-byte aligned.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    const unsigned w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const unsigned*>(&a);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}

// Two values times the scale's inverse, rounded to e4m3 (the first in the low byte).  v * 0 + v is v, and NaN for an infinity:
// what was not finite is NaN in 8 bits too.
__device__ __forceinline__ unsigned short pack2(float a, float b, float inv) {
    return __nv_cvt_float2_to_fp8x2(make_float2(fmaf(a, 0.f, a) * inv, fmaf(b, 0.f, b) * inv), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d, float inv) {
    return (unsigned)pack2(a, b, inv) | ((unsigned)pack2(c, d, inv) << 16);
}

}  // namespace fp8
