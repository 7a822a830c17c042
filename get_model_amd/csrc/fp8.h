// e4m3 values with one power-of-two scale per block of 128 (rmsnorm.hip leaves them, gemm_fp8.hip multiplies them).
#pragma once
#include "common.h"

// biased exponent of the smallest power of two 2^e with |amax| <= 448 * 2^e (448 = 1.75 * 2^8); 127 (scale 1) for an all-zero
// block and for one that holds an infinity or a NaN, which has no scale: its 128 values all become NaN.
__device__ __forceinline__ unsigned scale_byte(unsigned amax) {
    const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (amax == 0u || amax >= 0x7f800000u) ? 127u : (unsigned)max(b, 1);
}
__device__ __forceinline__ float scale_value(unsigned byte) { return __uint_as_float(byte << 23); }
// The conversion divides by the scale itself and rounds once (every float with the smallest scale that fits and the 20 next ones: the
// bytes of a product with 1 / scale and a plain conversion).
typedef __attribute__((ext_vector_type(2))) short fp8x4;
__device__ __forceinline__ unsigned pack4fp8(float a, float b, float c, float d, float scale, bool finite) {
    fp8x4 v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(fp8x4{0, 0}, a, b, scale, false);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(v, c, d, scale, true);
    return finite ? __builtin_bit_cast(unsigned, v) : 0x7f7f7f7fu;
}
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The same from bf16 pairs as they lie in memory: running maximum of both halves' magnitudes, its fp32 bit pattern, and four values
// (all 65536 with every scale they fit: the bytes of pack4fp8).
__device__ __forceinline__ unsigned max_abs_bf16(unsigned m, unsigned pair) {
    typedef __attribute__((ext_vector_type(2))) unsigned short us2;
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(us2, m), __builtin_bit_cast(us2, pair & 0x7fff7fffu)));
}
__device__ __forceinline__ unsigned abs_bits_bf16(unsigned m) { return max(m << 16, m & 0xffff0000u); }
__device__ __forceinline__ unsigned pack4fp8_bf16(unsigned ab, unsigned cd, float scale, bool finite) {
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    fp8x4 v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(fp8x4{0, 0}, __builtin_bit_cast(b2, ab), scale, false);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(b2, cd), scale, true);
    return finite ? __builtin_bit_cast(unsigned, v) : 0x7f7f7f7fu;
}
