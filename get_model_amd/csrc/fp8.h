// e4m3 values with one power-of-two scale per block of 128 (rmsnorm.hip leaves them, gemm_fp8.hip multiplies them).
#pragma once
#include "common.h"

// biased exponent of the smallest power of two 2^e with |amax| <= 448 * 2^e (448 = 1.75 * 2^8); 127 (scale 1) for an all-zero
// block and for one that holds an infinity or a NaN, which has no scale: its 128 values all become NaN.
__device__ __forceinline__ unsigned scale_byte(unsigned amax) {
    const int b = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (amax == 0u || amax >= 0x7f800000u) ? 127u : (unsigned)max(b, 1);
}
__device__ __forceinline__ float inv_scale(unsigned byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ unsigned pack4fp8(float a, float b, float c, float d, float inv, bool finite) {
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, v, true);
    return finite ? (unsigned)v : 0x7f7f7f7fu;
}
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
