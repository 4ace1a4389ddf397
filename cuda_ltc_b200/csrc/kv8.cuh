// What the kernels of the 8-bit key/value cache share: the e4m3 conversions, power-of-two scales, and their arguments.
#pragma once

#include <cuda_fp16.h>
#include <math.h>

#include <type_traits>

#include "host_common.h"
#include "sm100_ptx.cuh"

namespace ltca {

// Two values to e4m3, to nearest with ties to even, saturating at +-448 (NaN stays NaN); a in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
// Two codes to fp16, which holds every e4m3 value; the low byte's value in the low half.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t codes) {
    const uint32_t h = e4m3x2_to_half2(codes);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// |x| where it is finite, else 0: as bits, whose order is that of the values.
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
// The exponent e of the smallest power of two, from 2^-100 on, by which amax (as bits) comes down to top * 2^k, where `top`
// (its mantissa bits given) lies in [1, 2): an fp32 mantissa above top's asks for one power more.
__device__ __forceinline__ int pow2_exponent(uint32_t amax_bits, int k, uint32_t top_mantissa, int e_max) {
    const int e = (int)(amax_bits >> 23) - 127 - k + ((amax_bits & 0x7fffffu) > top_mantissa ? 1 : 0);
    return min(max(e, -100), e_max);
}
// 448 = 1.75 * 2^8
__device__ __forceinline__ int e4m3_exponent(uint32_t amax_bits) { return pow2_exponent(amax_bits, 8, 0x600000u, 120); }
// 127 = 1.984375 * 2^6
__device__ __forceinline__ int int8_exponent(uint32_t amax_bits) { return pow2_exponent(amax_bits, 6, 0x7e0000u, 121); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 .. 127

__device__ __forceinline__ float ld_value(const float* p) { return *p; }
__device__ __forceinline__ float ld_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void st_value(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Tokens of sequence b that are new, and how many it has with them (the latter not yet cut to the capacity).
__device__ __forceinline__ int new_tokens(const int32_t* new_len, int b, int n) {
    return new_len ? min(max(new_len[b], 0), n) : n;
}

}  // namespace ltca
