// 8-bit codes of the quantised K/V cache: what a code stands for, scales, and rounding to codes.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace oxi {

// The scale of a block whose largest magnitude is amax.  int8: amax / 127.  e4m3: the power of two s with
// amax / s in (224, 448], so that moving stored codes to a larger scale only changes their exponents.
template <uint32_t kFmt>
__device__ __forceinline__ float q8_scale(float amax) {
    if (kFmt == Q8_INT8) return __fdiv_rn(amax, 127.0f);
    if (!(amax > 0.0f)) return 0.0f;
    const uint32_t u = __float_as_uint(__fdiv_rn(amax, 448.0f));
    const uint32_t e = (u >> 23) + ((u & 0x7fffffu) ? 1u : 0u);
    return __uint_as_float((e < 1u ? 1u : e) << 23);
}

// One code (as a byte) for x at scale s > 0; ties to even, saturating.
template <uint32_t kFmt>
__device__ __forceinline__ uint32_t q8_code(float x, float s) {
    const float y = __fdiv_rn(x, s);
    if (kFmt == Q8_INT8) {
        const int c = __float2int_rn(y);
        return (uint32_t)min(127, max(-127, c)) & 0xffu;
    }
    return (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

template <uint32_t kFmt>
__device__ __forceinline__ float q8_value(uint32_t code) {
    if (kFmt == Q8_INT8) return (float)(int8_t)(uint8_t)code;
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}

}  // namespace oxi
