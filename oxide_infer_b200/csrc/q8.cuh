// 8-bit codes of the quantised K/V cache: what a code stands for, scales, and rounding to codes.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace oxi {

// V scales enter the exponents of the softmax as their log2 and leave the row sum as 1 / scale; a smaller scale, that of a block of
// zeros for one, counts as 2^-40.  Its values stay below 448 * 2^-40 < 2^-31, which an f16 result does not show (the smallest
// f16 has a scale of 2^-32), and the weights of its tokens, which the row sum needs, do not fall out of f32: with 2^-100 in its
// place a token of a zero block beside values of 3e4 got the weight 0 from e^-12 of the largest on, and 4,095 of them were
// missing from a row's sum (1 % of it).
constexpr float Q8_V_SCALE_MIN_LOG2 = -40.0f;

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

// What values are multiplied with before they are rounded to codes: 1 / scale, exact for e4m3; for int8 the quotient
// x / s is off by up to 2^-22 of itself, i.e. a value within 2^-15 of a step from a tie may go to the other side.
template <uint32_t kFmt>
__device__ __forceinline__ float q8_inverse(float scale) {
    return scale > 0.0f ? fminf(__fdiv_rn(1.0f, scale), 3.0e38f) : 0.0f;
}
// Codes of a (low byte) and b at inv = q8_inverse of a scale that covers them.
template <uint32_t kFmt>
__device__ __forceinline__ uint32_t q8_codes2(float a, float b, float inv) {
    if (kFmt == Q8_INT8) return (uint32_t)(__float2int_rn(a * inv) & 0xff) | ((uint32_t)(__float2int_rn(b * inv) & 0xff) << 8);
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
}

// the four codes of w as two f16 pairs, exact
template <uint32_t kFmt>
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (kFmt == Q8_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    } else {
        // c + 128 as the low bits of the f16 1024 + (c + 128), minus 1152
        const uint32_t u = w ^ 0x80808080u;
        const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), k), y = __hsub2(*reinterpret_cast<__half2*>(&b), k);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}

// The four codes of w moved to a scale that is 1 / ratio times theirs.  e4m3: ratio is a power of two (or 0), the f16 product
// is exact wherever its code is not 0.
template <uint32_t kFmt>
__device__ __forceinline__ uint32_t q8_moved(uint32_t w, float ratio) {
    uint32_t h[2], o = 0;
    codes_to_f16<kFmt>(w, h[0], h[1]);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const __half2 v = *reinterpret_cast<const __half2*>(&h[i]);
        if (kFmt == Q8_E4M3) {
            const __half2 m = __hmul2(v, __float2half2_rn(ratio));
            o |= (uint32_t)__nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&m), __NV_SATFINITE, __NV_E4M3) << (16 * i);
        } else {
            o |= q8_codes2<kFmt>(__low2float(v), __high2float(v), ratio) << (16 * i);
        }
    }
    return o;
}

}  // namespace oxi
