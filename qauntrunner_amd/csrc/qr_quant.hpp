// qr_quant.hpp -- rows of 8-bit caches: codes c of e4m3 (nearest even, largest 448) and one exponent e per row of a kv
// head's values, a value being c 2^e.  e is the smallest exponent of kMinExp .. kMaxExp that keeps the row's largest
// finite |x| at or below 448 2^e.  A power of two divides without rounding, so a value is rounded once, and it is a number
// of bf16 (4 of its 8 bits; the exponents keep the smallest, 2^-9 2^e, a normal number and the largest below infinity), so
// that products take it as it is.
#pragma once

#include "qr_common.hpp"

namespace qr {

constexpr int kMinExp = -117, kMaxExp = 119;

// Bits of the scale byte as the float 2^e (0: a slot never written, whose codes are 0).
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b << 23); }

// e of a largest |x|: 1.75 2^8 = 448.
__device__ __forceinline__ int quant_exp(float top) {
    const uint32_t b = __float_as_uint(top);
    return min(max(static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u), kMinExp), kMaxExp);
}
__device__ __forceinline__ int quant_exp(double top) {
    const unsigned long long b = __double_as_longlong(top);
    return min(max(static_cast<int>(b >> 52) - 1023 - 8 + ((b & 0xFFFFFFFFFFFFFull) > 0xC000000000000ull), kMinExp), kMaxExp);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Codes of two values and of four, |y| <= 448 or not finite (v_cvt_pk_fp8_f32 rounds to nearest even).
__device__ __forceinline__ float quant_clamp(float y) { return fabsf(y) <= 448.f || y != y ? y : copysignf(448.f, y); }
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// y to the nearest code's value in 64 bits (even on a tie): a sum with 1.5 2^52 steps leaves whole steps.  Rounded to 32
// bits first it could fall on a tie that it is not.
__device__ __forceinline__ float quant_round(double y) {
    const double a = fabs(y);
    if (!(a <= 448.0)) return y != y ? NAN : copysignf(448.f, static_cast<float>(y));
    const int e = max(static_cast<int>(static_cast<unsigned long long>(__double_as_longlong(a)) >> 52) - 1023, -6) - 3;
    const double big = __longlong_as_double((static_cast<unsigned long long>(e + 52 + 1023) << 52) | 0x8000000000000ull);
    return copysignf(static_cast<float>((a + big) - big), static_cast<float>(y));
}
// Value of a code, byte `i` of w.
template <int I> __device__ __forceinline__ float quant_value(uint32_t w) { return __builtin_amdgcn_cvt_f32_fp8(w, I); }

}  // namespace qr
