// Numbers of 8 bits (e4m3: sign, 4 bits of exponent, 3 of mantissa; largest 448, no infinity, NaN 0x7f) as the kernels over 8-bit weights and an
// 8-bit cache convert them.  Every e4m3 number is a half exactly.
#pragma once

#include "common.cuh"

namespace qt_fp8 {

constexpr int GROUP = 128;         // columns, and rows of a weight, that share a scale
constexpr float TOP = 448.f;       // the largest number
constexpr int MIN_POWER = -40, MAX_POWER = 40;      // of a cache block's scale

// Two floats, the first in the lower byte: nearest, ties to even; beyond 448 becomes 448, NaN stays NaN.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint16_t v;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
    return v;
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) { return pack2(a, b) | (pack2(c, d) << 16); }
// Two numbers as halves, the lower byte in the lower half.
__device__ __forceinline__ uint32_t halves(uint32_t two) {
    uint32_t v;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(v) : "h"((uint16_t)two));
    return v;
}
__device__ __forceinline__ float2 floats(uint32_t two) {
    const uint32_t v = halves(two);
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// Whether one of four numbers is NaN: all bits but the sign are set.
__device__ __forceinline__ uint32_t any_nan(uint32_t four) { return ((four & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// An infinity is held as NaN: 448 would be a number.
__device__ __forceinline__ float nan_if_infinite(float v) { return fabsf(v) < INFINITY ? v : __int_as_float(0x7fffffff); }

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }      // e between -126 and 127
// The smallest e with largest <= 448 * 2^e = 1.75 * 2^(8 + e), between MIN_POWER and MAX_POWER.
__device__ __forceinline__ int power_for(float largest) {
    const int bits = __float_as_int(largest);
    return min(max((bits >> 23) - 135 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), MIN_POWER), MAX_POWER);
}
// The smallest e with scale <= 2^e.
__device__ __forceinline__ int power_over(float scale) {
    const int bits = __float_as_int(scale);
    return min(max((bits >> 23) - 127 + ((bits & 0x7fffff) != 0 ? 1 : 0), MIN_POWER), MAX_POWER);
}

}  // namespace qt_fp8
