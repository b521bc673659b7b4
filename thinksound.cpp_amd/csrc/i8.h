// i8.h — rows of 8-bit integers with one scale each (TSK_TYPE_I8_SPLIT).
#pragma once

#include "tsk_common.h"

namespace tsk {

// A row's scale d = max(amax, 2^-100) / 127 and the integers nearest to x / d, ties
// to even. The floor keeps d and 1 / d normal numbers for rows of zeros (whose integers are 0).
constexpr float I8_TINY = 0x1p-100f;

// bytes from a row of K integers to the next: 16-byte starts, zeros past K
__host__ __device__ constexpr int64_t i8_ld(int64_t K) { return (K + 15) / 16 * 16; }

// |x| as bits that order like the magnitudes, infinities and NaNs (above 0x7f7fffff) on top
__device__ __forceinline__ uint32_t i8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct I8Scale {
    float d, inv, half;
};
// top: the row's largest i8_abs_bits. A row that holds an infinity or a NaN gets the
// scale NaN and integers 0: all its values are NaN.
__device__ __forceinline__ I8Scale i8_scale(uint32_t top) {
    I8Scale s;
    if (top > 0x7f7fffffu) {
        s.d = __uint_as_float(0x7fc00000u);
        s.inv = s.half = 0.0f;
    } else {
        s.d = fmaxf(__uint_as_float(top), I8_TINY) / 127.0f;
        s.inv = 1.0f / s.d;
        s.half = 0.5f * s.d;
    }
    return s;
}
// x / d to the nearest integer, ties to even. The product with 1 / d is within a few
// units of its last place of the quotient, so its nearest integer q is at most one off,
// and only next to a half; x - q d, an exact fp32 number there, settles it.
__device__ __forceinline__ int i8_code(float x, const I8Scale &s) {
    const float q = __builtin_rintf(x * s.inv);
    const float r = __builtin_fmaf(-q, s.d, x);
    const int i = (int) q;
    const float lim = s.half, a = __builtin_fabsf(r);
    const bool off = a > lim || (a == lim && (i & 1));
    return off ? i + (r > 0.0f ? 1 : -1) : i;
}
__device__ __forceinline__ uint32_t i8_pack4(const float *v, const I8Scale &s) {
    if (s.inv == 0.0f) return 0u;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= ((uint32_t) i8_code(v[e], s) & 255u) << 8 * e;
    return w;
}

}  // namespace tsk
