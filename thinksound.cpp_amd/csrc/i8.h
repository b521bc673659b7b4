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
// The codes of four values. x / d and x * (1 / d) are at most 127 and 2^-16 apart, so that the
// integer nearest to the product is that of the quotient, but where the product is within
// 2^-16 of a half: there i8_code decides. The sum with 1.5 * 2^23 rounds to an integer, whose
// low byte is the sum's. (8192 x 8192 bf16: 37.7 us, with i8_code for every value 40.2.)
__device__ __forceinline__ uint32_t i8_pack4(const float *v, const I8Scale &s) {
    if (s.inv == 0.0f) return 0u;
    uint32_t b[4];
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float m = __builtin_fmaf(v[e], s.inv, 12582912.0f);
        off = fmaxf(off, __builtin_fabsf(__builtin_fmaf(v[e], s.inv, 12582912.0f - m)));
        b[e] = __float_as_uint(m);
    }
    if (off > 0.5f - 0x1p-16f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (uint32_t) i8_code(v[e], s);
    }
    return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
}

// Vectors that start on any value: the memory takes them whole too (8191 x 8191 bf16, value
// by value 112.6 us, in vectors 55.2; aligned rows as long 37.8)
typedef __attribute__((__vector_size__(16), aligned(2))) uint32_t u32x4_any2;
typedef __attribute__((__vector_size__(16), aligned(4))) float f32x4_any4;

// 8 values of an f32 or bf16 row from column c on, those past K zeros; WIDE: the row starts on 16 bytes
template <bool BF16, bool WIDE>
__device__ __forceinline__ void i8_load8(const char *row, int c, int K, float *v) {
    if (c + 8 <= K) {
        if constexpr (BF16) {
            const u32x4 w = WIDE ? *(const u32x4 *) (row + (int64_t) c * 2) : (u32x4) *(const u32x4_any2 *) (row + (int64_t) c * 2);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[2 * q] = __uint_as_float(w[q] << 16);
                v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
            }
        } else {
            f32x4 a, b;
            if constexpr (WIDE) {
                a = ((const f32x4 *) (row + (int64_t) c * 4))[0];
                b = ((const f32x4 *) (row + (int64_t) c * 4))[1];
            } else {
                a = ((const f32x4_any4 *) (row + (int64_t) c * 4))[0];
                b = ((const f32x4_any4 *) (row + (int64_t) c * 4))[1];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = a[e];
                v[4 + e] = b[e];
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < K ? load_as_f32<BF16 ? Elt::BF16 : Elt::F32>(row, c + e) : 0.0f;
}

}  // namespace tsk
