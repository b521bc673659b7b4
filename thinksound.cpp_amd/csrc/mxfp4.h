// mxfp4.h — MXFP4 numbers (OCP Microscaling v1.0: 32 E2M1 codes sharing one
// E8M0 scale byte) as the gfx950 conversion instructions take them.
#pragma once

#include "tsk_common.h"

namespace tsk {

typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;

// |v| as an integer: the order of the magnitudes, with every NaN above infinity
__device__ __forceinline__ uint32_t mx_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// scale byte of a block whose largest mx_abs_bits is `top`: the exponent of the
// largest value less 2 (E2M1's own largest exponent), 0 at least (2^-127; the
// fp32 exponent field is 0 for zeros and subnormals), 255 for a non-finite one
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// the scale as the conversions read it: an fp32 power of two by its exponent
// field, where 0 is 2^-127 and 255 makes every value NaN
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// the largest of a group of four lanes (all of them active)
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
    v = max(v, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, 0xB1, 0xF, 0xF, false));   // quad [1, 0, 3, 2]
    return max(v, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, 0x4E, 0xF, 0xF, false));  // quad [2, 3, 0, 1]
}

// 8 values over `scale` -> 8 codes (v_cvt_scalef32_pk_fp4_f32: nearest, ties to
// the even code, saturating at 6); values of a block whose byte is not 255
__device__ __forceinline__ uint32_t mx_encode8(const float *v, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}

// 8 codes -> their values in bf16 (exact: 2 bits of mantissa; 2^-128 is a bf16
// subnormal), NaN where the scale's byte was 255
__device__ __forceinline__ bf16x8 mx_decode8_bf16(uint32_t w, float scale) {
    union { bf16x2 h[4]; bf16x8 v; } u;
    u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
    u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
    u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return u.v;
}
__device__ __forceinline__ void mx_decode8_f32(uint32_t w, float scale, float *v) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
    v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}

// MXFP4 blocks hold value i < 16 in byte i's low nibble and i >= 16 in byte
// (i - 16)'s high one; the planes hold values 2 i and 2 i + 1 in byte i. Codes
// 8 h .. 8 h + 7 of a block from / to its 16 bytes.
__device__ __forceinline__ uint32_t mx_block_codes8(const uint8_t *qs, int h) {
    uint32_t w = 0;
    for (int j = 0; j < 8; ++j) w |= (uint32_t) ((qs[(h & 1) * 8 + j] >> (h >> 1) * 4) & 15) << (4 * j);
    return w;
}

}  // namespace tsk
