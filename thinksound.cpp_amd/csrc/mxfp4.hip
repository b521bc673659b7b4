// mxfp4.hip — quantization to MXFP4 and back, and the repacking of its blocks.
//
// A block of 32 values x along a row with amax = max |x| takes the scale 2^e,
// e = floor(log2 amax) - 2 (amax / 2^e lies in [4, 8), the top of E2M1), and
// every value the nearest of E2M1's 15 numbers to x / 2^e. Both are exact in
// integer and hardware arithmetic: the exponent is the fp32 exponent field,
// the conversion instruction divides by a power of two and rounds once. Bound by
// memory throughout: each value is read once, each code and scale written once.
#include <algorithm>

#include "mxfp4.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

// The row and column of piece i, P pieces a row (one long row where rows follow
// each other without gaps: no division)
struct Rows {
    int64_t nb1, nb2, nb3;
    int ne1, ne2, packed;
};
__device__ __forceinline__ int64_t byte_at(const Rows &t, int64_t i, int P, int piece_bytes) {
    if (t.packed) return i * piece_bytes;
    const int64_t r = i / P;
    const int64_t i1 = r % t.ne1, q = r / t.ne1;
    return i1 * t.nb1 + q % t.ne2 * t.nb2 + q / t.ne2 * t.nb3 + (i - r * P) * piece_bytes;
}

// Rows on 16-byte starts into planes: a thread takes 8 values, four neighbours a
// block, so that a wave's loads and stores are runs of whole lines. 8192 x 8192
// values from f32 53 us (5.8 TB/s read and written; 70 in turns with as large a
// dequantization), from bf16 33 us (5.1 TB/s).
template <bool BF16>
__global__ void mx_quantize_kernel(const void *x, const Rows t, int64_t n8, int K8, uint8_t *codes, uint8_t *scales) {
    for (int64_t i = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t) gridDim.x * blockDim.x) {
        const char *p = (const char *) x + byte_at(t, i, K8, BF16 ? 16 : 32);
        float v[8];
        if constexpr (BF16) {
            const u32x4 w = *(const u32x4 *) p;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                v[2 * q] = __uint_as_float(w[q] << 16);
                v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
            }
        } else {
            const f32x4 a = ((const f32x4 *) p)[0], b = ((const f32x4 *) p)[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = a[e];
                v[4 + e] = b[e];
            }
        }
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, mx_abs_bits(v[e]));
        top = mx_quad_max(top);                                // (n8 is a multiple of 4: four active lanes, or none)
        const uint32_t byte = mx_scale_byte(top);
        ((uint32_t *) codes)[i] = byte == 255u ? 0u : mx_encode8(v, mx_scale(byte));
        if ((i & 3) == 0) scales[i / 4] = (uint8_t) byte;
    }
}

// Any rows, into planes or blocks: one thread per block of 32, whose lines its
// later loads find in L1. 8192 x 8192 f32 values from rows off 16 bytes 55 us, into
// blocks 63 us (4.8 TB/s).
template <bool BF16>
__global__ void mx_quantize_any_kernel(const void *x, const Rows t, int64_t nblk, int KB, uint8_t *codes, uint8_t *scales,
                                       uint8_t *blocks, int64_t ld_blocks) {
    for (int64_t blk = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; blk < nblk; blk += (int64_t) gridDim.x * blockDim.x) {
        const char *p = (const char *) x + byte_at(t, blk, KB, BF16 ? 64 : 128);
        float v[32];
        uint32_t top = 0;
        for (int j = 0; j < 32; ++j) {
            v[j] = load_as_f32<BF16 ? Elt::BF16 : Elt::F32>(p, j);
            top = max(top, mx_abs_bits(v[j]));
        }
        const uint32_t byte = mx_scale_byte(top);
        const float s = mx_scale(byte);
        uint32_t w[4];
        for (int h = 0; h < 4; ++h) w[h] = byte == 255u ? 0u : mx_encode8(v + 8 * h, s);
        if (blocks) {
            uint8_t *o = blocks + blk / KB * ld_blocks + blk % KB * 17;
            o[0] = (uint8_t) byte;
            for (int j = 0; j < 16; ++j)
                o[1 + j] = (uint8_t) (((w[j >> 3] >> 4 * (j & 7)) & 15) | ((w[2 + (j >> 3)] >> 4 * (j & 7)) & 15) << 4);
        } else {
            *(u32x4 *) (codes + blk * 16) = u32x4{w[0], w[1], w[2], w[3]};
            scales[blk] = (uint8_t) byte;
        }
    }
}

// One thread per 8 values, WIDE: to rows on 16-byte starts. 8192 x 8192 values to
// f32 61 us (5.0 TB/s), to bf16 35 us, from blocks to f32 77 us (their bytes are
// read one at a time).
template <bool BF16, bool WIDE>
__global__ void mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, const uint8_t *blocks, int64_t ld_blocks,
                                     void *y, const Rows t, int64_t n8, int K8) {
    for (int64_t i = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t) gridDim.x * blockDim.x) {
        uint32_t w, byte;
        if (blocks) {
            const int64_t k8 = i % K8;
            const uint8_t *o = blocks + i / K8 * ld_blocks + k8 / 4 * 17;
            byte = o[0];
            w = mx_block_codes8(o + 1, (int) (k8 & 3));
        } else {
            byte = scales[i / 4];
            w = ((const uint32_t *) codes)[i];
        }
        char *p = (char *) y + byte_at(t, i, K8, BF16 ? 16 : 32);
        if constexpr (BF16) {
            const u32x4 h = __builtin_bit_cast(u32x4, mx_decode8_bf16(w, mx_scale(byte)));
            if constexpr (WIDE) *(u32x4 *) p = h;
            else
                for (int j = 0; j < 8; ++j) ((uint16_t *) p)[j] = (uint16_t) (h[j >> 1] >> 16 * (j & 1));
        } else {
            float v[8];
            mx_decode8_f32(w, mx_scale(byte), v);
            if constexpr (WIDE) {
                ((f32x4 *) p)[0] = f32x4{v[0], v[1], v[2], v[3]};
                ((f32x4 *) p)[1] = f32x4{v[4], v[5], v[6], v[7]};
            } else {
                for (int j = 0; j < 8; ++j) ((float *) p)[j] = v[j];
            }
        }
    }
}

// One thread per block. 8192 x 8192 values 13 us (5.5 TB/s).
__global__ void mx_repack_kernel(const uint8_t *blocks, int64_t ld_blocks, int64_t rows, int K, uint8_t *codes,
                                 uint8_t *scales) {
    const int KB = K / 32;
    for (int64_t blk = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; blk < rows * KB; blk += (int64_t) gridDim.x * blockDim.x) {
        const uint8_t *o = blocks + blk / KB * ld_blocks + blk % KB * 17;
        *(u32x4 *) (codes + blk * 16) = u32x4{mx_block_codes8(o + 1, 0), mx_block_codes8(o + 1, 1), mx_block_codes8(o + 1, 2),
                                              mx_block_codes8(o + 1, 3)};
        scales[blk] = o[0];
    }
}

Rows rows_of(const View4 &t) {
    Rows r;
    const int64_t row = t.ne[0] * (t.type == TSK_TYPE_BF16 ? 2 : 4);
    r.nb1 = t.nb[1]; r.nb2 = t.nb[2]; r.nb3 = t.nb[3];
    r.ne1 = (int) t.ne[1]; r.ne2 = (int) t.ne[2];
    r.packed = (t.ne[1] == 1 || t.nb[1] == row) && (t.ne[2] == 1 || t.nb[2] == row * t.ne[1]) &&
               (t.ne[3] == 1 || t.nb[3] == row * t.ne[1] * t.ne[2]);
    return r;
}
bool on_16(const View4 &t) {
    bool ok = (uintptr_t) t.data % 16 == 0;
    for (int i = 1; i < 4; ++i) ok = ok && (t.ne[i] == 1 || t.nb[i] % 16 == 0);
    return ok;
}

// workgroups of 256 for n threads; the kernels stride past the most
dim3 grid_for(int64_t n) { return dim3((unsigned) std::min<int64_t>((n + 255) / 256, 1 << 20)); }

}  // namespace

hipError_t launch_mx_quantize(const View4 &x, uint8_t *codes, uint8_t *scales, uint8_t *blocks, int64_t ld_blocks,
                              hipStream_t s) {
    const int64_t n = x.ne[0] * x.ne[1] * x.ne[2] * x.ne[3];
    const int K = (int) x.ne[0];
    const bool bf16 = x.type == TSK_TYPE_BF16;
    const void *data = x.data;
    if (!blocks && on_16(x))
        launch_kernel(bf16 ? mx_quantize_kernel<true> : mx_quantize_kernel<false>, grid_for(n / 8), dim3(256), 0, s, data,
                      rows_of(x), n / 8, K / 8, codes, scales);
    else
        launch_kernel(bf16 ? mx_quantize_any_kernel<true> : mx_quantize_any_kernel<false>, grid_for(n / 32), dim3(256), 0, s,
                      data, rows_of(x), n / 32, K / 32, codes, scales, blocks, ld_blocks);
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, const uint8_t *blocks, int64_t ld_blocks,
                                const View4 &y, hipStream_t s) {
    const int64_t n = y.ne[0] * y.ne[1] * y.ne[2] * y.ne[3];
    const bool bf16 = y.type == TSK_TYPE_BF16, wide = on_16(y);
    launch_kernel(bf16 ? wide ? mx_dequantize_kernel<true, true> : mx_dequantize_kernel<true, false>
                       : wide ? mx_dequantize_kernel<false, true> : mx_dequantize_kernel<false, false>,
                  grid_for(n / 8), dim3(256), 0, s, codes, scales, blocks, ld_blocks, (void *) y.data, rows_of(y), n / 8,
                  (int) y.ne[0] / 8);
    return hipGetLastError();
}

hipError_t launch_mx_repack(const uint8_t *blocks, int64_t ld_blocks, int64_t rows, int64_t K, uint8_t *codes,
                            uint8_t *scales, hipStream_t s) {
    launch_kernel(mx_repack_kernel, grid_for(rows * (K / 32)), dim3(256), 0, s, blocks, ld_blocks, rows, (int) K, codes,
                  scales);
    return hipGetLastError();
}

}  // namespace tsk
