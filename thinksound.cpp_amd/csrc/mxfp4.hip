// mxfp4.hip — quantization to MXFP4 and back, and the repacking of its blocks.
//
// A block of 32 values x along a row with amax = max |x| takes the scale 2^e,
// e = floor(log2 amax) - 2 (amax / 2^e lies in [4, 8), the top of E2M1), and
// every value the nearest of E2M1's 15 numbers to x / 2^e. Both are exact in
// integer and hardware arithmetic: the exponent is the fp32 exponent field,
// the conversion instruction divides by a power of two and rounds once.
#include <algorithm>

#include "mxfp4.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

// one thread per block of 32
template <bool BF16>
__global__ void mx_quantize_kernel(const void *x, int64_t nb1, int64_t nb2, int64_t nb3, int ne1, int ne2, int64_t rows,
                                   int K, uint8_t *codes, uint8_t *scales, uint8_t *blocks, int64_t ld_blocks) {
    const int KB = K / 32;
    for (int64_t blk = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; blk < rows * KB; blk += (int64_t) gridDim.x * blockDim.x) {
    const int64_t r = blk / KB, kb = blk % KB;
    const int64_t i1 = r % ne1, i2 = r / ne1 % ne2, i3 = r / ne1 / ne2;
    const char *xr = (const char *) x + i1 * nb1 + i2 * nb2 + i3 * nb3;
    float v[32];
    uint32_t top = 0;
    for (int j = 0; j < 32; ++j) {
        v[j] = load_as_f32<BF16 ? Elt::BF16 : Elt::F32>(xr, kb * 32 + j);
        top = max(top, mx_abs_bits(v[j]));
    }
    const uint32_t byte = mx_scale_byte(top);
    const float s = mx_scale(byte);
    uint32_t w[4];
    for (int h = 0; h < 4; ++h) w[h] = byte == 255u ? 0u : mx_encode8(v + 8 * h, s);
    if (blocks) {
        uint8_t *o = blocks + r * ld_blocks + kb * 17;
        o[0] = (uint8_t) byte;
        for (int j = 0; j < 16; ++j)
            o[1 + j] = (uint8_t) (((w[j >> 3] >> 4 * (j & 7)) & 15) | ((w[2 + (j >> 3)] >> 4 * (j & 7)) & 15) << 4);
    } else {
        *(u32x4 *) (codes + blk * 16) = u32x4{w[0], w[1], w[2], w[3]};
        scales[blk] = (uint8_t) byte;
    }
    }
}

// one thread per 8 values
template <bool BF16>
__global__ void mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, const uint8_t *blocks, int64_t ld_blocks,
                                     int ne1, int ne2, int64_t rows, int K, void *y, int64_t nb1, int64_t nb2, int64_t nb3) {
    const int K8 = K / 8;
    for (int64_t i = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; i < rows * K8; i += (int64_t) gridDim.x * blockDim.x) {
    const int64_t r = i / K8, k8 = i % K8;
    uint32_t w, byte;
    if (blocks) {
        const uint8_t *o = blocks + r * ld_blocks + k8 / 4 * 17;
        byte = o[0];
        w = mx_block_codes8(o + 1, (int) (k8 & 3));
    } else {
        byte = scales[i / 4];
        w = ((const uint32_t *) codes)[i];
    }
    float v[8];
    mx_decode8_f32(w, mx_scale(byte), v);
    const int64_t i1 = r % ne1, i2 = r / ne1 % ne2, i3 = r / ne1 / ne2;
    char *yr = (char *) y + i1 * nb1 + i2 * nb2 + i3 * nb3;
    for (int j = 0; j < 8; ++j) store_from_f32<BF16 ? Elt::BF16 : Elt::F32>(yr, k8 * 8 + j, v[j]);
    }
}

// one thread per block
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

// workgroups of 256 for n threads; the kernels stride past the most
dim3 grid_for(int64_t n) { return dim3((unsigned) std::min<int64_t>((n + 255) / 256, 1 << 20)); }

}  // namespace

hipError_t launch_mx_quantize(const View4 &x, uint8_t *codes, uint8_t *scales, uint8_t *blocks, int64_t ld_blocks,
                              hipStream_t s) {
    const int64_t rows = x.ne[1] * x.ne[2] * x.ne[3];
    const int K = (int) x.ne[0];
    launch_kernel(x.type == TSK_TYPE_BF16 ? mx_quantize_kernel<true> : mx_quantize_kernel<false>, grid_for(rows * (K / 32)),
                  dim3(256), 0, s, (const void *) x.data, x.nb[1], x.nb[2], x.nb[3], (int) x.ne[1], (int) x.ne[2], rows, K,
                  codes, scales, blocks, ld_blocks);
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, const uint8_t *blocks, int64_t ld_blocks,
                                const View4 &y, hipStream_t s) {
    const int64_t rows = y.ne[1] * y.ne[2] * y.ne[3];
    const int K = (int) y.ne[0];
    launch_kernel(y.type == TSK_TYPE_BF16 ? mx_dequantize_kernel<true> : mx_dequantize_kernel<false>, grid_for(rows * (K / 8)),
                  dim3(256), 0, s, codes, scales, blocks, ld_blocks, (int) y.ne[1], (int) y.ne[2], rows, K, (void *) y.data,
                  y.nb[1], y.nb[2], y.nb[3]);
    return hipGetLastError();
}

hipError_t launch_mx_repack(const uint8_t *blocks, int64_t ld_blocks, int64_t rows, int64_t K, uint8_t *codes,
                            uint8_t *scales, hipStream_t s) {
    launch_kernel(mx_repack_kernel, grid_for(rows * (K / 32)), dim3(256), 0, s, blocks, ld_blocks, rows, (int) K, codes,
                  scales);
    return hipGetLastError();
}

}  // namespace tsk
