// gemm_mx.hip — products with MXFP4 weights (ggml_mul_mat nodes),
//
//   Y[n, m] = sum_k X[n, k] W[m, k] + bias[m],   W = codes * 2^(scale - 127) per 32 k,
//
// with X in bf16 (or f32, rounded to bf16 as it is read), or X in MXFP4 too.
#include "mxfp4.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

// 8 activations at element k of a row, as bf16
template <bool XF32>
__device__ __forceinline__ bf16x8 load_x8(const void *row, int64_t k) {
    if constexpr (XF32) {
        const f32x4 a = *(const f32x4 *) ((const float *) row + k), b = *(const f32x4 *) ((const float *) row + k + 4);
        bf16x8 r;
        for (int j = 0; j < 4; ++j) {
            r[j] = (__bf16) a[j];
            r[4 + j] = (__bf16) b[j];
        }
        return r;
    } else {
        return *(const bf16x8 *) ((const uint16_t *) row + k);
    }
}

// 4 outputs m .. m + 3 of row n (those below M)
__device__ __forceinline__ void store4(const MxGemm &p, int n, int m, f32x4 v) {
    if (n >= p.N || m >= p.M) return;
    const int64_t at = (int64_t) n * p.ld_y + m;
    if (p.bias) {
        if (m + 3 < p.M) v += *(const f32x4 *) (p.bias + m);
        else for (int i = 0; i < p.M - m; ++i) v[i] += p.bias[m + i];
    }
    if (m + 3 < p.M) {
        if (p.y_bf16) {
            u32x2 h;
            h[0] = f32_to_bf16_bits(v[0]) | (uint32_t) f32_to_bf16_bits(v[1]) << 16;
            h[1] = f32_to_bf16_bits(v[2]) | (uint32_t) f32_to_bf16_bits(v[3]) << 16;
            *(u32x2 *) ((uint16_t *) p.y + at) = h;
        } else {
            *(f32x4 *) ((float *) p.y + at) = v;
        }
        return;
    }
    for (int i = 0; i < p.M - m; ++i) {
        if (p.y_bf16) ((uint16_t *) p.y)[at + i] = f32_to_bf16_bits(v[i]);
        else ((float *) p.y)[at + i] = v[i];
    }
}

// One wave per 16 x 16 outputs. Lane l holds row l % 16 of either operand and
// of each 128 k the block of 32 number l / 16: the operand layout of
// v_mfma_scale_f32_16x16x128_f8f6f4, and with the k of four
// v_mfma_f32_16x16x32_bf16 taken in the same order on both sides, of those.
enum : int { X_BF16 = 0, X_F32 = 1, X_MX = 2 };

template <int XT>
__global__ __launch_bounds__(64) void mx_gemm_simple_kernel(const MxGemm p) {
    const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
    const int tiles_m = (p.M + 15) / 16;
    const int m0 = (int) (blockIdx.x % tiles_m) * 16, n0 = (int) (blockIdx.x / tiles_m) * 16;
    const int KB = p.K / 32;
    const int64_t m = min(m0 + r, p.M - 1), n = min(n0 + r, p.N - 1);
    const uint8_t *wc = p.wq + m * (p.K / 2), *ws = p.ws + m * KB;
    f32x4 acc = {0, 0, 0, 0};
    for (int kb = g; kb < (KB + 3) / 4 * 4; kb += 4) {
        const bool in = kb < KB;
        const u32x4 w = in ? *(const u32x4 *) (wc + kb * 16) : u32x4{0, 0, 0, 0};
        const uint32_t sb = in ? ws[kb] : 127u;
        if constexpr (XT == X_MX) {
            const u32x4 x = in ? *(const u32x4 *) (p.xq + n * (p.K / 2) + kb * 16) : u32x4{0, 0, 0, 0};
            const uint32_t xb = in ? p.xs[n * KB + kb] : 127u;
            const i32x8 a = {(int) w[0], (int) w[1], (int) w[2], (int) w[3], 0, 0, 0, 0};
            const i32x8 b = {(int) x[0], (int) x[1], (int) x[2], (int) x[3], 0, 0, 0, 0};
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, (int) sb, 0, (int) xb);
        } else {
            const void *xr = (const char *) p.x + n * p.ld_x * (XT == X_F32 ? 4 : 2);
            for (int j = 0; j < 4; ++j) {
                bf16x8 b = {0, 0, 0, 0, 0, 0, 0, 0};
                if (in) b = load_x8<XT == X_F32>(xr, (int64_t) kb * 32 + 8 * j);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_decode8_bf16(w[j], mx_scale(sb)), b, acc, 0, 0, 0);
            }
        }
    }
    store4(p, n0 + r, m0 + 4 * g, acc);
}

}  // namespace

hipError_t launch_gemm_mx(const MxGemm &p, hipStream_t s) {
    const int64_t tiles = (int64_t) ((p.M + 15) / 16) * ((p.N + 15) / 16);
    if (tiles > (1 << 26) - 1) return hipErrorInvalidValue;
    const dim3 grid((unsigned) tiles), block(64);
    if (p.xq) launch_kernel(mx_gemm_simple_kernel<X_MX>, grid, block, 0, s, p);
    else if (p.x_f32) launch_kernel(mx_gemm_simple_kernel<X_F32>, grid, block, 0, s, p);
    else launch_kernel(mx_gemm_simple_kernel<X_BF16>, grid, block, 0, s, p);
    return hipGetLastError();
}

}  // namespace tsk
