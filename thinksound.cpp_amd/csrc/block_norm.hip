// block_norm.hip — the norms, gate and residual between two blocks' matrices
// (x + gate * y, ggml_norm and modulate of src/mmdit.cpp:55-59, :231-234):
//
//   r   = res_scale * x + gate * post(y),  res = r in x's type
//   dst = pre(res) * pre_w * (1 + scale) + shift    (f32, bf16 or MXFP4)
//
// Bound by memory: x and y are read once, res and dst written once.
#include <algorithm>

#include "mxfp4.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

__device__ __forceinline__ float wg_sum(float v, float *red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.0f;
    for (int i = 0; i < (int) (blockDim.x >> 6); ++i) t += red[i];
    return t;
}

__device__ __forceinline__ float load_elt(const void *row, int bf16, int i) {
    return bf16 ? bf16_bits_to_f32(((const uint16_t *) row)[i]) : ((const float *) row)[i];
}
__device__ __forceinline__ float as_type(float v, int bf16) { return bf16 ? bf16_bits_to_f32(f32_to_bf16_bits(v)) : v; }

__device__ __forceinline__ const char *row_of(const BnView &t, int i1, int i2, int i3) {
    return (const char *) t.data + i1 * t.nb1 + i2 * t.nb2 + i3 * t.nb3;
}

// mean and 1 / sqrt(var + eps) of C values f(i) (layer norm: two passes, the
// deviations squared), or 0 and 1 / sqrt(mean of squares + eps)
template <class F>
__device__ __forceinline__ void row_stats(int kind, int C, float eps, float *red, F f, float *mean, float *inv) {
    *mean = 0.0f;
    *inv = 1.0f;
    if (kind == TSK_NORM_NONE) return;
    if (kind == TSK_NORM_LAYER) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < C; i += blockDim.x) s += f(i);
        *mean = wg_sum(s, red) / (float) C;
    }
    float q = 0.0f;
    for (int i = threadIdx.x; i < C; i += blockDim.x) {
        const float d = f(i) - *mean;
        q += d * d;
    }
    *inv = 1.0f / sqrtf(wg_sum(q, red) / (float) C + eps);
}

// One workgroup per row, which reads its row from memory for every pass.
__global__ __launch_bounds__(256) void block_norm_simple_kernel(const BlockNorm p) {
    __shared__ float red[4];
    const int64_t rows = (int64_t) p.n1 * p.n2 * p.n3;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int i1 = (int) (r % p.n1), i2 = (int) (r / p.n1 % p.n2), i3 = (int) (r / p.n1 / p.n2);
    const char *x = row_of(p.x, i1, i2, i3), *y = p.y.data ? row_of(p.y, i1, i2, i3) : nullptr;
    const float *gate = p.gate.data ? (const float *) row_of(p.gate, i1, i2, i3) : nullptr;
    const float *scale = p.scale.data ? (const float *) row_of(p.scale, i1, i2, i3) : nullptr;
    const float *shift = p.shift.data ? (const float *) row_of(p.shift, i1, i2, i3) : nullptr;
    float ymean = 0.0f, yinv = 1.0f, mean, inv;
    if (y) row_stats(p.post_norm, p.C, p.post_eps, red, [&](int i) { return load_elt(y, p.y_bf16, i); }, &ymean, &yinv);
    auto sum = [&](int i) {
        float v = p.res_scale * load_elt(x, p.x_bf16, i);
        if (y) {
            float b = load_elt(y, p.y_bf16, i);
            if (p.post_norm) b = (b - ymean) * yinv;
            if (p.post_w) b *= p.post_w[i];
            v += gate ? gate[i] * b : b;
        }
        return as_type(v, p.x_bf16);
    };
    if (p.dst.data || p.scales) {
        row_stats(p.pre_norm, p.C, p.pre_eps, red, sum, &mean, &inv);
        auto out = [&](int i) {
            float v = sum(i);
            if (p.pre_norm) v = (v - mean) * inv;
            if (p.pre_w) v *= p.pre_w[i];
            if (scale) v *= 1.0f + scale[i];
            if (shift) v += shift[i];
            return v;
        };
        if (p.scales) {
            for (int kb = threadIdx.x; kb < p.C / 32; kb += blockDim.x) {
                float v[32];
                uint32_t top = 0;
                for (int j = 0; j < 32; ++j) {
                    v[j] = out(kb * 32 + j);
                    top = max(top, mx_abs_bits(v[j]));
                }
                const uint32_t byte = mx_scale_byte(top);
                u32x4 w;
                for (int h = 0; h < 4; ++h) w[h] = byte == 255u ? 0u : mx_encode8(v + 8 * h, mx_scale(byte));
                *(u32x4 *) (p.codes + r * (p.C / 2) + kb * 16) = w;
                p.scales[r * (p.C / 32) + kb] = (uint8_t) byte;
            }
        } else {
            char *d = (char *) row_of(p.dst, i1, i2, i3);
            for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
                if (p.dst_bf16) ((uint16_t *) d)[i] = f32_to_bf16_bits(out(i));
                else ((float *) d)[i] = out(i);
            }
        }
    }
    if (p.res.data) {
        __syncthreads();                              // (res may be x)
        char *d = (char *) row_of(p.res, i1, i2, i3);
        for (int i = threadIdx.x; i < p.C; i += blockDim.x) {
            const float v = sum(i);
            if (p.x_bf16) ((uint16_t *) d)[i] = f32_to_bf16_bits(v);
            else ((float *) d)[i] = v;
        }
    }
    }
}

}  // namespace

hipError_t launch_block_norm(const BlockNorm &p, hipStream_t s) {
    const int64_t rows = (int64_t) p.n1 * p.n2 * p.n3;
    launch_kernel(block_norm_simple_kernel, dim3((unsigned) std::min<int64_t>(rows, 1 << 20)), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace tsk
