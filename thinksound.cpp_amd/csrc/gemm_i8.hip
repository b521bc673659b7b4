// gemm_i8.hip — products of 8-bit integer rows with a scale each (ggml_mul_mat nodes
// with I8_SPLIT weights),
//
//   Y[n, m] = (sum_k XQ[n, k] WQ[m, k]) * XD[n] * WD[m] + bias[m].
//
// Sums are int32 and exact (K below 2^17: 2^14 K stays below 2^31); they are
// rounded once to fp32, then scaled. v_mfma_i32_16x16x64_i8 multiplies.
#include <algorithm>

#include "i8.h"
#include "tsk_internal.h"
#include "tsk_runtime.h"

namespace tsk {

namespace {

// 4 outputs m .. m + 3 of row n (those below M) from their integer sums
__device__ __forceinline__ void store4(const I8Gemm &p, int n, int m, i32x4 acc) {
    if (n >= p.N || m >= p.M) return;
    const int64_t at = (int64_t) n * p.ld_y + m;
    const float xd = p.xd[n];
    float v[4];
    const int left = min(4, p.M - m);
    for (int i = 0; i < left; ++i) {
        v[i] = (float) acc[i] * xd * p.wd[m + i];
        if (p.bias) v[i] += p.bias[m + i];
    }
    if (left == 4) {
        if (p.y_bf16) {
            u32x2 h;
            h[0] = f32_to_bf16_bits(v[0]) | (uint32_t) f32_to_bf16_bits(v[1]) << 16;
            h[1] = f32_to_bf16_bits(v[2]) | (uint32_t) f32_to_bf16_bits(v[3]) << 16;
            *(u32x2 *) ((uint16_t *) p.y + at) = h;
        } else {
            *(f32x4 *) ((float *) p.y + at) = f32x4{v[0], v[1], v[2], v[3]};
        }
        return;
    }
    for (int i = 0; i < left; ++i) {
        if (p.y_bf16) ((uint16_t *) p.y)[at + i] = f32_to_bf16_bits(v[i]);
        else ((float *) p.y)[at + i] = v[i];
    }
}

// ---------------------------------------------------------------- few rows
// Operands straight into registers. NW waves share 16 MT x 16 NT outputs and
// deal the K range among them in turns of 128 k; their sums meet in LDS.
// Lane l holds row l % 16 of either operand and of each 64 k the 16 bytes l / 16.
template <int MT, int NT>
struct RowFrags {
    i32x4 a[MT][2], b[NT][2];
};

template <int MT, int NT, int NW>
__global__ __launch_bounds__(NW * 64) void i8_gemm_rows_kernel(const I8Gemm p, int tiles_m) {
    __shared__ __attribute__((aligned(16))) int red[NW > 1 ? NW * MT * NT * 256 : 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int m0 = (int) (blockIdx.x % tiles_m) * (16 * MT), n0 = (int) (blockIdx.x / tiles_m) * (16 * NT);
    const int64_t ld = i8_ld(p.K);
    const int nit = (int) ((ld + 127) / 128);
    // rows past M or N read the last one (their outputs are not stored)
    const int8_t *wq[MT], *xq[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) wq[i] = p.wq + (int64_t) min(m0 + 16 * i + r, p.M - 1) * ld + 16 * g;
#pragma unroll
    for (int j = 0; j < NT; ++j) xq[j] = p.xq + (int64_t) min(n0 + 16 * j + r, p.N - 1) * ld + 16 * g;
    auto load = [&](int it, RowFrags<MT, NT> &f) {
        const int64_t k0 = (int64_t) it * 128;
        const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const bool in = k0 + 64 * ks + 16 * g < ld;      // (rows are whole pieces of 16)
#pragma unroll
            for (int i = 0; i < MT; ++i) f.a[i][ks] = in ? *(const i32x4 *) (wq[i] + k0 + 64 * ks) : zero;
#pragma unroll
            for (int j = 0; j < NT; ++j) f.b[j][ks] = in ? *(const i32x4 *) (xq[j] + k0 + 64 * ks) : zero;
        }
    };
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    auto product = [&](const RowFrags<MT, NT> &f) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.a[i][ks], f.b[j][ks], acc[i][j], 0, 0, 0);
    };
    if (wave < nit) {
        RowFrags<MT, NT> f0, f1;
        load(wave, f0);
        int it = wave;
        for (; it + NW < nit; it += 2 * NW) {
            load(it + NW, f1);
            product(f0);
            if (it + 2 * NW < nit) load(it + 2 * NW, f0);
            product(f1);
        }
        if (it < nit) product(f0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) *(i32x4 *) (red + ((wave * MT * NT + i * NT + j) * 64 + lane) * 4) = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            if ((i * NT + j) % NW != wave) continue;
            i32x4 v = *(const i32x4 *) (red + ((i * NT + j) * 64 + lane) * 4);
            for (int w = 1; w < NW; ++w) v += *(const i32x4 *) (red + ((w * MT * NT + i * NT + j) * 64 + lane) * 4);
            store4(p, n0 + 16 * j + r, m0 + 16 * i + 4 * g, v);
        }
}

// A launch holds fewer than 2^32 threads: products of more are cut into two by their rows
constexpr int64_t MAX_THREADS = (int64_t) 1 << 31;
template <class F>
hipError_t in_two(const I8Gemm &p, F launch) {
    I8Gemm a = p, b = p;
    a.N = (p.N / 2 + 15) / 16 * 16;
    b.N = p.N - a.N;
    if (b.N < 1) return hipErrorInvalidValue;
    b.y = (char *) p.y + a.N * p.ld_y * (p.y_bf16 ? 2 : 4);
    b.xq = p.xq + (int64_t) a.N * i8_ld(p.K);
    b.xd = p.xd + a.N;
    const hipError_t e = launch(a);
    return e == hipSuccess ? launch(b) : e;
}

template <int MT, int NT, int NW>
hipError_t launch_rows(const I8Gemm &p, hipStream_t s) {
    const int tiles_m = (p.M + 16 * MT - 1) / (16 * MT), tiles_n = (p.N + 16 * NT - 1) / (16 * NT);
    const int64_t T = (int64_t) tiles_m * tiles_n;
    if (T * NW * 64 >= MAX_THREADS) return in_two(p, [&](const I8Gemm &q) { return launch_rows<MT, NT, NW>(q, s); });
    launch_kernel(i8_gemm_rows_kernel<MT, NT, NW>, dim3((unsigned) T), dim3(NW * 64), 0, s, p, tiles_m);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_gemm_i8(const I8Gemm &p, hipStream_t s) {
    return launch_rows<2, 2, 4>(p, s);
}

}  // namespace tsk
