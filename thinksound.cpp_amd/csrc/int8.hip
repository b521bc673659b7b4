// int8.hip — rows to 8-bit integers with one scale each, and back.
//
// d = max(amax, 2^-100) / 127, q = the integer nearest to x / d (i8.h). Bound by memory:
// a row is read once into the registers of the threads that share it, whose largest
// magnitude is found between the load and the store. A vector instruction takes a wave four
// cycles, so a value's few count: 8192 x 8192 bf16, 16 arrays in turn so that none is in a cache, 37.7 us
// (5.3 TB/s; a copy 5.1; with magnitudes of 32 bits and i8_code for every value 52.4; one array again and again
// 32), f32 60.0 (5.6).
#include <algorithm>
#include <type_traits>

#include "i8.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

// flat: rows nb1 apart throughout
struct Rows {
    int64_t nb1, nb2, nb3;
    int ne1, ne2;
    bool flat;
};
__device__ __forceinline__ int64_t row_at(const Rows &t, int64_t r) {
    if (t.flat) return r * t.nb1;
    const int64_t i1 = r % t.ne1, q = r / t.ne1;
    return i1 * t.nb1 + q % t.ne2 * t.nb2 + q / t.ne2 * t.nb3;
}

// the largest of the NT threads of a row: 8 to 64 lanes of a wave, or NT / 64 waves
template <int NT>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t *red) {
    // (magnitudes' bits order like unsigned integers, NaNs on top; DPP: swaps within quads, then mirrors of 8 and 16)
    v = max(v, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, 0x141, 0xF, 0xF, false));
    if constexpr (NT > 8) v = max(v, (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v, 0x140, 0xF, 0xF, false));
    if constexpr (NT > 16) {
        const auto s16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(s16[0], s16[1]);
    }
    if constexpr (NT > 32) {
        const auto s32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max(s32[0], s32[1]);
    }
    if constexpr (NT > 64) {
        uint32_t *own = red + threadIdx.x / NT * (NT / 64);
        __syncthreads();                                     // (the row before may still be read)
        if ((threadIdx.x & 63) == 0) own[threadIdx.x % NT >> 6] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) v = max(v, own[i]);
    }
    return v;
}

// 8 values as they are kept until their row's largest is known: bf16 ones in pairs, whose
// magnitudes are compared two at a time
template <bool BF16, bool WIDE> struct Vec8 {
    float v[8];
    __device__ __forceinline__ void load(const char *row, int c, int K) { i8_load8<BF16, WIDE>(row, c, K, v); }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = max(t, i8_abs_bits(v[e]));
        return t;
    }
    __device__ __forceinline__ void values(float *w) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = v[e];
    }
};
typedef __attribute__((__vector_size__(2 * sizeof(uint16_t)))) uint16_t u16x2;
template <bool WIDE> struct Vec8<true, WIDE> {
    u32x4 w;
    __device__ __forceinline__ void load(const char *row, int c, int K) {
        if (c + 8 <= K) {
            if constexpr (WIDE) w = *(const u32x4 *) (row + (int64_t) c * 2);
            else w = *(const u32x4_any2 *) (row + (int64_t) c * 2);
            return;
        }
        const uint16_t *h = (const uint16_t *) row;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (c + 2 * e < K ? h[c + 2 * e] : 0u) | (c + 2 * e + 1 < K ? (uint32_t) h[c + 2 * e + 1] << 16 : 0u);
    }
    __device__ __forceinline__ uint32_t top() const {
        u16x2 t = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
        return (uint32_t) max(t[0], t[1]) << 16;
    }
    __device__ __forceinline__ void values(float *v) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
};

// NT threads a row, VN vectors of 8 values each in registers; rows longer than that
// (LONG) are read a second time. Up to 2048 values a row is a wave's or less, without LDS or
// barriers (32768 rows of 2000, bf16, on 256 threads each 73 us, on a wave 45.5, and 37.5 with
// bf16 in pairs), and rows of up to 256 have lanes for their own vectors only (100000 of 192: 44.5
// us with 64 lanes each, 19.2). Longer ones: 8192 rows of 4096 on 256 threads 21.9, on a wave
// 26.9; of 5120 on 256 threads 31.7, on 512 41.4; 8192 bf16 ones of 8192 on 256 threads 37.7, on 512
// 41.3, but 8 of them 4.3 and 3.6, and f32 ones 61.0 and 60.0.
template <bool BF16, bool WIDE, int VN, int NT, bool LONG>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void i8_quantize_kernel(const void *x, const Rows t, int64_t rows, int K, int64_t ld,
                                                                          int8_t *q, float *d) {
    __shared__ uint32_t red[NT > 64 ? (NT < 256 ? 256 : NT) / 64 : 1];
    constexpr int RW = NT < 256 ? 256 / NT : 1;
    const int th = threadIdx.x % NT;
    for (int64_t r0 = (int64_t) blockIdx.x * RW; r0 < rows; r0 += (int64_t) gridDim.x * RW) {
        const bool mine = r0 + threadIdx.x / NT < rows;
        const int64_t r = mine ? r0 + threadIdx.x / NT : rows - 1;
        const char *row = (const char *) x + row_at(t, r);
        Vec8<BF16, WIDE> v[VN];
        uint32_t top = 0;
        if constexpr (LONG) {
            // (64 bits: a step past a row of nearly 2^31 values is not below it)
            for (int64_t c = th * 8; c < K; c += NT * 8) {
                v[0].load(row, (int) c, K);
                top = max(top, v[0].top());
            }
        } else {
#pragma unroll
            for (int j = 0; j < VN; ++j) v[j].load(row, (th + NT * j) * 8, K);
#pragma unroll
            for (int j = 0; j < VN; ++j) top = max(top, v[j].top());
        }
        top = row_max<NT>(top, red);
        const I8Scale s = i8_scale(top);
        if (!mine) continue;
        auto store = [&](int c, const Vec8<BF16, WIDE> &x) {
            float w[8];
            x.values(w);
            if (c < ld) *(u32x2 *) (q + r * ld + c) = u32x2{i8_pack4(w, s), i8_pack4(w + 4, s)};
        };
        if constexpr (LONG) {
            for (int64_t c = th * 8; c < ld; c += NT * 8) {
                v[0].load(row, (int) c, K);
                store((int) c, v[0]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < VN; ++j) store((th + NT * j) * 8, v[j]);
        }
        if (th == 0) d[r] = s.d;
    }
}

template <bool BF16, bool WIDE>
hipError_t launch_quantize(const void *x, const Rows &t, int64_t rows, int K, int64_t ld, int8_t *q, float *d, hipStream_t s) {
    auto go = [&](auto kern, int nt) {
        const int rw = nt < 256 ? 256 / nt : 1, threads = nt < 256 ? 256 : nt;
        // (a launch holds fewer than 2^32 threads; the rows left are taken in turns)
        launch_kernel(kern, dim3((unsigned) std::min<int64_t>((rows + rw - 1) / rw, (1 << 30) / threads)), dim3(threads), 0, s, x, t, rows, K,
                      ld, q, d);
        return hipGetLastError();
    };
    if (ld <= 8 * 8) return go(i8_quantize_kernel<BF16, WIDE, 1, 8, false>, 8);
    if (ld <= 16 * 8) return go(i8_quantize_kernel<BF16, WIDE, 1, 16, false>, 16);
    if (ld <= 32 * 8) return go(i8_quantize_kernel<BF16, WIDE, 1, 32, false>, 32);
    if (ld <= 64 * 8) return go(i8_quantize_kernel<BF16, WIDE, 1, 64, false>, 64);
    if (ld <= 64 * 16) return go(i8_quantize_kernel<BF16, WIDE, 2, 64, false>, 64);
    if (ld <= 64 * 32) return go(i8_quantize_kernel<BF16, WIDE, 4, 64, false>, 64);
    if (ld <= 256 * 16) return go(i8_quantize_kernel<BF16, WIDE, 2, 256, false>, 256);
    if (ld <= 256 * 24) return go(i8_quantize_kernel<BF16, WIDE, 3, 256, false>, 256);
    if (BF16 && ld <= 256 * 32 && rows > 256) return go(i8_quantize_kernel<BF16, WIDE, 4, 256, false>, 256);
    if (ld <= 512 * 16) return go(i8_quantize_kernel<BF16, WIDE, 2, 512, false>, 512);
    if (ld <= 1024 * 16) return go(i8_quantize_kernel<BF16, WIDE, 2, 1024, false>, 1024);
    return go(i8_quantize_kernel<BF16, WIDE, 1, 1024, true>, 1024);
}

// A thread takes 8 values, and others a grid of threads on: step_r rows and step_c times 8
// values, P times 8 a row.
template <bool BF16, bool WIDE>
__global__ void i8_dequantize_kernel(const int8_t *q, const float *d, int64_t rows, int K, int P, int64_t step_r, int step_c, void *y,
                                     const Rows t) {
    const int64_t ld = i8_ld(K);
    const unsigned first = blockIdx.x * blockDim.x + threadIdx.x;
    int p = (int) (first % (unsigned) P);
    for (int64_t r = first / (unsigned) P; r < rows; r += step_r, p += step_c) {
        if (p >= P) {
            p -= P;
            if (++r >= rows) break;
        }
        const int c = p * 8;
        const u32x2 w = *(const u32x2 *) (q + r * ld + c);
        const float s = d[r];
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s * (float) (int8_t) (w[e >> 2] >> 8 * (e & 3));
        char *row = (char *) y + row_at(t, r);
        if (c + 8 <= K) {
            if constexpr (BF16) {
                const bf16x8 h = {(__bf16) v[0], (__bf16) v[1], (__bf16) v[2], (__bf16) v[3], (__bf16) v[4], (__bf16) v[5], (__bf16) v[6], (__bf16) v[7]};
                if constexpr (WIDE) *(bf16x8 *) (row + (int64_t) c * 2) = h;
                else *(u32x4_any2 *) (row + (int64_t) c * 2) = __builtin_bit_cast(u32x4, h);
            } else {
                const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
                typedef typename std::conditional<WIDE, f32x4, f32x4_any4>::type T;
                ((T *) (row + (int64_t) c * 4))[0] = a;
                ((T *) (row + (int64_t) c * 4))[1] = b;
            }
            continue;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < K) store_from_f32<BF16 ? Elt::BF16 : Elt::F32>(row, c + e, v[e]);
    }
}

Rows rows_of(const View4 &t) {
    Rows r;
    r.nb1 = t.nb[1]; r.nb2 = t.nb[2]; r.nb3 = t.nb[3];
    r.ne1 = (int) t.ne[1]; r.ne2 = (int) t.ne[2];
    r.flat = (t.ne[2] == 1 || t.nb[2] == t.nb[1] * t.ne[1]) && (t.ne[3] == 1 || t.nb[3] == t.nb[1] * t.ne[1] * t.ne[2]);
    return r;
}
bool on_16(const View4 &t) {
    bool ok = (uintptr_t) t.data % 16 == 0;
    for (int i = 1; i < 4; ++i) ok = ok && (t.ne[i] == 1 || t.nb[i] % 16 == 0);
    return ok;
}

}  // namespace

hipError_t launch_i8_quantize(const View4 &x, int8_t *q, float *d, hipStream_t s) {
    const int64_t rows = x.ne[1] * x.ne[2] * x.ne[3], ld = i8_ld(x.ne[0]);
    const int K = (int) x.ne[0];
    const Rows t = rows_of(x);
    const bool wide = on_16(x);
    if (x.type == TSK_TYPE_BF16)
        return wide ? launch_quantize<true, true>(x.data, t, rows, K, ld, q, d, s) : launch_quantize<true, false>(x.data, t, rows, K, ld, q, d, s);
    return wide ? launch_quantize<false, true>(x.data, t, rows, K, ld, q, d, s) : launch_quantize<false, false>(x.data, t, rows, K, ld, q, d, s);
}

hipError_t launch_i8_dequantize(const int8_t *q, const float *d, const View4 &y, hipStream_t s) {
    const int64_t rows = y.ne[1] * y.ne[2] * y.ne[3];
    const bool bf16 = y.type == TSK_TYPE_BF16, wide = on_16(y);
    const int K = (int) y.ne[0], P = (K + 7) / 8;
    const int64_t threads = std::min<int64_t>((rows * P + 255) / 256, 1 << 20) * 256;
    launch_kernel(bf16 ? wide ? i8_dequantize_kernel<true, true> : i8_dequantize_kernel<true, false>
                       : wide ? i8_dequantize_kernel<false, true> : i8_dequantize_kernel<false, false>,
                  dim3((unsigned) (threads / 256)), dim3(256), 0, s, q, d, rows, K, P, threads / P, (int) (threads % P), (void *) y.data,
                  rows_of(y));
    return hipGetLastError();
}

}  // namespace tsk
