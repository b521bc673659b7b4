// block_norm.hip — the norms, gate and residual between two blocks' matrices
// (x + gate * y, ggml_norm and modulate of src/mmdit.cpp:55-59, :231-234):
//
//   r   = res_scale * x + gate * post(y),  res = r in x's type
//   dst = pre(res) * pre_w * (1 + scale) + shift    (f32, bf16 or MXFP4)
//
// Bound by memory: x and y are read once, res and dst written once (16384 bf16 rows
// of 4096 with both norms 123 us, 4.4 TB/s; 16384 f32 rows of 2048 with gate, scale
// and shift 111 us, 4.9 TB/s; 388 f32 rows of 1024 5.1 us, the launch). A row's
// values stay in the registers of one wave or workgroup between its passes:
// the branch's statistics (mean, then the squared deviations from it), the
// sum, the sum's statistics, the output.
#include <algorithm>

#include "mxfp4.h"
#include "tsk_internal.h"

// Products and sums are rounded one at a time in this file, but where it writes
// __builtin_fmaf: an element goes through the same operations in every kernel, and
// the second norm reads the residual that is stored.
#pragma clang fp contract(off)

namespace tsk {

namespace {

__device__ __forceinline__ float as_type(float v, int bf16) { return bf16 ? bf16_bits_to_f32(f32_to_bf16_bits(v)) : v; }

__device__ __forceinline__ char *row_of(const BnView &t, int i1, int i2, int i3) {
    return (char *) const_cast<void *>(t.data) + i1 * t.nb1 + i2 * t.nb2 + i3 * t.nb3;
}

// ---- V elements at a time: 8 as 16-byte accesses, or 1
template <int V>
__device__ __forceinline__ void load_f32(const float *p, float *v) {
    if constexpr (V == 1) {
        v[0] = p[0];
    } else {
        const f32x4 a = ((const f32x4 *) p)[0], b = ((const f32x4 *) p)[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = a[e];
            v[4 + e] = b[e];
        }
    }
}
template <int V>
__device__ __forceinline__ void load_bf16(const uint16_t *p, float *v) {
    if constexpr (V == 1) {
        v[0] = bf16_bits_to_f32(p[0]);
    } else {
        const u32x4 w = *(const u32x4 *) p;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[2 * q] = __uint_as_float(w[q] << 16);
            v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
        }
    }
}
template <int V>
__device__ __forceinline__ void store_f32(float *p, const float *v) {
    if constexpr (V == 1) {
        p[0] = v[0];
    } else {
        ((f32x4 *) p)[0] = f32x4{v[0], v[1], v[2], v[3]};
        ((f32x4 *) p)[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
}
template <int V>
__device__ __forceinline__ void store_bf16(uint16_t *p, const float *v) {
    if constexpr (V == 1) {
        p[0] = f32_to_bf16_bits(v[0]);
    } else {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = f32_to_bf16_bits(v[2 * q]) | (uint32_t) f32_to_bf16_bits(v[2 * q + 1]) << 16;
        *(u32x4 *) p = w;
    }
}

// ---- the arithmetic
__device__ __forceinline__ float branch(float y, int norm, float mean, float inv, bool has_w, float w) {
    const float b = norm ? (y - mean) * inv : y;
    return has_w ? b * w : b;
}
__device__ __forceinline__ float residual(float x, float s, float b, bool has_gate, float gate) {
    const float sx = s * x;
    return has_gate ? __builtin_fmaf(gate, b, sx) : sx + b;
}
__device__ __forceinline__ float modulated(float r, int norm, float mean, float inv, bool has_w, float w, bool has_scale,
                                           float scale, bool has_shift, float shift) {
    float h = norm ? (r - mean) * inv : r;
    if (has_w) h *= w;
    const float f = has_scale ? 1.0f + scale : 1.0f;
    return has_shift ? __builtin_fmaf(h, f, shift) : h * f;
}

// sum over the NT threads of a row: 16, 32 or 64 lanes of a wave (every lane of
// it active), or NT / 64 waves, whose sums meet in red; `turn` alternates
// between its halves, so that one barrier a sum is enough
template <int NT>
__device__ __forceinline__ float row_sum(float v, float *red, int &turn) {
    if constexpr (NT == 16) return row16_sum(v);
    if constexpr (NT == 32) return row_pair_sum(row16_sum(v));
    v = wave_sum(v);
    if constexpr (NT > 64) {
        float *half = red + (turn ^= 1) * (NT / 64);
        if ((threadIdx.x & 63) == 0) half[threadIdx.x % NT >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) v += half[i];
    }
    return v;
}

// One row: thread t holds the V-vectors t, t + NT, ..., VN of them at most.
// mean and 1 / sqrt(var + eps) of the C values (LAYER), or 0 and 1 / sqrt(mean of squares + eps) (RMS)
template <int V, int VN, int NT>
__device__ __forceinline__ void row_stats(int kind, int C, float eps, int t, const float (&v)[VN][V], float *red, int &turn,
                                          float &mean, float &inv) {
    mean = 0.0f;
    inv = 1.0f;
    if (kind == TSK_NORM_NONE) return;
    if (kind == TSK_NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < VN; ++j)
            if ((t + NT * j) * V < C)
#pragma unroll
                for (int e = 0; e < V; ++e) s += v[j][e];
        mean = row_sum<NT>(s, red, turn) / (float) C;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < VN; ++j)
        if ((t + NT * j) * V < C)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = v[j][e] - mean;
                q = __builtin_fmaf(d, d, q);
            }
    inv = 1.0f / sqrtf(row_sum<NT>(q, red, turn) / (float) C + eps);
}

// V vectors of a row into v (f32 or bf16)
template <int V, int VN, int NT>
__device__ __forceinline__ void load_row(const void *row, int bf16, int C, int t, float (&v)[VN][V]) {
    if (bf16) {
#pragma unroll
        for (int j = 0; j < VN; ++j)
            if ((t + NT * j) * V < C) load_bf16<V>((const uint16_t *) row + (t + NT * j) * V, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VN; ++j)
            if ((t + NT * j) * V < C) load_f32<V>((const float *) row + (t + NT * j) * V, v[j]);
    }
}
template <int V, int VN, int NT>
__device__ __forceinline__ void store_row(void *row, int bf16, int C, int t, const float (&v)[VN][V]) {
    if (bf16) {
#pragma unroll
        for (int j = 0; j < VN; ++j)
            if ((t + NT * j) * V < C) store_bf16<V>((uint16_t *) row + (t + NT * j) * V, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VN; ++j)
            if ((t + NT * j) * V < C) store_f32<V>((float *) row + (t + NT * j) * V, v[j]);
    }
}

// NT threads a row (fewer than 256: 256 / NT rows a workgroup), its values in
// registers. What a pass needs beside them (WTS: weights, MOD: gate, scale and
// shift) is loaded before the statistics that it waits for.
template <int V, int VN, int NT, bool WTS, bool MOD>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void block_norm_kernel(const BlockNorm p) {
    __shared__ float red[NT > 64 ? (NT < 256 ? 256 / NT : 1) * 2 * (NT / 64) : 1];
    constexpr int RW = NT < 256 ? 256 / NT : 1;                      // rows of a workgroup
    const int t = threadIdx.x % NT, C = p.C;
    float *my_red = red + (NT > 64 ? threadIdx.x / NT * 2 * (NT / 64) : 0);
    int turn = 0;
    const int64_t rows = (int64_t) p.n1 * p.n2 * p.n3;
    for (int64_t r0 = (int64_t) blockIdx.x * RW; r0 < rows; r0 += (int64_t) gridDim.x * RW) {
        // (threads past the last row work on it again and store nothing)
        const int64_t r = std::min<int64_t>(r0 + threadIdx.x / NT, rows - 1);
        const bool mine = r0 + threadIdx.x / NT < rows;
        const int i1 = (int) (r % p.n1), i2 = (int) (r / p.n1 % p.n2), i3 = (int) (r / p.n1 / p.n2);
        const bool has_y = p.y.data, has_gate = MOD && p.gate.data, has_scale = MOD && p.scale.data, has_shift = MOD && p.shift.data;
        const bool has_post_w = WTS && p.post_w, has_pre_w = WTS && p.pre_w;
        const bool has_out = p.dst.data || p.scales;
        float x[VN][V], y[VN][V], w[VN][V] = {}, f[VN][V] = {}, h[VN][V] = {}, mean, inv;
        load_row<V, VN, NT>(row_of(p.x, i1, i2, i3), p.x_bf16, C, t, x);
        if (has_y) {
            load_row<V, VN, NT>(row_of(p.y, i1, i2, i3), p.y_bf16, C, t, y);
            if (has_post_w) load_row<V, VN, NT>(p.post_w, 0, C, t, w);
            if (has_gate) load_row<V, VN, NT>(row_of(p.gate, i1, i2, i3), 0, C, t, f);
            row_stats<V, VN, NT>(p.post_norm, C, p.post_eps, t, y, my_red, turn, mean, inv);
#pragma unroll
            for (int j = 0; j < VN; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float b = branch(y[j][e], p.post_norm, mean, inv, has_post_w, w[j][e]);
                    x[j][e] = as_type(residual(x[j][e], p.res_scale, b, has_gate, f[j][e]), p.x_bf16);
                }
        } else {
#pragma unroll
            for (int j = 0; j < VN; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) x[j][e] = as_type(p.res_scale * x[j][e], p.x_bf16);
        }
        if (has_out) {
            if (has_pre_w) load_row<V, VN, NT>(p.pre_w, 0, C, t, w);
            if (has_scale) load_row<V, VN, NT>(row_of(p.scale, i1, i2, i3), 0, C, t, f);
            if (has_shift) load_row<V, VN, NT>(row_of(p.shift, i1, i2, i3), 0, C, t, h);
        }
        if (p.res.data && mine) store_row<V, VN, NT>(row_of(p.res, i1, i2, i3), p.x_bf16, C, t, x);
        if (!has_out) continue;
        row_stats<V, VN, NT>(p.pre_norm, C, p.pre_eps, t, x, my_red, turn, mean, inv);
#pragma unroll
        for (int j = 0; j < VN; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e)
                x[j][e] = modulated(x[j][e], p.pre_norm, mean, inv, has_pre_w, w[j][e], has_scale, f[j][e], has_shift, h[j][e]);
        if (p.dst.data) {
            if (mine) store_row<V, VN, NT>(row_of(p.dst, i1, i2, i3), p.dst_bf16, C, t, x);
        } else if constexpr (V == 8) {
            // a block of 32 is four threads' vectors (C % 32 == 0: all four hold one, or none)
#pragma unroll
            for (int j = 0; j < VN; ++j) {
                const int c = (t + NT * j) * V;
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) top = max(top, mx_abs_bits(x[j][e]));
                top = mx_quad_max(top);
                if (c >= C || !mine) continue;
                const uint32_t byte = mx_scale_byte(top);
                *(uint32_t *) (p.codes + r * (C / 2) + c / 2) = byte == 255u ? 0u : mx_encode8(x[j], mx_scale(byte));
                if ((t & 3) == 0) p.scales[r * (C / 32) + c / 32] = (uint8_t) byte;
            }
        }
    }
}

// Rows of any length, read from memory again in every pass, one value a load:
// longer ones than the registers of a workgroup hold (2000 bf16 rows of 16384, the
// longest that they hold, 71 us, 3.7 TB/s; of 16416, here, 456), and MXFP4 outputs
// of rows that are not aligned to 16 bytes (a thread holds whole blocks there, a
// lane of the register kernel one value: 16384 bf16 rows of 4096 1043 us, on 16-byte
// starts 124; f32 rows of 1024 325 and 36).
__device__ __forceinline__ float load_elt(const void *row, int bf16, int i) {
    return bf16 ? bf16_bits_to_f32(((const uint16_t *) row)[i]) : ((const float *) row)[i];
}
template <class F>
__device__ __forceinline__ void long_stats(int kind, int C, float eps, float *red, int &turn, F f, float &mean, float &inv) {
    mean = 0.0f;
    inv = 1.0f;
    if (kind == TSK_NORM_NONE) return;
    if (kind == TSK_NORM_LAYER) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < C; i += 256) s += f(i);
        mean = row_sum<256>(s, red, turn) / (float) C;
    }
    float q = 0.0f;
    for (int i = threadIdx.x; i < C; i += 256) {
        const float d = f(i) - mean;
        q = __builtin_fmaf(d, d, q);
    }
    inv = 1.0f / sqrtf(row_sum<256>(q, red, turn) / (float) C + eps);
}
__global__ __launch_bounds__(256) void block_norm_long_kernel(const BlockNorm p) {
    __shared__ float red[8];
    int turn = 0;
    const int C = p.C;
    const int64_t rows = (int64_t) p.n1 * p.n2 * p.n3;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int i1 = (int) (r % p.n1), i2 = (int) (r / p.n1 % p.n2), i3 = (int) (r / p.n1 / p.n2);
        const char *x = row_of(p.x, i1, i2, i3), *y = p.y.data ? row_of(p.y, i1, i2, i3) : nullptr;
        const float *gate = p.gate.data ? (const float *) row_of(p.gate, i1, i2, i3) : nullptr;
        const float *scale = p.scale.data ? (const float *) row_of(p.scale, i1, i2, i3) : nullptr;
        const float *shift = p.shift.data ? (const float *) row_of(p.shift, i1, i2, i3) : nullptr;
        float ymean = 0.0f, yinv = 1.0f, mean, inv;
        if (y) long_stats(p.post_norm, C, p.post_eps, red, turn, [&](int i) { return load_elt(y, p.y_bf16, i); }, ymean, yinv);
        auto sum = [&](int i) {
            const float xv = load_elt(x, p.x_bf16, i);
            if (!y) return as_type(p.res_scale * xv, p.x_bf16);
            const float b = branch(load_elt(y, p.y_bf16, i), p.post_norm, ymean, yinv, p.post_w, p.post_w ? p.post_w[i] : 0.0f);
            return as_type(residual(xv, p.res_scale, b, gate, gate ? gate[i] : 0.0f), p.x_bf16);
        };
        if (p.dst.data || p.scales) {
            long_stats(p.pre_norm, C, p.pre_eps, red, turn, sum, mean, inv);
            auto out = [&](int i) {
                return modulated(sum(i), p.pre_norm, mean, inv, p.pre_w, p.pre_w ? p.pre_w[i] : 0.0f, scale,
                                 scale ? scale[i] : 0.0f, shift, shift ? shift[i] : 0.0f);
            };
            if (p.scales) {
                for (int kb = threadIdx.x; kb < C / 32; kb += 256) {
                    float v[32];
                    uint32_t top = 0;
                    for (int j = 0; j < 32; ++j) {
                        v[j] = out(kb * 32 + j);
                        top = max(top, mx_abs_bits(v[j]));
                    }
                    const uint32_t byte = mx_scale_byte(top);
                    u32x4 w;
                    for (int h = 0; h < 4; ++h) w[h] = byte == 255u ? 0u : mx_encode8(v + 8 * h, mx_scale(byte));
                    *(u32x4 *) (p.codes + r * (C / 2) + kb * 16) = w;
                    p.scales[r * (C / 32) + kb] = (uint8_t) byte;
                }
            } else {
                char *d = row_of(p.dst, i1, i2, i3);
                for (int i = threadIdx.x; i < C; i += 256) {
                    if (p.dst_bf16) ((uint16_t *) d)[i] = f32_to_bf16_bits(out(i));
                    else ((float *) d)[i] = out(i);
                }
            }
        }
        if (p.res.data) {
            __syncthreads();                              // (res may be x: every thread has read the row)
            char *d = row_of(p.res, i1, i2, i3);
            for (int i = threadIdx.x; i < C; i += 256) {
                const float v = sum(i);
                if (p.x_bf16) ((uint16_t *) d)[i] = f32_to_bf16_bits(v);
                else ((float *) d)[i] = v;
            }
        }
    }
}

template <int V, int VN, int NT>
hipError_t launch_bn(const BlockNorm &p, int64_t rows, hipStream_t s) {
    constexpr int RW = NT < 256 ? 256 / NT : 1;
    const bool wts = p.post_w || p.pre_w, mod = p.gate.data || p.scale.data || p.shift.data;
    launch_kernel(wts ? mod ? block_norm_kernel<V, VN, NT, true, true> : block_norm_kernel<V, VN, NT, true, false>
                      : mod ? block_norm_kernel<V, VN, NT, false, true> : block_norm_kernel<V, VN, NT, false, false>,
                  dim3((unsigned) std::min<int64_t>((rows + RW - 1) / RW, 1 << 20)), dim3(NT < 256 ? 256 : NT), 0, s, p);
    return hipGetLastError();
}

template <int V, int NT>
hipError_t launch_nt(const BlockNorm &p, int64_t rows, hipStream_t s) {
    constexpr int MANY = V == 8 ? 2 : 8, FEW = MANY / 2;
    return p.C > V * NT * FEW ? launch_bn<V, MANY, NT>(p, rows, s) : launch_bn<V, FEW, NT>(p, rows, s);
}

// Threads a row: as few as hold it in 16 values each (8 where they come
// alone); more cost occupancy, fewer a longer chain of sums (us, each pair on one
// build: 16384 bf16 rows of 4096, 256 threads 138, 128 of 32 values 190, 512 145;
// 16384 of 1024, 64 threads 32.6, 256 51; 8192 f32 rows of 256, 16 threads 9.7, 64
// 11.3). Where the rows leave CUs idle, twice as many each time (388 f32 rows of
// 1024: 64 threads 5.3, 128 4.7, 256 5.2).
template <int V>
hipError_t launch_v(const BlockNorm &p, int64_t rows, hipStream_t s) {
    constexpr int MOST = V == 8 ? 16 : 8;
    const int n = (p.C + V - 1) / V;
    int nt = 16;
    while (nt < 1024 && p.C > MOST * nt) nt *= 2;
    while (nt < 1024 && rows * nt < 32768 && n > nt) nt *= 2;
    if (p.C <= MOST * nt) {
        switch (nt) {
            case 16: return launch_nt<V, 16>(p, rows, s);
            case 32: return launch_nt<V, 32>(p, rows, s);
            case 64: return launch_nt<V, 64>(p, rows, s);
            case 128: return launch_nt<V, 128>(p, rows, s);
            case 256: return launch_nt<V, 256>(p, rows, s);
            case 512: return launch_nt<V, 512>(p, rows, s);
            default: return launch_nt<V, 1024>(p, rows, s);
        }
    }
    launch_kernel(block_norm_long_kernel, dim3((unsigned) std::min<int64_t>(rows, 1 << 20)), dim3(256), 0, s, p);
    return hipGetLastError();
}

bool rows_on_16(const BnView &t) {
    return !t.data || ((uintptr_t) t.data % 16 == 0 && t.nb1 % 16 == 0 && t.nb2 % 16 == 0 && t.nb3 % 16 == 0);
}

}  // namespace

hipError_t launch_block_norm(const BlockNorm &p, hipStream_t s) {
    const int64_t rows = (int64_t) p.n1 * p.n2 * p.n3;
    // vectors of 8 where every row is whole vectors on 16-byte starts
    bool wide = p.C % 8 == 0 && (uintptr_t) p.post_w % 16 == 0 && (uintptr_t) p.pre_w % 16 == 0;
    for (const BnView *t : {&p.x, &p.y, &p.gate, &p.scale, &p.shift, &p.res, &p.dst}) wide = wide && rows_on_16(*t);
    if (wide) return launch_v<8>(p, rows, s);
    if (p.scales) {
        launch_kernel(block_norm_long_kernel, dim3((unsigned) std::min<int64_t>(rows, 1 << 20)), dim3(256), 0, s, p);
        return hipGetLastError();
    }
    return launch_v<1>(p, rows, s);
}

}  // namespace tsk
