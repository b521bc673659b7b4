// rope_axes.hip — rotary positions over several axes (time, height, width, ...), with
// the RMS norm of every head before them where it has one.
//
// Each pair (a, b) of a head belongs to an axis and becomes (a cos t - b sin t,
// a sin t + b cos t), t = position on that axis * the pair's frequency. The angle is
// formed in 64 bits as quarter turns, of which the fraction alone is kept: positions of
// 2^20 and more keep 24 bits of their angle, where an fp32 product would lose all but a
// few. Bound by memory: x is read and y written once; a lane forms the sines and cosines of its
// pairs once and uses them for every head that it turns.
#include <algorithm>

#include "tsk_common.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

// cos and sin of q quarter turns: the nearest whole quarter apart, Taylor's series of the
// rest, at most an eighth of a turn (the first terms left out: 1.2e-10 and 1.8e-9)
__device__ __forceinline__ void cos_sin(double q, float &c, float &s) {
    const double n = __builtin_rint(q);
    const float f = (float) (q - n) * 1.57079632679489662f, f2 = f * f;
    const float sn = f + f * f2 * (-1.0f / 6 + f2 * (1.0f / 120 + f2 * (-1.0f / 5040 + f2 * (1.0f / 362880))));
    const float cn = 1.0f + f2 * (-0.5f + f2 * (1.0f / 24 + f2 * (-1.0f / 720 + f2 * (1.0f / 40320 + f2 * (-1.0f / 3628800)))));
    // n modulo 4 (n is whole; of 2^53 and more it is a multiple of 4 or may as well be one)
    const int k = (int) (n - 4.0 * __builtin_floor(n * 0.25));
    const float a = k & 1 ? sn : cn, b = k & 1 ? cn : sn;
    c = k == 1 || k == 2 ? -a : a;
    s = k & 2 ? -b : b;
    if (!(__builtin_fabs(q) < __builtin_inf())) c = s = __uint_as_float(0x7fc00000u);
}

// A lane holds 8 values of a head: ADJ the 8 from 8 j on; else the pairs 4 j .. 4 j + 3
// (values 4 j + e and n / 2 + 4 j + e), and past the pairs the 8 from n + 8 (j - J) on.
struct Lane {
    int lo, hi, nlo, nhi;          // first indices and counts of its two runs of 4
    int pair;                      // first pair, of np that are turned
    int np;
};
__device__ __forceinline__ Lane lane_of(const RopeAxes &p, int D, int j) {
    Lane l;
    auto within = [](int n, int most) { return n < 0 ? 0 : n < most ? n : most; };
    const int h = p.n / 2, J = (h + 3) / 4;
    if (p.halves && j < J) {
        l.lo = 4 * j;
        l.hi = h + 4 * j;
        l.nlo = l.nhi = within(h - 4 * j, 4);
        l.pair = 4 * j;
        l.np = l.nlo;
        return l;
    }
    l.lo = p.halves ? p.n + 8 * (j - J) : 8 * j;
    l.hi = l.lo + 4;
    l.nlo = within(D - l.lo, 4);
    l.nhi = within(D - l.hi, 4);
    l.pair = l.lo / 2;
    l.np = p.halves ? 0 : within(h - l.pair, 4);
    return l;
}

template <bool BF16, bool WIDE>
__device__ __forceinline__ void load_run(const char *row, int i, int n, float *v) {
    if constexpr (WIDE) {
        if (n) {
            if constexpr (BF16) {
                const u32x2 w = *(const u32x2 *) (row + i * 2);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    v[2 * q] = __uint_as_float(w[q] << 16);
                    v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
                }
            } else {
                const f32x4 a = *(const f32x4 *) (row + i * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = a[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = 0.0f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < n ? load_as_f32<BF16 ? Elt::BF16 : Elt::F32>(row, i + e) : 0.0f;
    }
}
template <bool BF16, bool WIDE>
__device__ __forceinline__ void store_run(char *row, int i, int n, const float *v) {
    if constexpr (WIDE) {
        if (!n) return;
        if constexpr (BF16)
            *(u32x2 *) (row + i * 2) = u32x2{f32_to_bf16_bits(v[0]) | (uint32_t) f32_to_bf16_bits(v[1]) << 16,
                                            f32_to_bf16_bits(v[2]) | (uint32_t) f32_to_bf16_bits(v[3]) << 16};
        else *(f32x4 *) (row + i * 4) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) store_from_f32<BF16 ? Elt::BF16 : Elt::F32>(row, i + e, v[e]);
    }
}

// LPH lanes a head, 64 / LPH heads a wave at a time; a wave takes HW heads of one token.
template <bool XBF16, bool YBF16, bool WIDE, int LPH>
__global__ __launch_bounds__(256) void rope_axes_kernel(const RopeAxes p, int chunks, int heads_a_wave) {
    const int lane = threadIdx.x & 63, j = lane % LPH, D = (int) p.x.ne[0], H = (int) p.x.ne[1];
    const int64_t S = p.x.ne[2], units = S * p.x.ne[3] * chunks;
    const Lane l = lane_of(p, D, j);
    float w[8] = {};
    if (p.w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = e < l.nlo ? p.w[l.lo + e] : 0.0f;
            w[4 + e] = e < l.nhi ? p.w[l.hi + e] : 0.0f;
        }
    }
    for (int64_t u = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += (int64_t) gridDim.x * 4) {
        const int64_t tok = u / chunks, s = tok % S, b = tok / S;
        const int h0 = (int) (u % chunks) * heads_a_wave, h1 = min(H, h0 + heads_a_wave);
        float c[4], sn[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = 1.0f;
            sn[e] = 0.0f;
            if (e >= l.np) continue;
            const int i = l.pair + e;
            int a = 0;
            for (int t = 1; t < p.n_axes; ++t) a += i >= p.first[t];
            const char *at = (const char *) p.pos + a * p.pos_nb1 + b * p.pos_nb2 + s * 4;
            const double x = p.pos_f32 ? (double) *(const float *) at : (double) *(const int32_t *) at;
            cos_sin(x * p.quarters[i], c[e], sn[e]);
        }
        const char *xr = (const char *) p.x.data + s * p.x.nb[2] + b * p.x.nb[3];
        char *yr = (char *) p.y.data + s * p.y.nb[2] + b * p.y.nb[3];
        for (int hb = h0; hb < h1; hb += 64 / LPH) {
            const int h = hb + lane / LPH;
            const bool mine = h < h1;
            float v[8];
            const char *row = xr + (int64_t) (mine ? h : h1 - 1) * p.x.nb[1];
            load_run<XBF16, WIDE>(row, l.lo, l.nlo, v);
            load_run<XBF16, WIDE>(row, l.hi, l.nhi, v + 4);
            if (p.w) {
                float q = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) q = __builtin_fmaf(v[e], v[e], q);
#pragma unroll
                for (int m = 1; m < LPH; m *= 2) q += __shfl_xor(q, m);
                const float inv = 1.0f / sqrtf(q / (float) D + p.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * w[e];
            }
            float o[8];
            if (p.halves) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] = e < l.np ? v[e] * c[e] - v[4 + e] * sn[e] : v[e];
                    o[4 + e] = e < l.np ? v[e] * sn[e] + v[4 + e] * c[e] : v[4 + e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[2 * e] = e < l.np ? v[2 * e] * c[e] - v[2 * e + 1] * sn[e] : v[2 * e];
                    o[2 * e + 1] = e < l.np ? v[2 * e] * sn[e] + v[2 * e + 1] * c[e] : v[2 * e + 1];
                }
            }
            if (!mine) continue;
            char *out = yr + (int64_t) h * p.y.nb[1];
            store_run<YBF16, WIDE>(out, l.lo, l.nlo, o);
            store_run<YBF16, WIDE>(out, l.hi, l.nhi, o + 4);
        }
    }
}

template <bool XBF16, bool YBF16, bool WIDE>
hipError_t launch_lph(const RopeAxes &p, hipStream_t s) {
    const int D = (int) p.x.ne[0], H = (int) p.x.ne[1];
    const int groups = p.halves ? (p.n / 2 + 3) / 4 + (D - p.n + 7) / 8 : (D + 7) / 8;
    int lph = 1;
    while (lph < groups) lph *= 2;
    const int64_t tokens = p.x.ne[2] * p.x.ne[3];
    const int chunks = 1, heads = H;
    const int64_t units = tokens * chunks;
    const dim3 grid((unsigned) std::min<int64_t>((units + 3) / 4, 1 << 22));
    auto go = [&](auto kern) {
        launch_kernel(kern, grid, dim3(256), 0, s, p, chunks, heads);
        return hipGetLastError();
    };
    switch (lph) {
        case 1: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 1>);
        case 2: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 2>);
        case 4: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 4>);
        case 8: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 8>);
        case 16: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 16>);
        case 32: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 32>);
        default: return go(rope_axes_kernel<XBF16, YBF16, WIDE, 64>);
    }
}

bool rows_on(const View4 &t, int64_t bytes) {
    bool ok = (uintptr_t) t.data % bytes == 0;
    for (int i = 1; i < 4; ++i) ok = ok && (t.ne[i] == 1 || t.nb[i] % bytes == 0);
    return ok;
}

}  // namespace

hipError_t launch_rope_axes(const RopeAxes &p, hipStream_t s) {
    const int D = (int) p.x.ne[0];
    const bool xb = p.x.type == TSK_TYPE_BF16, yb = p.y.type == TSK_TYPE_BF16;
    // runs of 4 values on 4-value starts, whole ones
    const bool wide = rows_on(p.x, xb ? 8 : 16) && rows_on(p.y, yb ? 8 : 16) && D % 4 == 0 && (!p.halves || p.n % 8 == 0);
    auto go = [&](auto x, auto y) {
        return wide ? launch_lph<decltype(x)::value, decltype(y)::value, true>(p, s)
                    : launch_lph<decltype(x)::value, decltype(y)::value, false>(p, s);
    };
    std::true_type t;
    std::false_type f;
    return xb ? yb ? go(t, t) : go(t, f) : yb ? go(f, t) : go(f, f);
}

}  // namespace tsk
