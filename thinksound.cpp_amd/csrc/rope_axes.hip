// rope_axes.hip — rotary positions over several axes (time, height, width, ...), with
// the RMS norm of every head before them where it has one.
//
// Each pair (a, b) of a head belongs to an axis and becomes (a cos t - b sin t,
// a sin t + b cos t), t = position on that axis * the pair's frequency. The angle is
// formed in 64 bits as quarter turns, of which the fraction alone is kept: positions of
// 2^20 and more keep 24 bits of their angle, where an fp32 product would lose all but a
// few. Bound by memory: x is read and y written once. A vector instruction of a wave takes
// four cycles, so that some 500 of them a token are as long as its memory: each angle is formed
// by one lane of the wave and used for all heads, the values stay as loaded until their turn,
// and a wave goes on to other tokens. 16384 tokens of 16 heads of 128, bf16, x in no cache: 26.3 us, 5.1 TB/s (calls that
// follow one another 27.8, copies as long 26.3; angles formed by each lane for its own pairs 35.8, and one pass of heads
// in flight 42).
#include <algorithm>

#include "tsk_common.h"
#include "tsk_internal.h"

namespace tsk {

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4;
// vectors that start on any value: the memory takes them whole too (16384 tokens of 16 heads of
// 126, bf16: value by value 76.5 us, in vectors 41.9)
typedef __attribute__((__vector_size__(8), aligned(2))) uint32_t u32x2_any2;
typedef __attribute__((__vector_size__(8), aligned(2))) __bf16 bf16x4_any2;
typedef __attribute__((__vector_size__(16), aligned(4))) float f32x4_any4;

// cos and sin of pos * freq quarter turns: the nearest whole quarter apart, Taylor's series of the
// rest, at most an eighth of a turn (the first terms left out: 1.2e-10 and 1.8e-9). The rest is the exact
// product's; where the rounded one is off by a quarter and more itself, from 2^51 on, the rounded one's
__device__ __forceinline__ void cos_sin(double pos, double freq, float &c, float &s) {
    const double q = pos * freq, n = __builtin_rint(q), rest = __builtin_fabs(q) < 0x1p51 ? __builtin_fma(pos, freq, -n) : 0.0;
    const float f = (float) rest * 1.57079632679489662f, f2 = f * f;
    const float sn = f + f * f2 * (-1.0f / 6 + f2 * (1.0f / 120 + f2 * (-1.0f / 5040 + f2 * (1.0f / 362880))));
    const float cn = 1.0f + f2 * (-0.5f + f2 * (1.0f / 24 + f2 * (-1.0f / 720 + f2 * (1.0f / 40320 + f2 * (-1.0f / 3628800)))));
    // n modulo 4 (n is whole; of 2^53 and more it is a multiple of 4 or may as well be one)
    const int k = (int) (n - 4.0 * __builtin_floor(n * 0.25));
    const float a = k & 1 ? sn : cn, b = k & 1 ? cn : sn;
    c = k == 1 || k == 2 ? -a : a;
    s = k & 2 ? -b : b;
    if (!(__builtin_fabs(q) < __builtin_inf())) c = s = __uint_as_float(0x7fc00000u);
}

// A lane holds 8 values of a head in two runs of 4: adjacent pairs, the 8 from 8 j on; pairs
// of halves, the pairs 4 j .. 4 j + 3 (values 4 j + e and n / 2 + 4 j + e), and past the
// pairs the 8 from n + 8 (j - J) on.
struct Lane {
    int lo, hi, nlo, nhi;          // first indices and counts of its runs
    int pair, np;                  // first pair, number of pairs that are turned
};
template <bool HALVES>
__device__ __forceinline__ Lane lane_of(const RopeAxes &p, int D, int j) {
    Lane l;
    auto within = [](int n, int most) { return n < 0 ? 0 : n < most ? n : most; };
    const int h = p.n / 2, J = (h + 3) / 4;
    if (HALVES && j < J) {
        l.lo = 4 * j;
        l.hi = h + 4 * j;
        l.nlo = l.nhi = within(h - 4 * j, 4);
        l.pair = 4 * j;
        l.np = l.nlo;
        return l;
    }
    l.lo = HALVES ? p.n + 8 * (j - J) : 8 * j;
    l.hi = l.lo + 4;
    l.nlo = within(D - l.lo, 4);
    l.nhi = within(D - l.hi, 4);
    l.pair = l.lo / 2;
    l.np = HALVES ? 0 : within(h - l.pair, 4);
    return l;
}

// A run as it is loaded. WIDE: it is whole or empty, and an empty one reads the row's first
// values; else it starts on any value, and a part of one is read value by value.
template <bool BF16, bool WIDE> struct Run {
    typename std::conditional<BF16, u32x2, f32x4>::type raw;
    __device__ __forceinline__ void load(const char *row, int i, int n) {
        if constexpr (WIDE) raw = *(const decltype(raw) *) (row + (n ? i * (BF16 ? 2 : 4) : 0));
        else if (n == 4) raw = *(const typename std::conditional<BF16, u32x2_any2, f32x4_any4>::type *) (row + i * (BF16 ? 2 : 4));
        else if constexpr (BF16) {
            const uint16_t *h = (const uint16_t *) row;
            raw[0] = h[0 < n ? i : 0] | (uint32_t) h[1 < n ? i + 1 : 0] << 16;
            raw[1] = h[2 < n ? i + 2 : 0];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) raw[e] = ((const float *) row)[e < n ? i + e : 0];
        }
    }
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (BF16) return __uint_as_float(e & 1 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
        else return raw[e];
    }
};
template <bool BF16, bool WIDE>
__device__ __forceinline__ void store_run(char *row, int i, int n, const float *v) {
    if (n == 4) {
        if constexpr (BF16) {
            const bf16x4 h = {(__bf16) v[0], (__bf16) v[1], (__bf16) v[2], (__bf16) v[3]};
            *(typename std::conditional<WIDE, bf16x4, bf16x4_any2>::type *) (row + i * 2) = h;
        } else *(typename std::conditional<WIDE, f32x4, f32x4_any4>::type *) (row + i * 4) = f32x4{v[0], v[1], v[2], v[3]};
        return;
    }
    if constexpr (!WIDE) {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < n) store_from_f32<BF16 ? Elt::BF16 : Elt::F32>(row, i + e, v[e]);
    }
}

// 1 / sqrt(x), x >= 0, within 1 ulp (v_rsq_f32) also below the normal numbers
__device__ __forceinline__ float inverse_root(float x) {
    const bool tiny = x < 0x1p-96f;
    return __builtin_amdgcn_rsqf(tiny ? x * 0x1p64f : x) * (tiny ? 0x1p32f : 1.0f);
}

// One wave a workgroup: LPH lanes a head, so HPW = 64 / LPH heads a pass, U passes in flight
// (16384 tokens as above, U = 1: 28.1 us, 4: 26.7); blockIdx.y takes heads_a_wave heads of a
// token. The lanes form one angle each and hand the sines and cosines around through LDS, while
// the first heads are on their way. (Four waves a workgroup: 27.3 us.)
constexpr int U = 4;
template <bool XBF16, bool YBF16, bool WIDE, bool HALVES, int LPH>
__global__ __launch_bounds__(64) void rope_axes_kernel(const RopeAxes p, int heads_a_wave) {
    __shared__ alignas(16) float cosines[ROPE_AXES_PAIRS], sines[ROPE_AXES_PAIRS];
    constexpr int HPW = 64 / LPH;
    const int lane = threadIdx.x, hl = lane / LPH, D = (int) p.x.ne[0], H = (int) p.x.ne[1];
    const Lane l = lane_of<HALVES>(p, D, lane % LPH);
    const int h0 = (int) blockIdx.y * heads_a_wave, h1 = h0 + min(heads_a_wave, H - h0);   // (their sum may pass 2^31)
    const float over_D = 1.0f / (float) D;
    float w[8] = {};
    if (p.w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = p.w[WIDE ? (l.nlo ? l.lo : 0) + e : e < l.nlo ? l.lo + e : 0];
            w[4 + e] = p.w[WIDE ? (l.nhi ? l.hi : 0) + e : e < l.nhi ? l.hi + e : 0];
        }
    }
    for (int64_t b = blockIdx.z; b < p.x.ne[3]; b += gridDim.z)
        for (int64_t s = blockIdx.x; s < p.x.ne[2]; s += gridDim.x) {
            const char *xr = (const char *) p.x.data + s * p.x.nb[2] + b * p.x.nb[3];
            char *yr = (char *) p.y.data + s * p.y.nb[2] + b * p.y.nb[3];
            Run<XBF16, WIDE> v[U][2];
            f32x4 c, sn;
            // the lane's head of the HPW from h on; heads past the last are read as the last
            auto load = [&](int h, Run<XBF16, WIDE> *r) {
                const char *row = xr + (int64_t) min(h + hl, h1 - 1) * p.x.nb[1];
                r[0].load(row, l.lo, l.nlo);
                r[1].load(row, l.hi, l.nhi);
            };
            auto turn = [&](int h, const Run<XBF16, WIDE> *r) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = r[e / 4][e % 4];
                if (p.w) {
                    float q = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float y = e % 4 < (e < 4 ? l.nlo : l.nhi) ? x[e] : 0.0f;
                        q = __builtin_fmaf(y, y, q);
                    }
#pragma unroll
                    for (int t = 0; 1 << t < LPH && t < 4; ++t) q += dpp_f(q, t);
                    if (LPH > 16) q = row_pair_sum(q);
                    if (LPH > 32) q = half_pair_sum(q);
                    const float inv = inverse_root(__builtin_fmaf(q, over_D, p.eps));
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float &a = x[HALVES ? e : 2 * e], &b = x[HALVES ? 4 + e : 2 * e + 1];
                    const float y = a * c[e] - b * sn[e], z = a * sn[e] + b * c[e];
                    a = e < l.np ? y : a;
                    b = e < l.np ? z : b;
                }
                if (h + hl >= h1) return;
                char *row = yr + (int64_t) (h + hl) * p.y.nb[1];
                store_run<YBF16, WIDE>(row, l.lo, l.nlo, x);
                store_run<YBF16, WIDE>(row, l.hi, l.nhi, x + 4);
            };
            auto load_all = [&](int h) {
#pragma unroll
                for (int t = 0; t < U; ++t)
                    if (h + t * HPW < h1) load(h + t * HPW, v[t]);
            };
            load_all(h0);
            for (int i = lane; i < p.n / 2; i += 64) {
                const int a = (i >= p.first[1]) + (i >= p.first[2]) + (i >= p.first[3]);
                const char *at = (const char *) p.pos + a * p.pos_nb1 + b * p.pos_nb2 + s * 4;
                const int word = *(const int *) at;
                cos_sin(p.pos_f32 ? (double) __int_as_float(word) : (double) word, p.quarters[i], cosines[i], sines[i]);
            }
            __syncthreads();
            // (of a run's pairs past the last nothing is used)
            c = *(const f32x4 *) &cosines[l.np ? l.pair : 0];
            sn = *(const f32x4 *) &sines[l.np ? l.pair : 0];
            __syncthreads();
            for (int h = h0;;) {
#pragma unroll
                for (int t = 0; t < U; ++t)
                    if (h + t * HPW < h1) turn(h + t * HPW, v[t]);
                if ((h += U * HPW) >= h1) break;
                load_all(h);
            }
        }
}

// Tokens fewer than WAVES have their heads split among waves, whole passes each (1000 tokens of
// 32 heads of 128, f32: 9.3 us with 2048 waves wanted, 9.8 with 1024, 10.7 with 4096: each wave
// forms the angles again). More tokens than MOST are taken in turns: what a wave sets up is used
// again (32768 tokens of 16 heads of 64, bf16: 29.7 us, a wave each 32.1). Sequences are counted alike: 4096 of one token of
// 16 heads of 128, bf16, on 256 waves 26.4 us, on 4096 9.6.
constexpr int64_t WAVES = 2048, MOST = 8192;

template <bool XBF16, bool YBF16, bool WIDE, bool HALVES>
hipError_t launch_lph(const RopeAxes &p, hipStream_t s) {
    const int D = (int) p.x.ne[0], H = (int) p.x.ne[1];
    const int groups = p.halves ? (p.n / 2 + 3) / 4 + (D - p.n + 7) / 8 : (D + 7) / 8;
    int lph = 4;
    while (lph < groups) lph *= 2;
    const int hpw = 64 / lph, passes = (H + hpw - 1) / hpw;
    const int64_t tokens = p.x.ne[2] * p.x.ne[3];
    const int want = (int) std::min<int64_t>(passes, std::max<int64_t>(1, WAVES / tokens));
    const int heads = (passes + want - 1) / want * hpw;
    const dim3 grid((unsigned) std::min(p.x.ne[2], MOST), (unsigned) (((int64_t) H + heads - 1) / heads),
                    (unsigned) std::min(p.x.ne[3], std::max<int64_t>(1 << 8, MOST / p.x.ne[2])));
    auto go = [&](auto kern) {
        launch_kernel(kern, grid, dim3(64), 0, s, p, heads);
        return hipGetLastError();
    };
    switch (lph) {
        case 4: return go(rope_axes_kernel<XBF16, YBF16, WIDE, HALVES, 4>);
        case 8: return go(rope_axes_kernel<XBF16, YBF16, WIDE, HALVES, 8>);
        case 16: return go(rope_axes_kernel<XBF16, YBF16, WIDE, HALVES, 16>);
        case 32: return go(rope_axes_kernel<XBF16, YBF16, WIDE, HALVES, 32>);
        default: return go(rope_axes_kernel<XBF16, YBF16, WIDE, HALVES, 64>);
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
        constexpr bool X = decltype(x)::value, Y = decltype(y)::value;
        if (wide) return p.halves ? launch_lph<X, Y, true, true>(p, s) : launch_lph<X, Y, true, false>(p, s);
        return p.halves ? launch_lph<X, Y, false, true>(p, s) : launch_lph<X, Y, false, false>(p, s);
    };
    std::true_type t;
    std::false_type f;
    return xb ? yb ? go(t, t) : go(t, f) : yb ? go(f, t) : go(f, f);
}

}  // namespace tsk
