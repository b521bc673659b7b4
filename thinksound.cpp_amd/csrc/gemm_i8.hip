// gemm_i8.hip — products of 8-bit integer rows with a scale each (ggml_mul_mat nodes
// with I8_SPLIT weights),
//
//   Y[n, m] = (sum_k XQ[n, k] WQ[m, k]) * XD[n] * WD[m] + bias[m].
//
// Sums are int32 and exact (K below 2^17: 2^14 K stays below 2^31); they are
// rounded once to fp32, then scaled (few rows: v_mfma_i32_16x16x64_i8, tiles: v_mfma_i32_32x32x32_i8).
#include <algorithm>
#include <cmath>
#include <utility>

#include "i8.h"
#include "tsk_internal.h"
#include "tsk_runtime.h"

namespace tsk {

namespace {

typedef __attribute__((__vector_size__(16 * sizeof(int)))) int i32x16;

// scales and biases of 4 channels m .. m + 3 (those past M: zeros)
struct Channels {
    f32x4 d, bias;
};
__device__ __forceinline__ Channels channels(const I8Gemm &p, int m) {
    Channels c = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (m + 3 < p.M) {
        c.d = *(const f32x4 *) (p.wd + m);
        if (p.bias) c.bias = *(const f32x4 *) (p.bias + m);
    } else {
        for (int i = 0; i < p.M - m; ++i) {
            c.d[i] = p.wd[m + i];
            if (p.bias) c.bias[i] = p.bias[m + i];
        }
    }
    return c;
}
// (without a bias, 0 is added: -0 alone becomes 0)
__device__ __forceinline__ f32x4 scaled(i32x4 acc, float xd, const Channels &c) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf((float) acc[i] * xd, c.d[i], c.bias[i]);
    return v;
}
__device__ __forceinline__ u32x2 as_bf16(f32x4 v) {
    return u32x2{f32_to_bf16_bits(v[0]) | (uint32_t) f32_to_bf16_bits(v[1]) << 16, f32_to_bf16_bits(v[2]) | (uint32_t) f32_to_bf16_bits(v[3]) << 16};
}
// 4 outputs m .. m + 3 of row n (those below M)
__device__ __forceinline__ void store4(const I8Gemm &p, int n, int m, f32x4 v) {
    if (n >= p.N || m >= p.M) return;
    const int64_t at = (int64_t) n * p.ld_y + m;
    if (m + 3 < p.M) {
        if (p.y_bf16) *(u32x2 *) ((uint16_t *) p.y + at) = as_bf16(v);
        else *(f32x4 *) ((float *) p.y + at) = v;
        return;
    }
    for (int i = 0; i < p.M - m; ++i) {
        if (p.y_bf16) ((uint16_t *) p.y)[at + i] = f32_to_bf16_bits(v[i]);
        else ((float *) p.y)[at + i] = v[i];
    }
}

// ---------------------------------------------------------------- few rows
// Operands straight into registers. NW waves share 16 MT x 16 NT outputs and
// deal the K range among them in turns of 64 KS k; their sums meet in LDS.
// Lane l holds row l % 16 of either operand and of each 64 k the 16 bytes l / 16.
//
// Bound by the weights' bytes (8 x 8192, K = 8192, 48 matrices in turn so that none is in a cache: 15.7 us, 4.3 TB/s;
// one again and again 14.3) and, where they are few, by the launch; turns of 256 or 512 k and 8 waves are no
// faster (16.4 to 18.3, 8 matrices in turn).
//
// XT: f32 or bf16 activations, quantized by every workgroup into LDS while its first
// weights are on their way (gemm_i8_fits).
enum : int { X_I8 = 0, X_BF16 = 1, X_F32 = 2 };

constexpr int NW = 4, KS = 2;

template <int MT, int NT>
struct RowFrags {
    i32x4 a[MT][KS], b[NT][KS];
};

// bytes from a quantized row in LDS to the next: 16 rows start on 16 different 16-byte banks
__device__ __host__ constexpr int lds_row(int64_t ld) { return (int) ((ld + 255) / 256 * 256 + 16); }

// the activations into LDS, TPR threads a row (64: up to 2048 values, or all 256: up to 8192)
template <int XT, int TPR>
__device__ __forceinline__ void quantize_rows(const I8Gemm &p, int8_t *xs, float *xd, uint32_t *red) {
    constexpr int PER = 4;                                       // vectors of 8 a thread
    const int t = threadIdx.x % TPR, ld = (int) i8_ld(p.K), stride = lds_row(ld);
    for (int n = threadIdx.x / TPR; n < p.N; n += NW * 64 / TPR) {
        const char *row = (const char *) p.x + n * p.ld_x * (XT == X_F32 ? 4 : 2);
        float v[PER][8];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = (t + TPR * j) * 8;
            if (c < p.K) i8_load8<XT == X_BF16, true>(row, c, p.K, v[j]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, i8_abs_bits(v[j][e]));
        for (int m = 1; m < 64; m *= 2) top = max(top, (uint32_t) __shfl_xor((int) top, m));
        if constexpr (TPR > 64) {                                // (one row at a time: every thread comes here as often)
            __syncthreads();
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < TPR / 64; ++i) top = max(top, red[i]);
        }
        const I8Scale s = i8_scale(top);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int c = (t + TPR * j) * 8;
            if (c < ld) *(u32x2 *) (xs + n * stride + c) = u32x2{i8_pack4(v[j], s), i8_pack4(v[j] + 4, s)};
        }
        if (t == 0) xd[n] = s.d;
    }
    __syncthreads();
}

template <int MT, int NT, int XT, int TPR>
__global__ __launch_bounds__(NW * 64) void i8_gemm_rows_kernel(const I8Gemm p, int tiles_m) {
    __shared__ __attribute__((aligned(16))) int red[NW * MT * NT * 256];
    __shared__ float xds[16];
    extern __shared__ __attribute__((aligned(16))) int8_t xs[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int m0 = (int) (blockIdx.x % tiles_m) * (16 * MT), n0 = (int) (blockIdx.x / tiles_m) * (16 * NT);
    const int64_t ld = i8_ld(p.K);
    const int nit = (int) ((ld + 64 * KS - 1) / (64 * KS));
    // rows past M or N read the last one (their outputs are not stored)
    const int8_t *wq[MT], *xq[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) wq[i] = p.wq + (int64_t) min(m0 + 16 * i + r, p.M - 1) * ld + 16 * g;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = min(n0 + 16 * j + r, p.N - 1);
        xq[j] = XT == X_I8 ? p.xq + (int64_t) n * ld + 16 * g : xs + n * lds_row(ld) + 16 * g;
    }
    typedef RowFrags<MT, NT> Frags;
    const i32x4 zero = {0, 0, 0, 0};
    auto load_w = [&](int it, Frags &f) {
        const int64_t k0 = (int64_t) it * (64 * KS);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)                          // (rows are whole pieces of 16)
#pragma unroll
            for (int i = 0; i < MT; ++i) f.a[i][ks] = k0 + 64 * ks + 16 * g < ld ? *(const i32x4 *) (wq[i] + k0 + 64 * ks) : zero;
    };
    auto load_x = [&](int it, Frags &f) {
        const int64_t k0 = (int64_t) it * (64 * KS);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < NT; ++j) f.b[j][ks] = k0 + 64 * ks + 16 * g < ld ? *(const i32x4 *) (xq[j] + k0 + 64 * ks) : zero;
    };
    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = zero;
    auto product = [&](int it, Frags &f) {
        if constexpr (XT != X_I8) load_x(it, f);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.a[i][ks], f.b[j][ks], acc[i][j], 0, 0, 0);
    };
    auto load = [&](int it, Frags &f) {
        load_w(it, f);
        if constexpr (XT == X_I8) load_x(it, f);
    };
    Frags f0, f1;
    if (wave < nit) load(wave, f0);
    if constexpr (XT != X_I8) quantize_rows<XT, TPR>(p, xs, xds, (uint32_t *) red);
    if (wave < nit) {
        int it = wave;
        for (; it + NW < nit; it += 2 * NW) {
            load(it + NW, f1);
            product(it, f0);
            if (it + 2 * NW < nit) load(it + 2 * NW, f0);
            product(it + NW, f1);
        }
        if (it < nit) product(it, f0);
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
            const int n = n0 + 16 * j + r, m = m0 + 16 * i + 4 * g;
            if (n < p.N && m < p.M) store4(p, n, m, scaled(v, XT == X_I8 ? p.xd[n] : xds[n], channels(p, m)));
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

template <int MT, int NT>
hipError_t launch_rows(const I8Gemm &p, hipStream_t s) {
    const int tiles_m = (p.M + 16 * MT - 1) / (16 * MT), tiles_n = (p.N + 16 * NT - 1) / (16 * NT);
    const int64_t T = (int64_t) tiles_m * tiles_n;
    if (T * NW * 64 >= MAX_THREADS) return in_two(p, [&](const I8Gemm &q) { return launch_rows<MT, NT>(q, s); });
    launch_kernel(i8_gemm_rows_kernel<MT, NT, X_I8, 64>, dim3((unsigned) T), dim3(NW * 64), 0, s, p, tiles_m);
    return hipGetLastError();
}
// f32 / bf16 activations
hipError_t launch_fused(const I8Gemm &p, hipStream_t s) {
    const int tiles_m = (p.M + 15) / 16;                         // (M <= 2^26: 2^30 threads)
    auto kern = p.x_f32 ? p.N == 1 ? i8_gemm_rows_kernel<1, 1, X_F32, 256> : i8_gemm_rows_kernel<1, 1, X_F32, 64>
                        : p.N == 1 ? i8_gemm_rows_kernel<1, 1, X_BF16, 256> : i8_gemm_rows_kernel<1, 1, X_BF16, 64>;
    const size_t lds = (size_t) p.N * lds_row(i8_ld(p.K));
    launch_kernel(kern, dim3((unsigned) tiles_m), dim3(NW * 64), lds, s, p, tiles_m);
    return hipGetLastError();
}

// ---------------------------------------------------------------- tiles
typedef __attribute__((address_space(3))) void lds_void;

template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short) 0, (int) bytes, 0x00020000);
}

// Tiles. WM x WN waves share a BM x BN output tile, each TM x TN sub-tiles of 32 x 32
// (v_mfma_i32_32x32x32_i8), over stages of 128 k in a ring of R stages of LDS.
//
// A stage takes from LDS, per wave, TM + TN pieces of 1 KB each 32 k, from L2 (BM + BN)
// * 128 bytes, from the matrix unit 32 clocks an instruction. In turns these add up; so each
// product is followed by at most a read of what the next ones take and a load of a later
// stage, in the program's order. HALVES: the first half of a stage's products reads the
// second half's operands, the second half the next stage's first, with the one barrier of
// a stage inside it. Otherwise (small tiles, whose CU has other tiles to fill the waits) a
// whole stage is read while the one before is multiplied.
template <int WM_, int WN_, int TM_, int TN_, int R_, bool HALVES_>
struct Cfg {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, R = R_;
    static constexpr bool HALVES = HALVES_;
    static constexpr int NW = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32;
    static constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
    // loads of 1 KB (8 rows) a wave and stage; a wave without one of its own repeats another's
    static constexpr int UA = BM / 8, UB = BN / 8, LA = (UA + NW - 1) / NW, LB = (UB + NW - 1) / NW, LOADS = LA + LB;
    static constexpr size_t LDS = (size_t) R * STAGE;
    static_assert(NW % 4 == 0 && UA % 4 == 0 && UB % 4 == 0 && R >= 2 && LOADS * (R - 1) < 64 && LDS <= 160 * 1024, "tile");
};

// f(0), ..., f(N - 1), the arguments constants
template <class F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
#define EACH(q, from, to, ...) each([&](auto q##_) __attribute__((always_inline)) { constexpr int q = decltype(q##_)::value + (from); __VA_ARGS__ }, std::make_integer_sequence<int, ((to) > (from) ? (to) - (from) : 0)>{})

template <class C>
__global__ __launch_bounds__(C::NW * 64) void i8_gemm_tile_kernel(const I8Gemm p, int tiles_m, int tiles_n) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    constexpr int TM = C::TM, TN = C::TN, NW = C::NW, R = C::R;
    // workgroup L runs on XCD L % 8: each XCD takes a run of the tiles, eight tiles of m wide
    int tm, tn;
    {
        const int T = tiles_m * tiles_n, per = (T + 7) / 8, t = (int) (blockIdx.x & 7) * per + (int) (blockIdx.x >> 3);
        if ((int) (blockIdx.x >> 3) >= per || t >= T) return;
        const int band = t / (8 * tiles_n), w = min(8, tiles_m - 8 * band), in = t - band * 8 * tiles_n;
        tm = 8 * band + in % w;
        tn = in / w;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int l32 = lane & 31, hi = lane >> 5, wm = wave % C::WM, wn = wave / C::WM;
    const int m0 = tm * C::BM, n0 = tn * C::BN;
    const int ld = (int) i8_ld(p.K), pieces = ld / 16, nst = (pieces + 7) / 8;

    // Rows past M or N are past the descriptors' ends, pieces past a row's end are sent
    // FAR: the loads put zeros there
    const __amdgpu_buffer_rsrc_t ra = rsrc_of(p.wq + (int64_t) m0 * ld, (int64_t) min(C::BM, p.M - m0) * ld);
    const __amdgpu_buffer_rsrc_t rb = rsrc_of(p.xq + (int64_t) n0 * ld, (int64_t) min(C::BN, p.N - n0) * ld);
    constexpr int FAR = (int) 0x80000000u;
    // Piece c of row t lies at slot c ^ (t / 2 % 8). A 16-byte LDS read of a wave takes
    // four turns, of lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31, and the same 32
    // further: the 8 even and the 8 odd rows of a turn then take 8 slots each.
    const int chk = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));               // (a wave's loads are NW, a multiple of 4, apart)
    int from = (lane >> 3) * ld + chk * 16, at = l32 * 128 + ((hi ^ (l32 >> 1 & 7)) << 4);
    // load q of this wave's for stage t (stages past the last: zeros, so that every wait counts the same)
    auto issue_one = [&](int t, int slot, int q) __attribute__((always_inline)) {
        uint8_t *st = lds + slot * C::STAGE;
        const bool in = t * 8 + chk < pieces;
        if (q < C::LA) {
            const int u = (wave + NW * q) % C::UA;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void *) (st + u * 1024), 16, in ? u * 8 * ld + from : FAR, t * 128, 0, 0);
        } else {
            const int u = (wave + NW * (q - C::LA)) % C::UB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *) (st + C::A_BYTES + u * 1024), 16, in ? u * 8 * ld + from : FAR, t * 128, 0, 0);
        }
    };
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;

    // step s of a stage: lane half hi takes piece 2 s + hi of every row
    struct Frags {
        i32x4 a[4][TM], b[4][TN];
    };
    constexpr int NR = 4 * (TM + TN), NM = 4 * TM * TN;
    auto read_one = [&](int slot, Frags &f, int q) __attribute__((always_inline)) {
        const uint8_t *st = lds + slot * C::STAGE;
        const int s = q / (TM + TN), u = q % (TM + TN);
        if (u < TN) f.b[s][u] = *(const i32x4 *) (st + C::A_BYTES + (wn * TN + u) * 4096 + (at ^ 32 * s));
        else f.a[s][u - TN] = *(const i32x4 *) (st + (wm * TM + u - TN) * 4096 + (at ^ 32 * s));
    };
    auto multiply_one = [&](const Frags &f, int q) __attribute__((always_inline)) {
        const int s = q / (TM * TN), i = q / TN % TM, j = q % TN;
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.a[s][i], f.b[s][j], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int t = 0; t < R; ++t)
#pragma unroll
        for (int q = 0; q < C::LOADS; ++q) issue_one(t, t, q);
    Frags f0;
    wait_vm<(R - 1) * C::LOADS>();
    asm volatile("s_barrier" ::: "memory");
    EACH(q, 0, (C::HALVES ? NR / 2 : NR), read_one(0, f0, q););
    int slot = 0;                                                              // of stage t
    // past it every wave has stage t in registers, whose slot is refilled, and
    // every wave's loads of stage t + 1 have landed
    auto fill = [&]() __attribute__((always_inline)) {
        wait_vm<(R - 2) * C::LOADS>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto step = [&](int t, Frags &now, Frags &next) __attribute__((always_inline)) {
        const int s1 = slot + 1 == R ? 0 : slot + 1;
        asm volatile("" : "+v"(from), "+v"(at));              // (or the compiler keeps every whole offset in a register)
        if constexpr (C::HALVES) {
            constexpr int H = NM / 2, GB = TM * TN / 2, H0 = (3 * H + 3) / 4, N1 = NR / 2, H1 = H - GB;
            EACH(q, 0, H,
                multiply_one(now, q);
                EACH(u, q * N1 / H0, (q + 1) * N1 / H0 < N1 ? (q + 1) * N1 / H0 : N1, read_one(slot, now, N1 + u););
                __builtin_amdgcn_sched_barrier(0););
            EACH(q, 0, GB, multiply_one(now, H + q););
            __builtin_amdgcn_sched_barrier(0);
            fill();
            EACH(q, 0, H1,
                multiply_one(now, H + GB + q);
                EACH(u, q * N1 / H1, (q + 1) * N1 / H1, read_one(s1, next, u););
                EACH(u, q * C::LOADS / H1, (q + 1) * C::LOADS / H1, issue_one(t + R, slot, u););
                __builtin_amdgcn_sched_barrier(0););
        } else {
            constexpr int H0 = (NM * 3 + 3) / 4;
            fill();
            EACH(q, 0, NM,
                multiply_one(now, q);
                EACH(u, q * NR / H0, (q + 1) * NR / H0 < NR ? (q + 1) * NR / H0 : NR, read_one(s1, next, u););
                EACH(u, q * C::LOADS / NM, (q + 1) * C::LOADS / NM, issue_one(t + R, slot, u););
                __builtin_amdgcn_sched_barrier(0););
        }
        slot = s1;
    };
    int t = 0;
    if constexpr (C::HALVES) {
        for (; t < nst; ++t) {
            Frags next;
            step(t, f0, next);
            f0 = next;
        }
    } else {
        Frags f1;
        for (; t + 1 < nst; t += 2) {
            step(t, f0, f1);
            step(t + 1, f1, f0);
        }
        if (t < nst) step(t, f0, f1);
    }
    wait_vm<0>();
    float xd[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) xd[j] = p.xd[min(n0 + (wn * TN + j) * 32 + l32, p.N - 1)];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
            // two runs of 4 channels, 8 apart; the other half of the wave holds the 4 behind each
            const int m = m0 + (wm * TM + i) * 32 + 2 * e, mq[2] = {m + 4 * hi, m + 8 + 4 * hi};
            const Channels c[2] = {channels(p, mq[0]), channels(p, mq[1])};
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int n = n0 + (wn * TN + j) * 32 + l32;
                f32x4 v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    v[h] = scaled(i32x4{acc[i][j][e + 4 * h], acc[i][j][e + 4 * h + 1], acc[i][j][e + 4 * h + 2], acc[i][j][e + 4 * h + 3]}, xd[j], c[h]);
                if (p.y_bf16 && m + 15 < p.M) {
                    // the halves trade runs: each lane stores 8 channels, 16 bytes
                    const u32x2 x = as_bf16(v[0]), y = as_bf16(v[1]);
                    const auto s0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false), s1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
                    if (n < p.N) *(u32x4 *) ((uint16_t *) p.y + (int64_t) n * p.ld_y + m + 8 * hi) = u32x4{s0[0], s1[0], s0[1], s1[1]};
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) store4(p, n, mq[h], v[h]);
                }
            }
        }
}

template <class C>
hipError_t launch_tile(const I8Gemm &p, hipStream_t s) {
    const int tiles_m = (p.M + C::BM - 1) / C::BM, tiles_n = (p.N + C::BN - 1) / C::BN;
    const int64_t T = (int64_t) tiles_m * tiles_n;
    if ((T + 7) * C::NW * 64 >= MAX_THREADS) return in_two(p, [&](const I8Gemm &q) { return launch_tile<C>(q, s); });
    lds_opt_in((const void *) i8_gemm_tile_kernel<C>, C::LDS);
    launch_kernel(i8_gemm_tile_kernel<C>, dim3((unsigned) ((T + 7) / 8 * 8)), dim3(C::NW * 64), C::LDS, s, p, tiles_m, tiles_n);
    return hipGetLastError();
}

// Shapes, by number (TSK_I8_CFG), with outputs as M x N, and the us of one tile at K =
// 5120 without the launch: its fixed part (first loads, stores), and the rest alone / where
// all 256 CUs have one (the chip's clock falls, and L2 is shared) or take turns:
//   1   256 x 256, 8 waves   4.9 + 41.6 / 67.6
//   2   128 x 256, 8 waves   2.2 + 23.8 / 38.3
//   3   128 x 128, 4 waves   1.0 + 16.0 / 22.5
//   4   64 x 128, 4 waves    0.5 + 11.7 / 13.5
//   5   64 x 64, 4 waves     0.3 + 8.0 / 8.1
//   6   192 x 128, 8 waves   3.0 + 19.0 / 30.0
//   7   128 x 192, 8 waves   1.5 + 18.0 / 30.5
//   8   192 x 256, 8 waves   3.5 + 33.5 / 53.5
//   11  rows kernel, 16 x 16 outputs,  12  32 x 16,  13  32 x 32
//
// Tiles: the shape of the least time. Some pairs (us, taken / next; rows x M): 8192^3
// 1 457 / 8 508; 4096 x 4096, K = 5120 1 76 / 2 86; 2047 x 2050, K = 5120 7 29.0 / 2
// 32.3 / 3 43; 4096 x 2048, K = 5120 2 43 / 8 49; 2048 x 2048, K = 5120 3 26 / 7 28; 1292
// x 1024, K = 4096 4 13.4 / 3 17 / 5 13.9; 388 x 1024, K = 1024 5 5.0 / 3 7.2.
// Few rows: the rows kernel in the smallest of its shapes that gives no CU two
// workgroups, 16 x 16 for up to 16 rows (8 x 8192, K = 8192 11 15.4 / 12 20.8 / 5 20.9; 64
// x 1024, K = 8192 11 9.6 / 12 12.9 / 5 14.8; 32 x 4096, K = 1024 12 3.9 / 11 4.2 / 5 4.8;
// 64 x 4096, K = 4096 13 10.5 / 5 12.6), and tiles where none does (64 x 8192, K =
// 8192 5 23.7 / 13 39; 256 x 4096, K = 1024 5 5.3 / 13 9.8).
int shape_for(const I8Gemm &p) {
    if (tuning().i8_cfg) return tuning().i8_cfg;
    auto tiles = [&](int bm, int bn) { return (int64_t) ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    if (p.N <= 16 || tiles(16, 16) <= 256) return 11;
    if (tiles(32, 16) <= 256) return 12;
    if (tiles(32, 32) <= 256) return 13;
    struct Shape { int bm, bn; double fixed, alone, full; };
    constexpr Shape shapes[8] = {{256, 256, 4.9, 41.6, 67.6}, {128, 256, 2.2, 23.8, 38.3}, {128, 128, 1.0, 16.0, 22.5}, {64, 128, 0.5, 11.7, 13.5},
                                 {64, 64, 0.3, 8.0, 8.1},     {192, 128, 3.0, 19.0, 30.0}, {128, 192, 1.5, 18.0, 30.5}, {192, 256, 3.5, 33.5, 53.5}};
    int best = 0;
    double least = 0;
    for (int i = 0; i < 8; ++i) {
        const Shape &c = shapes[i];
        const double n = (double) tiles(c.bm, c.bn), each = std::ceil(n / 256);       // tiles of a CU
        const double run = each == 1 ? c.alone + (c.full - c.alone) * n / 256 : each * c.full;
        const double cost = each * c.fixed + run * p.K / 5120;
        if (!best || cost < least) {
            best = i + 1;
            least = cost;
        }
    }
    return best;
}

}  // namespace

// f32 / bf16 activations: a launch that quantizes them and the product's wait for it cost
// 3 us; every workgroup's own quantization, of one row by all its threads or of up to
// four by a wave each (us, inside / two launches; rows x M): 1 x 6144, K = 1024 5.2 /
// 6.9; 1 x 8192, K = 8192 18.9 / 20.4; 3 x 6144, K = 1024 5.8 / 6.9; 4 x 2048, K = 2048
// 6.9 / 7.2; 8 x 1024, K = 1024 6.6 / 6.4; 2 x 8192, K = 8192 22.6 / 20.4.
bool gemm_i8_fits(int64_t N, int64_t K) { return N == 1 ? K <= 8192 : N <= 4 && K <= 2048 && N * K <= 4096; }
// Each workgroup of 16 channels does so, and from some 32768 channels on they cost more than the launch
// (weights that are in no cache): 1 x 32768, K = 1024 10.8 / 11.5, x 65536 16.9 / 16.5, x 152064 32.7 / 29.7; K = 256
// 7.4 / 6.6, 11.5 / 8.0, 22.1 / 12.5; 2 x 32768, K = 2048 18.2 / 17.7, x 152064 63.5 / 55.4; 4 x 32768, K = 1024 11.9 / 12.0,
// x 152064 40.9 / 33.7. One row of 2048 and more hides behind its weights: K = 2048 x 152064 50.6 / 53.3, K = 4096 111.6 / 119.9,
// K = 8192 210.8 / 212.5.
bool gemm_i8_fused(int64_t N, int64_t K, int64_t M) { return gemm_i8_fits(N, K) && (M <= 32768 || (N == 1 && K >= 2048)); }

hipError_t launch_gemm_i8(const I8Gemm &p, hipStream_t s) {
    if (!p.xq) return launch_fused(p, s);
    switch (shape_for(p)) {
        case 1: return launch_tile<Cfg<2, 4, 4, 2, 2, true>>(p, s);
        case 2: return launch_tile<Cfg<2, 4, 2, 2, 3, true>>(p, s);
        case 3: return launch_tile<Cfg<2, 2, 2, 2, 3, false>>(p, s);
        case 4: return launch_tile<Cfg<2, 2, 1, 2, 3, true>>(p, s);
        case 6: return launch_tile<Cfg<2, 4, 3, 1, 3, true>>(p, s);
        case 7: return launch_tile<Cfg<4, 2, 1, 3, 3, true>>(p, s);
        case 8: return launch_tile<Cfg<2, 4, 3, 2, 2, true>>(p, s);
        case 11: return launch_rows<1, 1>(p, s);
        case 12: return launch_rows<2, 1>(p, s);
        case 13: return launch_rows<2, 2>(p, s);
        default: return launch_tile<Cfg<2, 2, 1, 1, 4, false>>(p, s);
    }
}

}  // namespace tsk
