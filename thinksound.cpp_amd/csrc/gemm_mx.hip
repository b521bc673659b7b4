// gemm_mx.hip — products with MXFP4 weights (ggml_mul_mat nodes),
//
//   Y[n, m] = sum_k X[n, k] W[m, k] + bias[m],   W = codes * 2^(scale - 127) per 32 k,
//
// with X in bf16 (or f32, rounded to bf16 as it is read), or X in MXFP4 too.
// Sums are f32. With bf16 X a code times its scale is a bf16 number exactly
// (the conversion instruction takes the scale; 2^128 and up become infinite), so
// v_mfma_f32_16x16x32_bf16 adds exact products; with MXFP4 X v_mfma_scale_f32_16x16x128_f8f6f4 takes
// codes and scale bytes as they lie in memory.
//
// Bound: few rows by the weights' bytes (8 x 8192, K = 8192 12.6 us, 2.8 TB/s);
// many rows by the matrix units, LDS and power together: 8192 x 8192, K = 8192
// 275 us with MXFP4 X (4.0 PFLOP/s; products alone, without their loads, take
// 200), 850-930 us with bf16 X (1.2-1.3 PFLOP/s).
#include <algorithm>
#include <cmath>
#include <utility>

#include "mxfp4.h"
#include "tsk_internal.h"
#include "tsk_runtime.h"

namespace tsk {

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(int)))) int i32x8;

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

enum : int { X_BF16 = 0, X_F32 = 1, X_MX = 2 };

// ---------------------------------------------------------------- few rows
// Operands straight into registers. NW waves share 16 MT x 16 NT outputs and
// deal the K range among them in turns of 256 k; their sums meet in LDS, in
// wave order. Lane l holds row l % 16 of either operand and of each 128 k the
// block of 32 number l / 16: the layout of v_mfma_scale_f32_16x16x128_f8f6f4,
// and with the k of four v_mfma_f32_16x16x32_bf16 taken in the same order on
// both sides, of those. Bound by the weights' bytes and the latency of the first
// loads: each wave keeps the loads of its next turn in flight (8 x 8192, K = 8192
// 12.6 us, 2.8 TB/s; 1 x 6144, K = 1024 4.0 us); 8 and 16 waves are no faster.
template <int XT, int MT, int NT>
struct RowFrags {
    static constexpr int BQ = XT == X_MX ? 1 : XT == X_BF16 ? 4 : 8;       // 16-byte pieces of an activation block
    u32x4 a[MT][2], b[NT][2][BQ];
    u32x2 sa[MT], sb[XT == X_MX ? NT : 1];
};

template <int XT, int MT, int NT, int NW>
__device__ __forceinline__ void mx_gemm_rows(const MxGemm &p, int tiles_m, float *red) {
    constexpr bool MX = XT == X_MX;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int m0 = (int) (blockIdx.x % tiles_m) * (16 * MT), n0 = (int) (blockIdx.x / tiles_m) * (16 * NT);
    const int64_t K2 = p.K / 2, KB = p.K / 32;
    const int nit = (int) ((KB + 7) / 8);
    typedef RowFrags<XT, MT, NT> Frags;
    // rows past M or N read the last one (their outputs are not stored)
    const uint8_t *wq[MT], *ws[MT], *xq[NT], *xs[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = min(m0 + 16 * i + r, p.M - 1);
        wq[i] = p.wq + m * K2 + 16 * g;
        ws[i] = p.ws + m * KB;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = min(n0 + 16 * j + r, p.N - 1);
        xq[j] = MX ? p.xq + n * K2 + 16 * g : (const uint8_t *) p.x + n * p.ld_x * (XT == X_F32 ? 4 : 2) + (16 * Frags::BQ) * g;
        xs[j] = MX ? p.xs + n * KB : nullptr;
    }
    auto load = [&](int it, Frags &f) {
        const int64_t b0 = (int64_t) it * 8;
        if (b0 + 8 <= KB) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) f.a[i][ks] = *(const u32x4 *) (wq[i] + (b0 + 4 * ks) * 16);
                __builtin_memcpy(&f.sa[i], ws[i] + b0, 8);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int h = 0; h < Frags::BQ; ++h)
                        f.b[j][ks][h] = *(const u32x4 *) (xq[j] + (b0 + 4 * ks) * (16 * Frags::BQ) + 16 * h);
                if constexpr (MX) __builtin_memcpy(&f.sb[j], xs[j] + b0, 8);
            }
            return;
        }
        // the last turn's blocks past K: zeros
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const int64_t blk = b0 + 4 * ks + g;
            const bool in = blk < KB;
            const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                f.a[i][ks] = in ? *(const u32x4 *) (wq[i] + (b0 + 4 * ks) * 16) : zero;
                f.sa[i][ks] = in ? (uint32_t) ws[i][blk] << 8 * g : 0u;
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int h = 0; h < Frags::BQ; ++h)
                    f.b[j][ks][h] = in ? *(const u32x4 *) (xq[j] + (b0 + 4 * ks) * (16 * Frags::BQ) + 16 * h) : zero;
                if constexpr (MX) f.sb[j][ks] = in ? (uint32_t) xs[j][blk] << 8 * g : 0u;
            }
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    auto product = [&](const Frags &f) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if constexpr (MX) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const i32x8 av = {(int) f.a[i][ks][0], (int) f.a[i][ks][1], (int) f.a[i][ks][2], (int) f.a[i][ks][3], 0, 0, 0, 0};
                        const i32x8 bv = {(int) f.b[j][ks][0][0], (int) f.b[j][ks][0][1], (int) f.b[j][ks][0][2], (int) f.b[j][ks][0][3], 0, 0, 0, 0};
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[i][j], 4, 4, 0, (int) (f.sa[i][ks] >> 8 * g), 0,
                                                                                     (int) (f.sb[j][ks] >> 8 * g));
                    }
            } else {
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    bf16x8 b[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if constexpr (XT == X_F32) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                b[j][e] = (__bf16) __uint_as_float(f.b[j][ks][2 * h][e]);
                                b[j][4 + e] = (__bf16) __uint_as_float(f.b[j][ks][2 * h + 1][e]);
                            }
                        } else {
                            b[j] = __builtin_bit_cast(bf16x8, f.b[j][ks][h]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const bf16x8 av = mx_decode8_bf16(f.a[i][ks][h], mx_scale(f.sa[i][ks] >> 8 * g & 255u));
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, b[j], acc[i][j], 0, 0, 0);
                    }
                }
            }
        }
    };
    if (wave < nit) {
        Frags f0, f1;
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
    if constexpr (NW > 1) {
        // [wave][tile][lane] partial sums, four floats each
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) *(f32x4 *) (red + ((wave * MT * NT + i * NT + j) * 64 + lane) * 4) = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if ((i * NT + j) % NW != wave) continue;
                f32x4 v = *(const f32x4 *) (red + ((i * NT + j) * 64 + lane) * 4);
                for (int w = 1; w < NW; ++w) v += *(const f32x4 *) (red + ((w * MT * NT + i * NT + j) * 64 + lane) * 4);
                store4(p, n0 + 16 * j + r, m0 + 16 * i + 4 * g, v);
            }
    } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) store4(p, n0 + 16 * j + r, m0 + 16 * i + 4 * g, acc[i][j]);
    }
}

template <int XT, int MT, int NT, int NW>
__global__ __launch_bounds__(NW * 64) void mx_gemm_rows_kernel(const MxGemm p, int tiles_m) {
    __shared__ __attribute__((aligned(16))) float red[NW > 1 ? NW * MT * NT * 256 : 4];
    mx_gemm_rows<XT, MT, NT, NW>(p, tiles_m, red);
}
// A launch holds fewer than 2^32 threads: products of more are cut into two by
// their rows (16 rows at least, of M < 2^26 outputs each: 2^30 threads).
constexpr int64_t MAX_THREADS = (int64_t) 1 << 31;
template <class F>
hipError_t in_two(const MxGemm &p, F launch) {
    MxGemm a = p, b = p;
    a.N = (p.N / 2 + 15) / 16 * 16;
    b.N = p.N - a.N;
    if (b.N < 1) return hipErrorInvalidValue;
    b.y = (char *) p.y + a.N * p.ld_y * (p.y_bf16 ? 2 : 4);
    if (p.xq) {
        b.xq = p.xq + (int64_t) a.N * (p.K / 2);
        b.xs = p.xs + (int64_t) a.N * (p.K / 32);
    } else {
        b.x = (const char *) p.x + a.N * p.ld_x * (p.x_f32 ? 4 : 2);
    }
    const hipError_t e = launch(a);
    return e == hipSuccess ? launch(b) : e;
}

template <int XT, int MT, int NT, int NW>
hipError_t launch_rows(const MxGemm &p, hipStream_t s) {
    const int tiles_m = (p.M + 16 * MT - 1) / (16 * MT), tiles_n = (p.N + 16 * NT - 1) / (16 * NT);
    const int64_t T = (int64_t) tiles_m * tiles_n;
    if (T * NW * 64 >= MAX_THREADS) return in_two(p, [&](const MxGemm &q) { return launch_rows<XT, MT, NT, NW>(q, s); });
    launch_kernel(mx_gemm_rows_kernel<XT, MT, NT, NW>, dim3((unsigned) T), dim3(NW * 64), 0, s, p, tiles_m);
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

// BYTES per lane, zero-extended, to LDS at dst + 4 * lane
template <int BYTES>
__device__ __forceinline__ void load_scales(__amdgpu_buffer_rsrc_t rsrc, uint8_t *dst, int off) {
    if constexpr (BYTES == 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *) dst, 2, off, 0, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *) dst, 1, off, 0, 0, 0);
}

// Tiles. WM x WN waves share a BM x BN output tile, each TM x TN sub-tiles of
// 16 x 16, over stages of SK blocks of 32 k in a ring of R stages of LDS.
// Scales (SCB bytes a load and lane): with SCB = 16 in chunks of 1024 k beside
// the ring (rows of scale bytes dword-aligned, K % 128 == 0; a stage's own few
// bytes cost as many L2 requests as its codes: 8192^3 357 us against 326), else
// with their stage.
//
// A stage takes from LDS, per wave, TM + TN pieces of 1 KB each 128 k (128 bytes
// a clock and CU), from L2 64 bytes a clock, from the matrix unit 16 clocks an
// instruction. In turns these add up; so each product is followed by at most a
// read of what the next ones take and a load of a later stage, in the program's
// order (sched_barrier). HALVES: the first half of a stage's products reads
// the second half's operands, the second half the next stage's first, with the
// one barrier of a stage inside it. Otherwise (the tiles of four waves, whose CU has
// other tiles to fill the waits) a whole stage is read while the one before is
// multiplied. Three stages where they leave a CU two tiles or more: longer rings
// only delay the first products (64 x 128, 1292 x 1024, K = 4096, five stages 11.9,
// three 11.1; 64 x 32, 14.1 and 11.4). Measured (us): all reads before the products,
// loads before the reads 8192^3 320-333, 4096 x 4096, K = 5120 56; whole stages in
// order, 128 x 256 tiles 8192^3 397, halves 322; halves, 256 x 256 tiles 275-302 and
// 49-51; 1292 x 1024, K = 4096, 64 x 32 tiles of five stages halves 16.2, whole
// 14.4, 64 x 64 tiles halves 11.9, whole 11.1.
template <int XT_, int WM_, int WN_, int TM_, int TN_, int SK_, int R_, int SCB_, bool HALVES_>
struct Cfg {
    static constexpr int XT = XT_, WM = WM_, WN = WN_, TM = TM_, TN = TN_, SK = SK_, R = R_, SCB = SCB_;
    static constexpr bool HALVES = HALVES_;
    static constexpr int NW = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
    static constexpr bool MX = XT == X_MX, CHUNK = SCB == 16;
    static constexpr int XROW = MX ? SK * 16 : SK * 64;                    // bytes of an activation row per stage
    static constexpr int SROW = CHUNK ? 0 : SK / SCB * 4;                  // bytes of a row's scales per stage
    static constexpr int SROWS = BM + (MX ? BN : 0);                       // rows with scales
    // LDS of a stage: weight codes, activations, weight scales, activation scales
    static constexpr int A_BYTES = BM * SK * 16, B_BYTES = BN * XROW, S_BYTES = SROWS * SROW;
    static constexpr int STAGE = A_BYTES + B_BYTES + S_BYTES;
    // chunks: CS stages each, a part loaded with every stage: with a ring of two
    // stages from a chunk's first stage on, when the chunk before the one that is
    // read has been read, longer ones one stage earlier and into a third buffer
    static constexpr int CS = 32 / SK, CHUNK_BYTES = CHUNK ? SROWS * 32 : 0, CHUNKS = !CHUNK ? 0 : R == 2 ? 2 : 3;
    // loads of a wave per stage: 64 lanes x 16 bytes of codes or bf16, x 4 bytes of scales
    static constexpr int UA = A_BYTES / 1024, UB = B_BYTES / 1024, US = CHUNK ? SROWS / 32 : S_BYTES / 256;
    static constexpr int USP = CHUNK ? (US + CS - 1) / CS : US;   // scale loads with one stage
    // (a wave without a load of its own repeats another's: the waits count the same for all)
    static constexpr int LA = (UA + NW - 1) / NW, LB = (UB + NW - 1) / NW, LS = (USP + NW - 1) / NW;
    static constexpr int LOADS = LA + LB + LS;
    static constexpr size_t LDS = (size_t) R * STAGE + CHUNKS * CHUNK_BYTES;
    static_assert(NW % 4 == 0 && UA % 4 == 0 && UB % 4 == 0 && R >= 2 && R <= 5 && LOADS * (R - 1) < 64 && LDS <= 160 * 1024, "tile");
};

// f(0), ..., f(N - 1), the arguments constants
template <class F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
#define EACH(q, from, to, ...) each([&](auto q##_) __attribute__((always_inline)) { constexpr int q = decltype(q##_)::value + (from); __VA_ARGS__ }, std::make_integer_sequence<int, ((to) > (from) ? (to) - (from) : 0)>{})

template <class C>
__device__ __forceinline__ void mx_gemm_tile(const MxGemm &p, int tiles_m, int tiles_n, uint8_t *lds) {
    constexpr int TM = C::TM, TN = C::TN, SK = C::SK, NW = C::NW, SCB = C::SCB, R = C::R;
    constexpr bool MX = C::MX, CHUNK = C::CHUNK;
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
    const int r = lane & 15, g = lane >> 4, wm = wave % C::WM, wn = wave / C::WM;
    const int m0 = tm * C::BM, n0 = tn * C::BN;
    const int K2 = p.K / 2, KB = p.K / 32;
    const int nst = (KB + SK - 1) / SK;

    // Rows past M or N are past the descriptors' ends by the lane's own offset:
    // the loads put zeros there. So do blocks past K, sent FAR with the last
    // stage; a scale past K is zeroed like its codes (it would be the next
    // row's, and could be a NaN).
    const int rm = min(C::BM, p.M - m0), rn = min(C::BN, p.N - n0);
    const int64_t xrow = MX ? K2 : p.ld_x * 2;                                 // bytes between activation rows
    const __amdgpu_buffer_rsrc_t ra = rsrc_of(p.wq + (int64_t) m0 * K2, (int64_t) rm * K2);
    const __amdgpu_buffer_rsrc_t rsa = rsrc_of(p.ws + (int64_t) m0 * KB, (int64_t) rm * KB);
    const __amdgpu_buffer_rsrc_t rb = MX ? rsrc_of(p.xq + (int64_t) n0 * K2, (int64_t) rn * K2)
                                         : rsrc_of((const char *) p.x + n0 * xrow, (rn - 1) * xrow + (int64_t) p.K * 2);
    const __amdgpu_buffer_rsrc_t rsb = MX ? rsrc_of(p.xs + (int64_t) n0 * KB, (int64_t) rn * KB) : rsa;
    constexpr int FAR = (int) 0x80000000u;
    // A lane's part of a load: rows of SK 16-byte chunks of codes, 64 / SK rows
    // a load, chunk c of row t at slot c ^ key(t). A 16-byte LDS read of a wave
    // takes four turns, of lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31, and the
    // same 32 further: 8 rows of one lane group's chunk and the other 8 of its
    // neighbour's. The keys spread these over all 256 bytes of banks (a quarter of
    // the 16 rows takes its own part of the chunks, in the order 0, 2, 3, 1: 8192^3
    // 6.5 million cycles of conflicts and 275 us; in the order 0 to 3 every read
    // meets itself twice, 45 million and 285).
    constexpr int AR = 64 / SK;
    auto quarter = [](int row) {
        const int t = row >> 2 & 3;
        return ((t ^ t >> 1) & 1) << 1 | t >> 1;
    };
    auto key = [&](int row) { return SK == 8 ? quarter(row) << 1 | (row >> 1 & 1) : quarter(row); };
    auto bf16_key = [&](int row) { return quarter(row) << 2 | (row & 3); };
    const int a_chk = (lane % SK) ^ key(wave * AR + lane / SK);                // (a wave's loads are NW, a multiple of 4, apart)
    // bf16 rows: 16 chunks, 4 rows a load, chunk c of row t at slot c ^ bf16_key(t)
    static_assert(MX || SK == 4, "bf16 rows of 256 bytes");
    constexpr int BC = MX ? SK : 4 * SK, BR = 64 / BC;
    const int b_row = wave * BR + lane / BC;
    const int b_chk = (lane % BC) ^ (MX ? key(b_row) : bf16_key(b_row)), b_blk = MX ? b_chk : b_chk / 4;
    // scales with their stage: SCB bytes a lane, zero-extended to a dword; chunks: 16
    // bytes of a row's 32, the halves of rows 8 to 15 of 16 swapped (banks again)
    constexpr int SL = CHUNK ? 2 : SK / SCB, SR = 64 / SL;
    const int s_row = lane / SL, s_blk = (CHUNK ? lane % SL ^ (s_row >> 3 & 1) : lane % SL) * SCB, s_off = s_row * KB + s_blk;
    uint8_t *chunks = lds + R * C::STAGE;

    // scale load f (of SR rows: the weights' first, then the activations') from block blk on
    auto scale_load = [&](int f, uint8_t *dst, int blk, bool past) {
        constexpr int FA = C::BM / SR;
        const bool b = MX && f >= FA;
        const int off = past ? FAR : (b ? f - FA : f) * SR * KB + blk + s_off;
        if constexpr (CHUNK) __builtin_amdgcn_raw_ptr_buffer_load_lds(b ? rsb : rsa, (lds_void *) (dst + f * 1024), 16, off, 0, 0, 0);
        else load_scales<C::SCB>(b ? rsb : rsa, dst + f * 256, off);
    };
    // a lane's own parts of these offsets. The loop takes them as new in every
    // stage, or the compiler keeps each load's whole offset in a register.
    int a_lane = lane / SK * K2 + a_chk * 16, b_lane = (int) (lane / BC * xrow) + b_chk * 16;
    int a_at = r * (SK * 16) + ((SK / 4 * g) ^ key(r)) * 16, s_at;
    if constexpr (CHUNK) s_at = r * 32 + (SK == 8 ? 2 * g : g);
    else if constexpr (SK == 8) s_at = r * C::SROW + (SCB == 2 ? 4 : 8) * g;
    else s_at = r * C::SROW + (SCB == 2 ? (g >> 1) * 4 + (g & 1) : 4 * g);
    // load q of this wave's for stage t (stages past the last: zeros, so that every wait counts the same)
    auto issue_one = [&](int t, int slot, int q) __attribute__((always_inline)) {
        uint8_t *st = lds + slot * C::STAGE;
        const int blk = t * SK;
        if (q < C::LA) {
            const int u = (wave + NW * q) % C::UA;
            const int off = u * (AR * K2) + a_lane;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void *) (st + u * 1024), 16, blk + a_chk < KB ? off : FAR, blk * 16, 0, 0);
        } else if (q < C::LA + C::LB) {
            const int u = (wave + NW * (q - C::LA)) % C::UB;
            const int off = u * (int) (BR * xrow) + b_lane;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *) (st + C::A_BYTES + u * 1024), 16, blk + b_blk < KB ? off : FAR,
                                                     t * C::XROW, 0, 0);
        } else {
            const int u = wave + NW * (q - C::LA - C::LB);
            if constexpr (!CHUNK) {
                scale_load(u % C::US, st + C::A_BYTES + C::B_BYTES, blk, blk + s_blk >= KB);
            } else {
                const int w = t + (R == 2 ? C::CS - 1 : C::CS), c = w / C::CS;
                scale_load(((w % C::CS) * C::USP + u % C::USP) % C::US, chunks + c % C::CHUNKS * C::CHUNK_BYTES, c * 32, false);
            }
        }
    };
    auto issue = [&](int t, int slot) {
#pragma unroll
        for (int q = 0; q < C::LOADS; ++q) issue_one(t, slot, q);
    };

    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    // Step ks of a stage: lane group g takes block SK / 4 * g + ks of every row.
    // The scale bytes of this lane's blocks of a stage, byte ks for step ks: base at its row 16 u
    auto scale_at = [&](const uint8_t *base, int u) __attribute__((always_inline)) -> int {
        const uint8_t *q = base + u * (CHUNK ? 512 : 16 * C::SROW) + s_at;
        if constexpr (CHUNK) return SK == 8 ? *(const uint16_t *) q : *q;
        else if constexpr (SK == 8) return SCB == 2 ? *(const int *) q : q[0] | q[4] << 8;
        else return *q;
    };
    constexpr int KS = SK / 4;
    struct Frags {
        u32x4 a[KS][TM], b[KS][MX ? TN : 4 * TN];
        int sa[TM], sx[MX ? TN : 1];
    };
    // read q of a stage's fragments
    constexpr int NSC = TM + (MX ? TN : 0), NKS = TM + (MX ? TN : 4 * TN), NR = NSC + KS * NKS;
    auto read_one = [&](int t, int slot, Frags &f, int q) __attribute__((always_inline)) {
        const uint8_t *st = lds + slot * C::STAGE, *sb = st + C::A_BYTES;
        if (q < NSC) {
            const uint8_t *ss = CHUNK ? chunks + t / C::CS % C::CHUNKS * C::CHUNK_BYTES + (t % C::CS * SK ^ (r >> 3) * 16) : sb + C::B_BYTES;
            const bool x = q >= TM;
            if (x) f.sx[MX ? q - TM : 0] = scale_at(ss, C::BM / 16 + wn * TN + q - TM);
            else f.sa[q] = scale_at(ss, wm * TM + q);
            return;
        }
        // what the first half of the products takes, then the rest of the second; activations first
        if constexpr (MX) {
            const int ks = (q - NSC) / NKS, u = (q - NSC) % NKS;
            if (u < TN) f.b[ks][u] = *(const u32x4 *) (sb + (wn * TN + u) * (16 * SK * 16) + (a_at ^ 16 * ks));
            else f.a[ks][u - TN] = *(const u32x4 *) (st + (wm * TM + u - TN) * (16 * SK * 16) + (a_at ^ 16 * ks));
        } else {
            const int u = q - NSC, a = u - 2 * TN, h = u < 2 * TN ? u : u - TM;
            if (a >= 0 && a < TM) f.a[0][a] = *(const u32x4 *) (st + (wm * TM + a) * (16 * SK * 16) + a_at);
            else f.b[0][h] = *(const u32x4 *) (sb + ((wn * TN + h % TN) * 16 + r) * C::XROW + ((4 * g + h / TN) ^ bf16_key(r)) * 16);
        }
    };
    constexpr int NR0 = MX ? NSC + NKS : NSC + 2 * TN + TM;               // reads of the first half
    // chunks hold the next row's scales past K (K % 128 == 0: past K for all of a lane group's blocks or none)
    auto scales_of = [&](int t, Frags &f) __attribute__((always_inline)) {
        if constexpr (CHUNK) {
            const int in = t * SK + KS * g < KB ? -1 : 0;
            EACH(q, 0, TM, f.sa[q] &= in;);
            if constexpr (MX) EACH(q, 0, TN, f.sx[q] &= in;);
        }
    };
    // product q of a stage
    constexpr int NM = (MX ? KS : 4) * TM * TN;
    bf16x8 av;
    auto multiply_one = [&](const Frags &f, int q) __attribute__((always_inline)) {
        const int ks = q / (TM * TN), i = q / TN % TM, j = q % TN;
        if constexpr (MX) {
            const u32x4 &a = f.a[ks][i], &b = f.b[ks][j];
            const i32x8 av = {(int) a[0], (int) a[1], (int) a[2], (int) a[3], 0, 0, 0, 0};
            const i32x8 bv = {(int) b[0], (int) b[1], (int) b[2], (int) b[3], 0, 0, 0, 0};
            if (ks == 1) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[i][j], 4, 4, 1, f.sa[i], 1, f.sx[j]);
            else acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[i][j], 4, 4, 0, f.sa[i], 0, f.sx[j]);
        } else {
            if (j == 0) av = mx_decode8_bf16(f.a[0][i][ks], mx_scale((uint32_t) f.sa[i] & 255u));
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(bf16x8, f.b[0][ks * TN + j]), acc[i][j], 0, 0, 0);
        }
    };

    if constexpr (CHUNK) {
        for (int f = wave; f < C::US; f += NW) scale_load(f, chunks, 0, false);
    }
#pragma unroll
    for (int s = 0; s < R; ++s) issue(s, s);
    Frags f0;
    wait_vm<(R - 1) * C::LOADS>();
    asm volatile("s_barrier" ::: "memory");
    EACH(q, 0, (C::HALVES ? NR0 : NR), read_one(0, 0, f0, q););
    scales_of(0, f0);
    int slot = 0;                                                              // of stage t
    // past it every wave has stage t in registers, whose slot is refilled, and
    // every wave's loads of stage t + 1 have landed
    auto fill = [&]() __attribute__((always_inline)) {
        wait_vm<(R - 2) * C::LOADS>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto step = [&](int t, Frags &now, Frags &next) __attribute__((always_inline)) {
        const int s1 = slot + 1 == R ? 0 : slot + 1;
        asm volatile("" : "+v"(a_lane), "+v"(b_lane), "+v"(a_at), "+v"(s_at));
        if constexpr (C::HALVES) {
            constexpr int H = NM / 2, GB = TM / 4 * TN * (MX ? 1 : 2), H0 = TM < 8 ? (3 * H + 3) / 4 : H, N1 = NR - NR0, H1 = H - GB;
            EACH(q, 0, H,
                multiply_one(now, q);
                EACH(u, q * N1 / H0, (q + 1) * N1 / H0 < N1 ? (q + 1) * N1 / H0 : N1, read_one(t, slot, now, NR0 + u););
                __builtin_amdgcn_sched_barrier(0););
            EACH(q, 0, GB, multiply_one(now, H + q););
            __builtin_amdgcn_sched_barrier(0);
            fill();
            EACH(q, 0, H1,
                multiply_one(now, H + GB + q);
                EACH(u, q * NR0 / H1, (q + 1) * NR0 / H1, read_one(t + 1, s1, next, u););
                EACH(u, q * C::LOADS / H1, (q + 1) * C::LOADS / H1, issue_one(t + R, slot, u););
                __builtin_amdgcn_sched_barrier(0););
        } else {
            constexpr int H0 = NM * 3 / 4;
            fill();
            EACH(q, 0, NM,
                multiply_one(now, q);
                EACH(u, q * NR / H0, (q + 1) * NR / H0 < NR ? (q + 1) * NR / H0 : NR, read_one(t + 1, s1, next, u););
                EACH(u, q * C::LOADS / NM, (q + 1) * C::LOADS / NM, issue_one(t + R, slot, u););
                __builtin_amdgcn_sched_barrier(0););
        }
        scales_of(t + 1, next);
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
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) store4(p, n0 + (wn * TN + j) * 16 + r, m0 + (wm * TM + i) * 16 + 4 * g, acc[i][j]);
}

template <class C>
__global__ __launch_bounds__(C::NW * 64) void mx_gemm_tile_kernel(const MxGemm p, int tiles_m, int tiles_n) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    mx_gemm_tile<C>(p, tiles_m, tiles_n, lds);
}

template <class C>
hipError_t launch_tile(const MxGemm &p, hipStream_t s) {
    const int tiles_m = (p.M + C::BM - 1) / C::BM, tiles_n = (p.N + C::BN - 1) / C::BN;
    const int64_t T = (int64_t) tiles_m * tiles_n;
    if ((T + 7) * C::NW * 64 >= MAX_THREADS) return in_two(p, [&](const MxGemm &q) { return launch_tile<C>(q, s); });
    lds_opt_in((const void *) mx_gemm_tile_kernel<C>, C::LDS);
    launch_kernel(mx_gemm_tile_kernel<C>, dim3((unsigned) ((T + 7) / 8 * 8)), dim3(C::NW * 64), C::LDS, s, p, tiles_m, tiles_n);
    return hipGetLastError();
}
template <int XT, int WM, int WN, int TM, int TN, int SK, int R, bool HALVES>
hipError_t launch_tile_k(const MxGemm &p, hipStream_t s) {
    if (p.K % 128 == 0) return launch_tile<Cfg<XT, WM, WN, TM, TN, SK, R, 16, HALVES>>(p, s);
    if (p.K % 64 == 0) return launch_tile<Cfg<XT, WM, WN, TM, TN, SK, R, 2, HALVES>>(p, s);
    return launch_tile<Cfg<XT, WM, WN, TM, TN, SK, R - (R > 2), 1, HALVES>>(p, s);
}

// Shapes, by number (TSK_MX_CFG), and the us of one tile a CU at K = 5120 without
// the launch (64 x 32 and 64 x 64: alone on a CU / among two or three). All were
// measured with scales in chunks; where K % 128 != 0 they come with their stage and
// the same table serves, though tiles then take longer (K = 5120 / 5056 / 5088:
// 4096 x 4096, MXFP4 49 / 58 / 65, 2047 x 2050, bf16 54 / 55 / 57; K = 4096 / 4032 /
// 4064: 1292 x 1024, MXFP4 11.8 / 13.0 / 15.2):
//        both operands MXFP4                  bf16 activations
//   1    256 x 256, 8 waves     44            -
//   2    128 x 256, 8 waves     26            256 x 128, 8 waves    72
//   3    128 x 128, 8 waves     16            the same              42
//   4    64 x 128, 8 waves      9             the same              26
//   5    64 x 32, 4 waves       3.4 / 3.4     the same              12.6 / 8.3
//   6    192 x 128, 8 waves     17.5          the same              50
//   7    128 x 192, 8 waves     17            the same              49
//   8    192 x 256, 8 waves     31            -
//   9    64 x 64, 4 waves       5.5 / 5       the same              19 / 13.9
//   11   rows kernel, 16 x 16 outputs (f32 activations too, as 12 to 15)
//   12   32 x 16,  13  32 x 32,  14  64 x 32,  15  64 x 16
//
// The choice is the shape of the least time: its tiles on the fullest of 256 CUs
// times that of one, by K, and 0.8 for every time that a CU starts over (first
// loads, stores). Some pairs (us, taken / next; outputs as rows x M): MXFP4,
// 4096 x 4096, K = 5120 256 x 256 49 / 128 x 256 65; 2047 x 2050, K = 5120 128 x 192
// 22.0 / 128 x 256 (144 tiles) 27.0 / 128 x 128 (272) 34.8, with bf16 activations
// 48.1 / 61.0 / 73.9; 1292 x 1024, K = 4096 64 x 128 11.2 / 64 x 64 11.0 / 128 x 128
// 14.8; 388 x 4096, K = 1024 64 x 128 5.7 / 128 x 128 7.4, with bf16 9.2 / 11.2;
// 1024 x 1024, K = 1024 64 x 64 4.8 / 64 x 128 5.6; 388 x 1024, K = 4096 64 x 32 6.9 /
// 64 x 64 8.4, with bf16 14.1 / 19.5.
// Few rows, or too few tiles of the smallest shape: the rows kernel (us, 64 x 32
// tiles / rows: MXFP4, 17 x 8192, K = 8192 11.4 / 12.9; 64 x 4096, K = 4096, 128
// tiles 6.8 / 7.8, with bf16 activations 14.0 / 12.6; 32 x 4096, 64 tiles 6.7 / 6.5;
// bf16, 64 x 8192, K = 8192, 256 tiles 25.1 / 28.7), in the largest of its shapes
// that more than half of the CUs get, since of the next there would be two each
// (bf16, 96 x 1500, K = 2048, 141 of 32 x 32 7.3 / 282 of 32 x 16 8.4; 16 rows, M = K =
// 4096, 256 of 16 x 16 7.1 / 128 of 32 x 16 8.7; 8 rows, M = K = 8192, 256 of 32 x 16
// 12.6 / 128 of 64 x 16 18).
template <int XT>
int shape_for(const MxGemm &p) {
    if (tuning().mx_cfg) return tuning().mx_cfg;
    auto tiles = [&](int bm, int bn) { return (int64_t) ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    if constexpr (XT != X_F32) {
        constexpr bool MX = XT == X_MX;
        struct Shape { int bm, bn, on_a_cu; double alone, us; };
        constexpr Shape shapes[9] = {{256, 256, 1, 0, 44},
                                     {MX ? 128 : 256, MX ? 256 : 128, 1, 0, MX ? 26 : 72},
                                     {128, 128, 1, 0, MX ? 16 : 42},
                                     {64, 128, 1, 0, MX ? 9 : 26},
                                     {64, 32, 3, MX ? 3.4 : 12.6, MX ? 3.4 : 8.3},
                                     {192, 128, 1, 0, MX ? 17.5 : 50},
                                     {128, 192, 1, 0, MX ? 17 : 49},
                                     {192, 256, 1, 0, 31},
                                     {64, 64, 2, MX ? 5.5 : 19, MX ? 5 : 13.9}};
        if (p.N > (MX ? 16 : 32) && tiles(64, 32) >= (MX ? 100 : 130)) {
            int best = 0;
            double least = 0;
            for (int i = 0; i < 9; ++i) {
                const Shape &c = shapes[i];
                if (!MX && (i == 0 || i == 7)) continue;
                const double each = (double) ((tiles(c.bm, c.bn) + 255) / 256);      // tiles of a CU
                const double cost = std::max(c.alone, each * c.us) * p.K / 5120 + std::ceil(each / c.on_a_cu) * 0.8;
                if (!best || cost < least) {
                    best = i + 1;
                    least = cost;
                }
            }
            return best;
        }
    }
    if (p.N <= 16) return tiles(64, 16) > 128 ? 15 : tiles(32, 16) > 128 ? 12 : 11;
    return tiles(64, 32) > 128 ? 14 : tiles(32, 32) > 128 ? 13 : tiles(32, 16) > 128 ? 12 : 11;
}

template <int XT>
hipError_t launch_kind(const MxGemm &p, hipStream_t s) {
    int shape = shape_for<XT>(p);
    if constexpr (XT != X_F32) {
        constexpr bool MX = XT == X_MX;
        // a tile's offsets have 31 bits (else the rows kernel, whose addresses have 64)
        const int64_t xrow = MX ? p.K / 2 : p.ld_x * 2, most = (int64_t) 1 << 31;
        if (256 * (int64_t) (p.K / 2) >= most || 256 * xrow + (int64_t) p.K * 2 >= most) shape = std::max(shape, 11);
        switch (shape) {
            case 1: if constexpr (MX) return launch_tile_k<XT, 2, 4, 8, 4, 8, 2, true>(p, s);
            [[fallthrough]];
            case 2: if constexpr (MX) return launch_tile_k<XT, 2, 4, 4, 4, 8, 2, true>(p, s);
                    else return launch_tile_k<XT, 4, 2, 4, 4, 4, 2, true>(p, s);
            case 3: if constexpr (MX) return launch_tile_k<XT, 2, 4, 4, 2, 8, 3, true>(p, s);
                    else return launch_tile_k<XT, 4, 2, 2, 4, 4, 3, true>(p, s);
            case 4: return launch_tile_k<XT, 2, 4, 2, 2, MX ? 8 : 4, 3, true>(p, s);
            case 5: return launch_tile_k<XT, 4, 1, 1, 2, MX ? 8 : 4, 3, false>(p, s);
            case 6: return launch_tile_k<XT, 4, 2, 3, 4, MX ? 8 : 4, MX ? 3 : 2, true>(p, s);
            case 7: if constexpr (MX) return launch_tile_k<XT, 2, 4, 4, 3, 8, 3, true>(p, s);
                    else return launch_tile_k<XT, 4, 2, 2, 6, 4, 2, true>(p, s);
            case 8: if constexpr (MX) return launch_tile_k<XT, 2, 4, 6, 4, 8, 2, true>(p, s);
                    break;
            case 9: return launch_tile_k<XT, 2, 2, 2, 2, MX ? 8 : 4, 3, false>(p, s);
        }
    }
    switch (shape) {
        case 14: return launch_rows<XT, 4, 2, 4>(p, s);
        case 15: return launch_rows<XT, 4, 1, 4>(p, s);
        case 13: return launch_rows<XT, 2, 2, 4>(p, s);
        case 12: return launch_rows<XT, 2, 1, 4>(p, s);
        default: return launch_rows<XT, 1, 1, 4>(p, s);
    }
}

}  // namespace

hipError_t launch_gemm_mx(const MxGemm &p, hipStream_t s) {
    return p.xq ? launch_kind<X_MX>(p, s) : p.x_f32 ? launch_kind<X_F32>(p, s) : launch_kind<X_BF16>(p, s);
}

}  // namespace tsk
