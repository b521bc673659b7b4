// attn_cross.hip — attention of tokens to an encoder's states of another length,
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j]  over the states j that count,
//
// in one pass over the states with a running maximum and sum. A state counts if it is
// below its sequence's length and its flag is set; where none does, o is 0. The query heads that
// share a key and value head stand below one another as rows of one problem.
//
// A wave holds 32 rows. Per tile of states (v_mfma_f32_32x32x16, fp32 sums):
//   S^T = K Q^T      states x rows: lane l owns row l % 32 and half of the states,
//   P^T = exp2(scale log2(e) S^T - m) in K's 16-bit type,
//   O^T += V^T P^T   the sums of the first product lie as the second one's operand does.
// P is rounded to K's type (bf16 within 2^-8, f16 2^-11), its row sum adds the same rounded
// values, so that the weights add up to 1. With TWO (the caller's choice), what that rounding loses is a
// second part of K's type, which multiplies V as well, and the sum adds the weights as they are. Error of the
// norm into f32, 512 tokens to 4096 states of heads of 128, and us of 4096 tokens to 8192 states of 16 heads of 128 / of one
// token of 4 x 32 heads to 16384 states of 8: bf16 one part 1.4e-3, 267 / 57.9, two 2.0e-6, 358 / 58.3; f16 one 1.7e-4, 270,
// two 2.8e-7, 368. (Rounding an output to bf16 alone is 1.7e-3, to f16 2.1e-4.)
#include <algorithm>
#include <utility>

#include "tsk_common.h"
#include "tsk_internal.h"
#include "tsk_runtime.h"

namespace tsk {

namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// In each group of 16 lanes, lane i gets, as element j, element i % 4 of the 8
// bytes that lane 4 j + i / 4 addresses: with lane s at row r0 + s / 4, columns c0 +
// 4 (s % 4) .. + 3, lane i receives rows r0 .. r0 + 3 of column c0 + i
__device__ __forceinline__ s16x4 read_turned(const uint16_t *p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *) (p)); }

// Piece c (16 bytes) of row t of a tile in LDS lies at slot c ^ key(t). K: a 16-byte read of a wave
// takes one piece of 32 rows in turns of 16 lanes (0-3, 12-15, 20-27; 4-11, 16-19, 28-31; ...): the
// keys send those to 16 places. V: the four rows of a transposing read, 64 bytes each
// Values of a state's row in LDS (64 or 128, which the keys below need), of which the first DQ, D
// rounded up to 32, are multiplied: 4096 tokens to 8192 states of 16 heads of 72 217 us (all 128
// 240), of 96 216 (238), of 32 132 (64: 140)
constexpr int row_of_lds(int DQ) { return DQ <= 64 ? 64 : 128; }
template <int DP> __device__ __forceinline__ int k_key(int row) { return DP == 128 ? row & 15 : row >> 1 & 7; }
template <int DP> __device__ __forceinline__ int v_key(int row) { return (DP == 128 ? 4 : 2) * (row & 3); }

// 16 bytes a lane from base + off (the lane's) + at into LDS at byte dst + 16 * lane; zeros where off + at (it does not wrap) passes
// `bytes`. In assembly, since the compiler waits for every load into LDS before a transposing
// read, whose address it does not see; it has no result register, and the waits for it are
// written out where its bytes are read.
__device__ __forceinline__ void load_lds(const void *base, int bytes, int off, int at, uint32_t dst) {
    auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };   // (all the same for every lane)
    const i32x4 rs = {scalar((int) (uint32_t) (uintptr_t) base), scalar((int) ((uint32_t) ((uintptr_t) base >> 32) & 0xffffu)), scalar(bytes), 0x00020000};
    const int m = scalar((int) dst);
    uint32_t kept;                                             // (m0 is the compiler's; s_nop: scalars that a vector unit has just written)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(kept) : "s"(m), "v"(off), "s"(rs), "s"(scalar(at)) : "memory");
}

__device__ __forceinline__ uint32_t lds_byte(uint16_t *p) { return (uint32_t) (uintptr_t) (lds_void *) p; }

template <bool BF16> struct Half;
template <> struct Half<true> {
    typedef bf16x8 x8;
    typedef bf16x2 x2;
    typedef __bf16 one;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float add2(uint32_t p, float s) {
        const x2 ones = {(one) 1.0f, (one) 1.0f};
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(x2, p), ones, s, false);
    }
    static __device__ __forceinline__ uint32_t pack2(float f, float g) {
        const x2 v = {(one) f, (one) g};
        return __builtin_bit_cast(uint32_t, v);
    }
    // what f and g lose in pack2
    static __device__ __forceinline__ uint32_t rest2(float f, float g, uint32_t two) {
        const float a = __uint_as_float(two << 16), b = __uint_as_float(two & 0xffff0000u);
        return pack2(f - a, g - b);
    }
};
template <> struct Half<false> {
    typedef f16x8 x8;
    typedef f16x2 x2;
    typedef _Float16 one;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ float add2(uint32_t p, float s) {
        const x2 ones = {(one) 1.0f, (one) 1.0f};
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(x2, p), ones, s, false);
    }
    static __device__ __forceinline__ uint32_t pack2(float f, float g) {
        const x2 v = {(one) f, (one) g};
        return __builtin_bit_cast(uint32_t, v);
    }
    // what f and g lose in pack2
    static __device__ __forceinline__ uint32_t rest2(float f, float g, uint32_t two) {
        const x2 h = __builtin_bit_cast(x2, two);
        const float a = (float) h[0], b = (float) h[1];
        return pack2(f - a, g - b);
    }
};

// 8 values of a query row in K's type
template <bool BF16>
__device__ __forceinline__ u32x4 load_q8(const char *row, int d, int type) {
    if (type == (BF16 ? TSK_TYPE_BF16 : TSK_TYPE_F16)) return *(const u32x4 *) (row + 2 * d);
    float f[8];
    if (type == TSK_TYPE_F32) {
        const f32x4 a = *(const f32x4 *) (row + 4 * d), b = *(const f32x4 *) (row + 4 * d + 16);
        for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
    } else {
        const u32x4 r = *(const u32x4 *) (row + 2 * d);
        for (int i = 0; i < 8; ++i) {
            const uint16_t h = (uint16_t) (r[i / 2] >> 16 * (i & 1));
            f[i] = BF16 ? f16_bits_to_f32(h) : bf16_bits_to_f32(h);
        }
    }
    u32x4 o;
    for (int i = 0; i < 4; ++i) o[i] = Half<BF16>::pack2(f[2 * i], f[2 * i + 1]);
    return o;
}

// f(0), ..., f(N - 1), the arguments constants
template <class F, int... I>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
#define EACH(q, from, to, ...) each([&](auto q##_) __attribute__((always_inline)) { constexpr int q = decltype(q##_)::value + (from); __VA_ARGS__ }, std::make_integer_sequence<int, ((to) > (from) ? (to) - (from) : 0)>{})

// piece f of a step's 2 NK operands: two of K, one of V, ..., what is left of V
__host__ __device__ constexpr bool piece_of_k(int NK, int f) { return f < NK / 2 * 3 && f % 3 != 2; }
__host__ __device__ constexpr int piece_index(int NK, int f) { return f >= NK / 2 * 3 ? f - NK : f % 3 == 2 ? f / 3 : f / 3 * 2 + f % 3; }

// A launch's unit: a tile of rows of one key and value head, and (splits > 1) one of the
// ranges that its sequence's tiles of states are dealt to. The ranges go by the sequence's own
// length, which the device alone knows: `per` tiles each, the last ones empty.
struct Unit {
    int b, hk, nkv, nq, tile0, tile1, split;
    int64_t r0, R;
    bool none;
};
template <int KT>
__device__ __forceinline__ Unit unit_of(const CrossAttn &p, int qtiles, int rows) {
    Unit u;
    // Workgroup L runs on XCD L % 8. From 8 key and value heads on (of all sequences), XCD x takes
    // heads x, x + 8, ...: a head's states stay in one L2, neighbouring heads are read at the
    // same time, and sequences of other lengths spread over all XCDs. Units are numbered with
    // the ranges fastest, then the tiles of rows, then the heads
    // (fewer than 2^23; the quotients come from vector units, and are the same for every lane)
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int per_head = qtiles * p.splits, heads = p.Hkv * p.B;
    int head, in;
    if (heads >= 8) {
        const int j = (int) (blockIdx.x >> 3), g = uniform(j / per_head);
        head = 8 * g + (int) (blockIdx.x & 7);
        in = j - g * per_head;
    } else {
        head = uniform((int) blockIdx.x / per_head);
        in = (int) blockIdx.x - head * per_head;
    }
    u.none = head >= heads;
    if (u.none) return u;
    const int qt = uniform(in / p.splits);
    u.split = in - qt * p.splits;
    u.b = uniform(head / p.Hkv);
    u.hk = head - u.b * p.Hkv;
    u.nkv = uniform(p.kv_len ? max(0, min(p.kv_len[u.b], p.Nkv)) : p.Nkv);
    u.nq = uniform(p.q_len ? max(0, min(p.q_len[u.b], p.Nq)) : p.Nq);
    const int G = p.H / p.Hkv, tiles = (u.nkv + KT - 1) / KT, per = uniform((tiles + p.splits - 1) / p.splits);
    u.R = (int64_t) G * p.Nq;
    u.r0 = (int64_t) qt * rows;
    u.tile0 = u.split * per;
    u.tile1 = min(tiles, u.tile0 + per);
    // (a first range without states writes its zeros)
    u.none = u.nq == 0 || (G == 1 && u.r0 >= u.nq) || (u.split > 0 && u.tile0 >= u.tile1);
    return u;
}
// ranges of a sequence that hold states (1 for one that has none)
template <int KT>
__device__ __forceinline__ int used_splits(const CrossAttn &p, int nkv) {
    const int tiles = (nkv + KT - 1) / KT, per = (tiles + p.splits - 1) / p.splits;
    return per ? (tiles + per - 1) / per : 1;
}

// head and token of row r of a key and value head's rows
__device__ __forceinline__ void row_of(const CrossAttn &p, int hk, int64_t r, int &h, int &iq) {
    const int g = (int) (r / p.Nq);
    h = hk * (p.H / p.Hkv) + g;
    iq = (int) (r - (int64_t) g * p.Nq);
}
// (tokens past the sequence's last may hold anything, and a wave's rows decide together when their maxima move: they are zeros)
template <int DQ, bool BF16>
__device__ __forceinline__ void load_q(const CrossAttn &p, const Unit &u, int h, int iq, int hi, typename Half<BF16>::x8 (&q)[DQ / 16]) {
    const char *row = (const char *) p.q + iq * p.q_nb1 + h * p.q_nb2 + u.b * p.q_nb3;
#pragma unroll
    for (int ks = 0; ks < DQ / 16; ++ks) {
        const int d = 16 * ks + 8 * hi;
        const u32x4 zero = {0, 0, 0, 0};
        q[ks] = __builtin_bit_cast(typename Half<BF16>::x8, iq < u.nq && d < p.D ? load_q8<BF16>(row, d, p.q_type) : zero);
    }
}
// a rounded product, whatever is added to it
__device__ __forceinline__ float times(float a, float b) {
    float v = a * b;
    asm volatile("" : "+v"(v));
    return v;
}
// 1 / the sum of the weights; 0 where there are none, and a NaN stays
__device__ __forceinline__ float inverse(float l) { return l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l; }
// 4 values of an output row from dim d on
__device__ __forceinline__ void store_o4(const CrossAttn &p, char *row, int d, f32x4 v) {
    if (p.o_type == TSK_TYPE_F32) {
        *(f32x4 *) (row + d * 4) = v;
    } else if (p.o_type == TSK_TYPE_BF16) {
        *(u32x2 *) (row + d * 2) = u32x2{f32_to_bf16_bits(v[0]) | (uint32_t) f32_to_bf16_bits(v[1]) << 16,
                                        f32_to_bf16_bits(v[2]) | (uint32_t) f32_to_bf16_bits(v[3]) << 16};
    } else {
        *(u32x2 *) (row + d * 2) = u32x2{f32_to_f16_bits(v[0]) | (uint32_t) f32_to_f16_bits(v[1]) << 16,
                                        f32_to_f16_bits(v[2]) | (uint32_t) f32_to_f16_bits(v[3]) << 16};
    }
}
__device__ __forceinline__ char *o_row(const CrossAttn &p, int b, int h, int iq) {
    return (char *) p.o + h * p.o_nb1 + iq * p.o_nb2 + b * p.o_nb3;
}
// Scratch of splits > 1: per range and row (i = (b * Hkv + hk) * R + r) D sums, then for all of
// them the maximum and the sum of the weights
__device__ __forceinline__ int64_t all_rows(const CrossAttn &p) { return (int64_t) p.B * p.H * p.Nq; }
__device__ __forceinline__ float *part_o(const CrossAttn &p, int split, int64_t i) { return p.part + (split * all_rows(p) + i) * p.D; }
__device__ __forceinline__ float *part_ml(const CrossAttn &p, int split, int64_t i) {
    return p.part + (int64_t) p.splits * all_rows(p) * p.D + (split * all_rows(p) + i) * 2;
}

// ---------------------------------------------------------------- few rows
// A workgroup takes 32 rows, its four waves tiles of 32 states in turns, each through a ring
// of its own in LDS: no barrier until their sums meet. Bound by the states' bytes: one token of
// 4 sequences of 32 heads to 16384 states of 8 heads of 128, bf16, in 16 ranges: 57.5 us, 4.7 TB/s
// (a copy 5.1); with the kernel for many rows 62.
template <int DQ, bool BF16, bool TWO>
__global__ __launch_bounds__(256) void cross_attn_few_kernel(const CrossAttn p, int qtiles) {
    typedef Half<BF16> T;
    typedef typename T::x8 x8;
    constexpr int DP = row_of_lds(DQ), KT = 32, CH = DP / 8, RL = 64 / CH, NL = KT / RL, TILE = KT * DP, NB = 2;
    constexpr int FAR = (int) 0x80000000u, OS = DP + 4;
    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];           // [wave][NB][K tile, V tile]
    __shared__ float mls[4][2][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const Unit u = unit_of<KT>(p, qtiles, 32);
    if (u.none) return;
    int h, iq;
    row_of(p, u.hk, std::min<int64_t>(u.r0 + l32, u.R - 1), h, iq);
    const char *kp = (const char *) p.k + u.hk * p.k_nb2 + u.b * p.k_nb3, *vp = (const char *) p.v + u.hk * p.v_nb2 + u.b * p.v_nb3;
    const uint8_t *flags = p.kv_valid ? p.kv_valid + u.b * p.kv_valid_nb : nullptr;
    const int lr = lane / CH;
    uint16_t *ring = lds + wave * NB * 2 * TILE;
    const uint32_t ring0 = lds_byte(ring);
    auto issue = [&](int tile, int buf) {
        const uint32_t dst = ring0 + buf * (4 * TILE);
        const int left = min(KT, u.nkv - tile * KT);
        const int64_t k0 = (int64_t) tile * KT;
        const char *ks = kp + k0 * p.k_nb1, *vs = vp + k0 * p.v_nb1;
        // rows past the last state read as zeros
        const int k_bytes = (int) ((left - 1) * p.k_nb1) + 2 * p.D, v_bytes = (int) ((left - 1) * p.v_nb1) + 2 * p.D;
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const int kc = (lane % CH) ^ k_key<DP>(j * RL + lr), vc = (lane % CH) ^ v_key<DP>(lr);
            load_lds(ks, k_bytes, kc * 8 < p.D ? (int) (lr * p.k_nb1) + kc * 16 : FAR, (int) (j * RL * p.k_nb1), dst + j * 1024);
            load_lds(vs, v_bytes, vc * 8 < p.D ? (int) (lr * p.v_nb1) + vc * 16 : FAR, (int) (j * RL * p.v_nb1), dst + 2 * TILE + j * 1024);
        }
    };
    const int first = u.tile0 + wave;
    if (first < u.tile1) issue(first, 0);
    x8 q[DQ / 16];
    load_q<DQ, BF16>(p, u, h, iq, hi, q);
    f32x16 o[DQ / 32];
#pragma unroll
    for (int db = 0; db < DQ / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] = 0.0f;
    float m_run = -__builtin_inff(), l_run = 0.0f;
    const float c = p.c;
    const int l16 = lane & 15, grp = (lane >> 4) & 1, vrow = 4 * hi + (l16 >> 2);
    int buf = 0;
    for (int t = first; t < u.tile1; t += 4, buf ^= 1) {
        const int left = u.nkv - t * KT;
        uint32_t count = left >= KT ? ~0u : (1u << left) - 1;
        if (flags) count &= (uint32_t) __ballot(l32 < left && flags[(int64_t) t * KT + l32]);
        // (the flags' loads are the wave's last: with them the tile has landed too)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t + 4 < u.tile1) issue(t + 4, buf ^ 1);
        uint16_t *kb = ring + buf * 2 * TILE, *vb = kb + TILE;
        if (count == 0) continue;
        if (flags && count != ~0u) {
            // a state that does not count may hold anything: 0 times it may not be 0
            if (!(count >> l32 & 1))
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) *(u32x4 *) (vb + l32 * DP + hi * (DP / 2) + i * 8) = u32x4{0, 0, 0, 0};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        f32x16 s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < DQ / 16; ++ks) s = T::mfma(*(const x8 *) (kb + l32 * DP + (((2 * ks + hi) ^ k_key<DP>(l32)) << 3)), q[ks], s);
        if (count != ~0u) {
            const uint32_t mine = count >> 4 * hi;
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!(mine >> (8 * (e >> 2) + (e & 3)) & 1)) s[e] = -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        const float m_new = fmaxf(m_run, times(half_pair_max(top), c));
        const float sub = m_new == -__builtin_inff() ? 0.0f : m_new, alpha = __builtin_amdgcn_exp2f(m_run - sub);
        if (__any(m_new > m_run)) {
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < DQ / 32; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
        }
        m_run = m_new;
        u32x4 pf[TWO ? 2 : 1][2];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            // (logits times c are rounded as the maximum was: no weight is above 1)
            const float w0 = __builtin_amdgcn_exp2f(times(s[e], c) - sub), w1 = __builtin_amdgcn_exp2f(times(s[e + 1], c) - sub);
            const uint32_t two = T::pack2(w0, w1);
            pf[0][e / 8][e % 8 / 2] = two;
            if constexpr (TWO) {
                pf[1][e / 8][e % 8 / 2] = T::rest2(w0, w1, two);
                l_run += w0 + w1;
            } else l_run = T::add2(two, l_run);
        }
#pragma unroll
        for (int kg = 0; kg < 2; ++kg)
#pragma unroll
            for (int db = 0; db < DQ / 32; ++db) {
                const int ch = 4 * db + 2 * grp + ((l16 & 3) >> 1);
                const uint16_t *at = vb + (16 * kg + vrow) * DP + ((ch ^ v_key<DP>(l16 >> 2)) << 3) + 4 * (l16 & 1);
                const s16x4 a = read_turned(at), a2 = read_turned(at + 8 * DP);
                const s16x8 a8 = {a[0], a[1], a[2], a[3], a2[0], a2[1], a2[2], a2[3]};
#pragma unroll
                for (auto &part : pf) o[db] = T::mfma(__builtin_bit_cast(x8, a8), __builtin_bit_cast(x8, part[kg]), o[db]);
            }
        // (the next turn's loads land in the buffer read here: every read is done)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    // the four waves' sums, brought to one maximum, meet in LDS: [wave][row][dim]
    const float l_all = half_pair_sum(l_run);
    if (hi == 0) {
        mls[wave][0][l32] = m_run;
        mls[wave][1][l32] = l_all;
    }
    __syncthreads();
    float *os = (float *) lds;
    float m = mls[0][0][l32];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, mls[w][0][l32]);
    const float f = __builtin_amdgcn_exp2f(m_run - (m == -__builtin_inff() ? 0.0f : m));
#pragma unroll
    for (int db = 0; db < DQ / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *(f32x4 *) (os + (wave * 32 + l32) * OS + 32 * db + 2 * e + 4 * hi) = f32x4{o[db][e], o[db][e + 1], o[db][e + 2], o[db][e + 3]} * f;
    __syncthreads();
    const int64_t left = u.R - u.r0;
    const int rows = left < 32 ? (int) left : 32, D4 = p.D / 4;
    for (int i = tid; i < rows * D4; i += 256) {
        const int r = i / D4, d = (i - r * D4) * 4;
        float mr = mls[0][0][r], l = 0.0f;
        for (int w = 1; w < 4; ++w) mr = fmaxf(mr, mls[w][0][r]);
        const float sub = mr == -__builtin_inff() ? 0.0f : mr;
        f32x4 v = {0, 0, 0, 0};
        for (int w = 0; w < 4; ++w) {
            l += mls[w][1][r] * __builtin_amdgcn_exp2f(mls[w][0][r] - sub);
            v += *(const f32x4 *) (os + (w * 32 + r) * OS + d);
        }
        int hr, iqr;
        row_of(p, u.hk, u.r0 + r, hr, iqr);
        if (iqr >= u.nq) continue;
        if (p.splits > 1) {
            const int64_t at = ((int64_t) u.b * p.Hkv + u.hk) * u.R + u.r0 + r;
            *(f32x4 *) (part_o(p, u.split, at) + d) = v;
            if (d == 0) {
                float *ml = part_ml(p, u.split, at);
                ml[0] = mr;
                ml[1] = l;
            }
        } else {
            store_o4(p, o_row(p, u.b, hr, iqr), d, v * inverse(l));
        }
    }
}

// The ranges of a row brought together: a thread takes 4 dims and every G-th range, all of
// whose reads are on their way at once; G threads' sums meet in LDS (G a power of two, ranges
// up to 256 / (DP / 4))
template <int KT, int DP>
__global__ __launch_bounds__(256) void cross_attn_join_kernel(const CrossAttn p, int G) {
    constexpr int T4 = DP / 4, NG = 256 / T4, MOST = CROSS_ATTN_SPLITS / NG;
    __shared__ float ms[NG], ls[NG];
    __shared__ __attribute__((aligned(16))) f32x4 vs[256];
    const int seat = threadIdx.x / T4, g = seat % G, d = threadIdx.x % T4 * 4;
    const int64_t mine = (int64_t) blockIdx.x * (NG / G) + seat / G, rows = all_rows(p), at = std::min<int64_t>(mine, rows - 1);
    const int64_t R = (int64_t) (p.H / p.Hkv) * p.Nq, unit = at / R;
    const int b = (int) (unit / p.Hkv), hk = (int) (unit % p.Hkv);
    int h, iq;
    row_of(p, hk, at - unit * R, h, iq);
    // (rows of tokens past the last are in no range, and are not stored)
    const bool there = mine < rows && !(p.q_len && iq >= p.q_len[b]);
    const int used = there ? used_splits<KT>(p, p.kv_len ? max(0, min(p.kv_len[b], p.Nkv)) : p.Nkv) : 0;
    float mv[MOST], lv[MOST], m = -__builtin_inff(), l = 0.0f;
    f32x4 ov[MOST], v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int s = g + G * i;
        const bool in = s < used;
        mv[i] = in ? part_ml(p, s, at)[0] : -__builtin_inff();
        lv[i] = in ? part_ml(p, s, at)[1] : 0.0f;
        ov[i] = in && d < p.D ? *(const f32x4 *) (part_o(p, s, at) + d) : v;
    }
#pragma unroll
    for (int i = 0; i < MOST; ++i) m = fmaxf(m, mv[i]);
    const float sub = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const float f = __builtin_amdgcn_exp2f(mv[i] - sub);
        l += lv[i] * f;
        v += ov[i] * f;
    }
    if (d == 0) {
        ms[seat] = m;
        ls[seat] = l;
    }
    vs[threadIdx.x] = v;
    __syncthreads();
    if (g > 0 || d >= p.D || !there) return;
    for (int i = 1; i < G; ++i) m = fmaxf(m, ms[seat + i]);
    const float all = m == -__builtin_inff() ? 0.0f : m;
    l = 0.0f;
    v = f32x4{0, 0, 0, 0};
    for (int i = 0; i < G; ++i) {
        const float f = __builtin_amdgcn_exp2f(ms[seat + i] - all);
        l += ls[seat + i] * f;
        v += vs[threadIdx.x + i * T4] * f;
    }
    store_o4(p, o_row(p, b, h, iq), d, v * inverse(l));
}

// ---------------------------------------------------------------- many rows
// A workgroup takes 32 NW rows, 32 a wave, and tiles of 64 states through a ring of four in
// LDS. Half a tile (32 states) at a time, a wave multiplies the next half's K with Q and the
// last half's V with P while it turns this half's logits into weights: three steps of three
// halves without a dependence, so that the matrix unit and the rest of the SIMD work at once.
// Products, LDS reads, loads and the softmax's operations are in the program's order
// (sched_barrier). 4096 tokens to 8192 states of 16 heads of 128, bf16: 243 us, 1130 TF/s (a
// library's matrix product of 8192^3 1390; 249 to 267 on other cards); the matrix unit is busy for 54 % of the cycles and
// the vector unit's exponentials, sums and roundings for most of the others. One half a step, each
// after the other, took 325 us, a largest logit found before each weight 251.
template <int DQ, bool BF16, int NW, bool TWO>
__global__ __launch_bounds__(NW * 64) void cross_attn_kernel(const CrossAttn p, int qtiles) {
    typedef Half<BF16> T;
    typedef typename T::x8 x8;
    constexpr int DP = row_of_lds(DQ), KT = 64, CH = DP / 8, RL = 64 / CH, NL = KT / RL / NW, TILE = KT * DP;     // 16-byte pieces a row, rows a load, loads a wave
    constexpr int FAR = (int) 0x80000000u;
    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];           // [4][K tile, V tile]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const Unit u = unit_of<KT>(p, qtiles, 32 * NW);
    if (u.none) return;
    const int64_t row = u.r0 + wave * 32 + l32;
    int h, iq;
    row_of(p, u.hk, std::min<int64_t>(row, u.R - 1), h, iq);
    x8 q[DQ / 16];
    load_q<DQ, BF16>(p, u, h, iq, hi, q);
    const char *kp = (const char *) p.k + u.hk * p.k_nb2 + u.b * p.k_nb3, *vp = (const char *) p.v + u.hk * p.v_nb2 + u.b * p.v_nb3;
    const uint8_t *flags = p.kv_valid ? p.kv_valid + u.b * p.kv_valid_nb : nullptr;
    // (a wave's loads are NW * RL rows apart, which the keys do not see)
    const int lr = lane / CH, kc = (lane % CH) ^ k_key<DP>(wave * RL + lr), vc = (lane % CH) ^ v_key<DP>(lr);
    const int koff = kc * 8 < p.D ? (int) (lr * p.k_nb1) + kc * 16 : FAR, voff = vc * 8 < p.D ? (int) (lr * p.v_nb1) + vc * 16 : FAR;
    // tile t into slot s, a load at a time; tiles past the last: zeros, so that every wait counts the same
    struct Source {
        const char *k, *v;
        int k_bytes, v_bytes;                                  // up to the last state that counts: rows past it read as zeros
    };
    auto source_of = [&](int t) {
        const int left = t < u.tile1 ? min(KT, u.nkv - t * KT) : 0;
        const int64_t k0 = t < u.tile1 ? (int64_t) t * KT : 0;
        return Source{kp + k0 * p.k_nb1, vp + k0 * p.v_nb1, left ? (int) ((left - 1) * p.k_nb1) + 2 * p.D : 0,
                      left ? (int) ((left - 1) * p.v_nb1) + 2 * p.D : 0};
    };
    const uint32_t lds0 = lds_byte(lds);
    constexpr int LOADS = 2 * NL;                              // of a wave and tile: K's and V's in turn
    auto issue_one = [&](const Source &src, int s, int i) __attribute__((always_inline)) {
        const int j = wave + NW * (i / 2);
        const uint32_t dst = lds0 + s * (4 * TILE) + i % 2 * (2 * TILE) + j * 1024;
        if (i % 2 == 0) load_lds(src.k, src.k_bytes, koff, (int) (j * RL * p.k_nb1), dst);
        else load_lds(src.v, src.v_bytes, voff, (int) (j * RL * p.v_nb1), dst);
    };
    // bit s: state s of tile t counts
    auto counted = [&](int t) -> uint64_t {
        const int left = u.nkv - t * KT;
        if (t >= u.tile1) return 0;
        uint64_t m = left >= KT ? ~(uint64_t) 0 : ((uint64_t) 1 << left) - 1;
        if (flags) m &= __ballot(lane < left && flags[(int64_t) t * KT + lane]);
        return m;
    };
    // a state that does not count may hold anything, and 0 times it may not be 0: its V becomes zeros
    auto clear = [&](uint64_t count, int s) {
        if (!flags || count == ~(uint64_t) 0) return;
        const int r = tid / NW;                                  // NW threads a row
        if (!(count >> r & 1))
#pragma unroll
            for (int i = 0; i < CH / NW; ++i) *(u32x4 *) (lds + s * 2 * TILE + TILE + r * DP + (tid % NW * (CH / NW) + i) * 8) = u32x4{0, 0, 0, 0};
        __syncthreads();
    };
    f32x16 o[DQ / 32];
#pragma unroll
    for (int db = 0; db < DQ / 32; ++db) o[db] = f32x16{};
    float m = -3.40282347e38f, l = 0.0f;                         // (below any logit; -inf would be no number less itself)
    float most = 256.0f;                                         // sum of a half's weights that stay as they are
    const float c = p.c;
    const int l16 = lane & 15, grp = (lane >> 4) & 1, vrow = 4 * hi + (l16 >> 2);
    struct Weights {
        u32x4 w[TWO ? 2 : 1][2];                                 // pairs, of each part
        float sum;
    };
    // A step's operands in LDS, K's of one half of a tile and V's of another, in the order of
    // their products: two of K, one of V, ..., what is left of V; each read AHEAD products early
    constexpr int NK = DQ / 16, NF = 2 * NK, AHEAD = 4, SLOTS = AHEAD + 1;
    struct Pieces {
        x8 f[SLOTS];
    };
    auto read_piece = [&](const uint16_t *kb, const uint16_t *vb, int f, Pieces &x) __attribute__((always_inline)) {
        const int j = piece_index(NK, f);
        if (piece_of_k(NK, f)) {
            x.f[f % SLOTS] = *(const x8 *) (kb + l32 * DP + (((2 * j + hi) ^ k_key<DP>(l32)) << 3));
        } else {
            const int kg = j / (DQ / 32), db = j % (DQ / 32), ch = 4 * db + 2 * grp + ((l16 & 3) >> 1);
            const uint16_t *at = vb + (16 * kg + vrow) * DP + ((ch ^ v_key<DP>(l16 >> 2)) << 3) + 4 * (l16 & 1);
            const s16x4 a = read_turned(at), a2 = read_turned(at + 8 * DP);
            const s16x8 a8 = {a[0], a[1], a[2], a[3], a2[0], a2[1], a2[2], a2[3]};
            x.f[f % SLOTS] = __builtin_bit_cast(x8, a8);
        }
    };
    auto k_at = [&](int slot, int half) { return lds + slot * 2 * TILE + 32 * half * DP; };
    auto v_at = [&](int slot, int half) { return lds + slot * 2 * TILE + TILE + 32 * half * DP; };
    // A logit becomes a weight in three turns, each some products after the one before (a wave
    // waits for its own results): the exponent, its power, and two of them rounded and added
    struct Turns {
        float v[16];
    };
    auto turn1 = [&](const f32x16 &n, Turns &r, int e) __attribute__((always_inline)) {
        float v = __builtin_fmaf(n[e], c, -m);
        asm volatile("" : "+v"(v));                              // (worked out here and not where it is used)
        r.v[e] = v;
    };
    auto turn2 = [&](Turns &r, int e) __attribute__((always_inline)) {
        float v = __builtin_amdgcn_exp2f(r.v[e]);
        asm volatile("" : "+v"(v));
        r.v[e] = v;
    };
    auto turn3 = [&](const Turns &r, Weights &w, int e) __attribute__((always_inline)) {
        uint32_t two = T::pack2(r.v[e], r.v[e + 1]);
        float sum = e == 0 ? 0.0f : w.sum;
        if constexpr (TWO) {
            uint32_t rest = T::rest2(r.v[e], r.v[e + 1], two);
            sum += r.v[e] + r.v[e + 1];
            asm volatile("" : "+v"(rest));
            w.w[1][e / 8][e % 8 / 2] = rest;
        } else sum = T::add2(two, sum);
        asm volatile("" : "+v"(two), "+v"(sum));
        w.sum = sum;
        w.w[0][e / 8][e % 8 / 2] = two;
    };
    constexpr int PER = (16 + NF - 1) / NF;                      // logits between two products
    auto first_turns = [&](const f32x16 &n, Turns &r) __attribute__((always_inline)) {
        EACH(e, 0, 2 * PER, turn1(n, r, e););
        EACH(e, 0, PER, turn2(r, e););
        __builtin_amdgcn_sched_barrier(0);
    };
    auto first_pieces = [&](const uint16_t *kb, const uint16_t *vb, Pieces &x) __attribute__((always_inline)) {
        EACH(f, 0, AHEAD, read_piece(kb, vb, f, x););
        __builtin_amdgcn_sched_barrier(0);
    };
    // piece j of V times its weights
    auto add_v = [&](const x8 &v, const Weights &w, auto j) __attribute__((always_inline)) {
        constexpr int KG = decltype(j)::value / (DQ / 32), DB = decltype(j)::value % (DQ / 32);
        o[DB] = T::mfma(v, __builtin_bit_cast(x8, w.w[0][KG]), o[DB]);
        if constexpr (TWO) o[DB] = T::mfma(v, __builtin_bit_cast(x8, w.w[1][KG]), o[DB]);
    };
    // the products of next (K . Q of a half) and of before (V of another), `now` weighed between
    // them, and one half (part) of the loads of a later tile
    auto step = [&](const uint16_t *kb, const uint16_t *vb, Pieces &x, const f32x16 &now, Turns &r, Weights &w, f32x16 &next,
                    const Weights &before, const Source &src, int to, auto part) __attribute__((always_inline)) {
        constexpr int L0 = decltype(part)::value * LOADS / 2, L1 = LOADS / 2;
        EACH(f, 0, NF,
            constexpr int J = piece_index(NK, f);
            if constexpr (piece_of_k(NK, f)) next = T::mfma(x.f[f % SLOTS], q[J], J == 0 ? f32x16{} : next);
            else add_v(x.f[f % SLOTS], before, std::integral_constant<int, J>{});
            if constexpr (f + AHEAD < NF) read_piece(kb, vb, f + AHEAD, x);
            EACH(i, f * L1 / NF, (f + 1) * L1 / NF, issue_one(src, to, L0 + i););
            EACH(i, 0, PER,
                if constexpr ((f + 2) * PER + i < 16) turn1(now, r, (f + 2) * PER + i);
                if constexpr ((f + 1) * PER + i < 16) turn2(r, (f + 1) * PER + i);
                if constexpr ((f * PER + i) % 2 && f * PER + i < 16) turn3(r, w, f * PER + i - 1););
            __builtin_amdgcn_sched_barrier(0););
    };
    // the same alone, before the first step and after the last
    auto multiply_k = [&](const uint16_t *kb, f32x16 &n) __attribute__((always_inline)) {
        n = f32x16{};
        EACH(f, 0, NF, if constexpr (piece_of_k(NK, f)) {
            Pieces x;
            read_piece(kb, kb, f, x);
            n = T::mfma(x.f[f % SLOTS], q[piece_index(NK, f)], n);
        });
    };
    auto multiply_v = [&](const uint16_t *vb, const Weights &w) __attribute__((always_inline)) {
        EACH(f, 0, NF, if constexpr (!piece_of_k(NK, f)) {
            constexpr int J = piece_index(NK, f);
            Pieces x;
            read_piece(vb, vb, f, x);
            add_v(x.f[f % SLOTS], w, std::integral_constant<int, J>{});
        });
    };
    auto weigh = [&](const f32x16 &n, Weights &w) __attribute__((always_inline)) {
        Turns r;
        EACH(e, 0, 16, r.v[e] = times(n[e], c) - m; turn2(r, e););
        EACH(e, 0, 8, turn3(r, w, 2 * e););
    };
    // states of a half that do not count leave before they are weighed
    auto leave = [&](f32x16 &n, uint64_t count, int half) __attribute__((always_inline)) {
        const uint32_t part = (uint32_t) (count >> 32 * half);
        if (part == ~0u) return;
        uint32_t mine = part >> 4 * hi;
        asm volatile("" : "+v"(mine));                           // (nothing of this is worked out ahead)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (!(mine >> (8 * (e >> 2) + (e & 3)) & 1)) n[e] = -__builtin_inff();
    };
    // Weights that have grown past 2^8 together (or are not finite): the maximum moves to a whole
    // number (log2 domain), what has been summed shrinks by a power of two, exactly, and they are
    // worked out again, from logits rounded as the maximum was, which leaves no weight above 1. The
    // sums tell it, so the logits' maximum is looked for only then. Past 2^22 the steps' unrounded
    // products with c differ from the rounded maximum by halves and more: there, all are
    // worked out again
    auto settle = [&](const f32x16 &n, Weights &w) __attribute__((always_inline)) {
        if (__any(!(w.sum <= most))) {
            float top = n[0];
            asm volatile("" : "+v"(top));
#pragma unroll
            for (int e = 1; e < 16; ++e) top = fmaxf(top, n[e]);
            const float to = fmaxf(m, __builtin_ceilf(times(half_pair_max(top), c))), f = __builtin_amdgcn_exp2f(m - to);
            m = to;
            most = __builtin_fabsf(to) < 0x1p22f ? 256.0f : -1.0f;
            l *= f;
#pragma unroll
            for (int db = 0; db < DQ / 32; ++db) o[db] *= f;
            weigh(n, w);
        }
        l += w.sum;
    };
    if (u.tile0 < u.tile1) {
        for (int t = 0; t < 3; ++t) {
            const Source src = source_of(u.tile0 + t);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) issue_one(src, t, i);
        }
        f32x16 na, nb;
        Weights wa, wb;
        uint64_t count = counted(u.tile0), next = counted(u.tile0 + 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");           // (tiles 0 and 1)
        __syncthreads();
        clear(count, 0);
        clear(next, 1);
        multiply_k(k_at(0, 0), na);
        leave(na, count, 0);
        weigh(na, wa);
        settle(na, wa);
        multiply_k(k_at(0, 1), nb);
        int slot = 0;
        Pieces x;
        Turns r;
        for (int t = u.tile0; t + 1 < u.tile1; ++t) {
            const int s1 = (slot + 1) & 3, s2 = (slot + 2) & 3, s3 = (slot + 3) & 3;
            // second half of tile t; tile t + 3 goes where tile t - 1 was, which every wave is done with
            const Source src = source_of(t + 3);
            first_pieces(k_at(s1, 0), v_at(slot, 0), x);
            leave(nb, count, 1);
            first_turns(nb, r);
            step(k_at(s1, 0), v_at(slot, 0), x, nb, r, wb, na, wa, src, s3, std::integral_constant<int, 0>{});
            // first half of tile t + 1
            first_pieces(k_at(s1, 1), v_at(slot, 1), x);
            settle(nb, wb);
            leave(na, next, 0);
            first_turns(na, r);
            step(k_at(s1, 1), v_at(slot, 1), x, na, r, wa, nb, wb, src, s3, std::integral_constant<int, 1>{});
            settle(na, wa);
            count = next;
            next = counted(t + 2);
            // tile t + 2 has landed (t + 3 may be on its way)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
            __syncthreads();
            clear(next, s2);
            slot = s1;
        }
        leave(nb, count, 1);
        weigh(nb, wb);
        multiply_v(v_at(slot, 0), wa);
        settle(nb, wb);
        multiply_v(v_at(slot, 1), wb);
        // (no load may land in an LDS that is another workgroup's by then)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const float la = half_pair_sum(l), inv = inverse(la);
    if (row >= u.R || iq >= u.nq) return;
    const int64_t at = ((int64_t) u.b * p.Hkv + u.hk) * u.R + row;
    if (p.splits > 1 && hi == 0) {
        float *ml = part_ml(p, u.split, at);
        ml[0] = m;
        ml[1] = la;
    }
#pragma unroll
    for (int db = 0; db < DQ / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * db + 2 * e + 4 * hi;
            if (d >= p.D) continue;
            const f32x4 v = {o[db][e], o[db][e + 1], o[db][e + 2], o[db][e + 3]};
            if (p.splits > 1) *(f32x4 *) (part_o(p, u.split, at) + d) = v;
            else store_o4(p, o_row(p, u.b, h, iq), d, v * inv);
        }
}

template <class F>
hipError_t launch_units(F kern, const CrossAttn &p, int rows, int threads, size_t lds, hipStream_t s) {
    const int64_t R = (int64_t) (p.H / p.Hkv) * p.Nq, qtiles = (R + rows - 1) / rows, heads = (int64_t) p.Hkv * p.B;
    const int64_t units = (heads >= 8 ? (heads + 7) / 8 * 8 : heads) * qtiles * p.splits;
    if (units >= (int64_t) 1 << 23) return hipErrorInvalidValue;
    lds_opt_in((const void *) kern, lds);
    launch_kernel(kern, dim3((unsigned) units), dim3(threads), lds, s, p, (int) qtiles);
    return hipGetLastError();
}

template <int DQ, bool BF16, bool TWO>
hipError_t launch_dp(const CrossAttn &p, const CrossAttnPlan &plan, hipStream_t s) {
    constexpr int DP = row_of_lds(DQ);
    hipError_t e;
    if (plan.rows == 32) e = launch_units(cross_attn_few_kernel<DQ, BF16, TWO>, p, 32, 256, 4 * 2 * 2 * 32 * DP * 2, s);
    else if (plan.rows == 128) e = launch_units(cross_attn_kernel<DQ, BF16, 4, TWO>, p, 128, 256, 4 * 2 * 64 * DP * 2, s);
    else e = launch_units(cross_attn_kernel<DQ, BF16, 8, TWO>, p, 256, 512, 4 * 2 * 64 * DP * 2, s);
    if (e != hipSuccess || p.splits == 1) return e;
    constexpr int NG = 256 / (DP / 4);
    int G = 1;
    while (G < p.splits && G < NG) G *= 2;
    // (fewer than 2^24 rows, plan_cross_attn)
    const dim3 grid((unsigned) (((int64_t) p.B * p.H * p.Nq + NG / G - 1) / (NG / G)));
    if (plan.rows == 32) launch_kernel(cross_attn_join_kernel<32, DP>, grid, dim3(256), 0, s, p, G);
    else launch_kernel(cross_attn_join_kernel<64, DP>, grid, dim3(256), 0, s, p, G);
    return hipGetLastError();
}

}  // namespace

// Rows of a workgroup (32: cross_attn_few_kernel; 128, 256) and ranges of the states, by what
// each is estimated to take: turns of the workgroups that 256 CUs hold (two a CU of small ones),
// a turn's fixed part and tiles in us (alone on a CU, or sharing it), and the join of the ranges. The
// constants were fitted to such pairs (us, bf16; rows x ranges, the rule's first):
//   B 2, 646 tokens,   77 states, 16 heads of  64: 128 x 1   7.2, 32 x 1  10.2, 256 x 1   8.6
//   B 1, 4096,       8192,        16 heads of 128: 256 x 1 243.5, 128 x 1 308.9, 256 x 4 333.5
//   B 1, 4096,       8192,         2 heads of 128: 128 x 4  58.3, 256 x 4  70.9, 128 x 1 149.7
//   B 1, 300,        3000,         4 heads of 128:  32 x 4  18.4, 128 x 16 20.1, 32 x 1   32.2
//   B 4, 1000,       1000,         4 heads of 128: 128 x 1  25.3, 32 x 1  29.3, 256 x 1   32.7
//   B 4, 1,  16384, 32 heads on 8 of 128:           32 x 16 57.5, 128 x 16 61.9, 32 x 1  179.6
//   B 1, 1,   8192,        16 heads of  64:         32 x 16 13.4, 128 x 16 16.7, 32 x 1   46.3
// Lengths that are shorter than the states are not known here; then it may be some 20 % off. The constants are those of
// heads of 64 and of 128, which smaller heads of either kind take too.
CrossAttnPlan plan_cross_attn(int D, int64_t Nq, int64_t Nkv, int64_t H, int64_t Hkv, int64_t B) {
    CrossAttnPlan c = {128, 1, 0};
    const int64_t R = H / Hkv * Nq;
    const bool wide = D > 64;
    double least = 0;
    for (int kind = 0; kind < 3; ++kind) {
        const int rows = kind == 0 ? 32 : kind == 1 ? 128 : 256;
        const double units = (double) ((R + rows - 1) / rows) * (double) (Hkv * B);
        const double tiles = kind == 0 ? (double) ((Nkv + 127) / 128) : (double) ((Nkv + 63) / 64);     // of a wave
        const int on_a_cu = wide || kind == 2 ? 1 : 2;
        const double fixed = kind == 0 ? 3 : 2.5, alone = wide ? kind == 0 ? 1.12 : kind == 1 ? 1.2 : 1.93 : kind == 0 ? 0.55 : kind == 1 ? 0.84 : 1.17,
                     full = wide ? alone : kind == 0 ? 0.9 : kind == 1 ? 1.28 : 1.17;
        for (int s = 1; s <= CROSS_ATTN_SPLITS; s *= 2) {
            if (s > 1 && (s > (int) tiles || B * H * Nq >= (int64_t) 1 << 24)) break;
            const double on = units * s / 256, turns = std::ceil(on / on_a_cu), each = on <= 1 ? alone : full;
            double cost = turns * (fixed + std::ceil(tiles / s) * each);
            if (s > 1) cost += 3 + (double) (B * H * Nq) * s * D * 8 / 3e6;
            if (!least || cost < least) {
                least = cost;
                c.rows = rows;
                c.splits = s;
            }
        }
    }
    const int cfg = tuning().cross_cfg, forced = cfg / 100;
    if (forced == 32 || forced == 128 || forced == 256) {
        c.rows = forced;
        c.splits = std::max(1, std::min(cfg % 100, CROSS_ATTN_SPLITS));
    }
    c.bytes = c.splits > 1 ? (size_t) c.splits * (size_t) (B * H * Nq) * (size_t) (D + 2) * 4 : 0;
    c.bytes = (c.bytes + 255) / 256 * 256;
    return c;
}

hipError_t launch_cross_attn(const CrossAttn &p, const CrossAttnPlan &plan, hipStream_t s) {
    auto go = [&](auto bf16, auto two) {
        constexpr bool BF16 = decltype(bf16)::value, TWO = decltype(two)::value;
        if (p.D <= 32) return launch_dp<32, BF16, TWO>(p, plan, s);
        if (p.D <= 64) return launch_dp<64, BF16, TWO>(p, plan, s);
        if (p.D <= 96) return launch_dp<96, BF16, TWO>(p, plan, s);
        return launch_dp<128, BF16, TWO>(p, plan, s);
    };
    std::true_type t;
    std::false_type f;
    return p.kv_bf16 ? p.two_parts ? go(t, t) : go(t, f) : p.two_parts ? go(f, t) : go(f, f);
}

}  // namespace tsk
