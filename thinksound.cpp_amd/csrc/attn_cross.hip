// attn_cross.hip — attention of tokens to an encoder's states of another length,
//
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j]  over the states j that count,
//
// in one pass over the states with a running maximum and sum. A state counts if it is
// below its sequence's length and its flag is set; where none does, o is 0. The query heads that
// share a key and value head stand below one another as rows of one problem.
//
// A wave holds 32 rows. Per tile of 64 states (v_mfma_f32_32x32x16, fp32 sums):
//   S^T = K Q^T      states x rows: lane l owns row l % 32 and half of the states,
//   P^T = exp2(scale log2(e) S^T - m) in K's 16-bit type,
//   O^T += V^T P^T   the sums of the first product lie as the second one's operand does.
// P is rounded to K's type (bf16: half of 2^-8 a weight), its row sum adds the same rounded
// values, so that the weights add up to 1.
#include <algorithm>

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

constexpr int KT = 64;                  // states a tile

// In each group of 16 lanes, lane i gets, as element j, element i % 4 of the 8
// bytes that lane 4 j + i / 4 addresses: with lane s at row r0 + s / 4, columns c0 +
// 4 (s % 4) .. + 3, lane i receives rows r0 .. r0 + 3 of column c0 + i
__device__ __forceinline__ s16x4 read_turned(const uint16_t *p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *) (p)); }

template <bool BF16> struct Half;
template <> struct Half<true> {
    typedef bf16x8 x8;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint16_t bits(float f) { return f32_to_bf16_bits(f); }
    static __device__ __forceinline__ float sum2(x8 p, int i, float s) {
        const bf16x2 v = {p[i], p[i + 1]}, one = {(__bf16) 1.0f, (__bf16) 1.0f};
        return __builtin_amdgcn_fdot2_f32_bf16(v, one, s, false);
    }
    static __device__ __forceinline__ void set(x8 &p, int i, float f) { p[i] = (__bf16) f; }
};
template <> struct Half<false> {
    typedef f16x8 x8;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ uint16_t bits(float f) { return f32_to_f16_bits(f); }
    static __device__ __forceinline__ float sum2(x8 p, int i, float s) {
        const f16x2 v = {p[i], p[i + 1]}, one = {(_Float16) 1.0f, (_Float16) 1.0f};
        return __builtin_amdgcn_fdot2(v, one, s, false);
    }
    static __device__ __forceinline__ void set(x8 &p, int i, float f) { p[i] = (_Float16) f; }
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
    for (int i = 0; i < 4; ++i) o[i] = Half<BF16>::bits(f[2 * i]) | (uint32_t) Half<BF16>::bits(f[2 * i + 1]) << 16;
    return o;
}

// DP: the head size rounded up to 64 or 128; the values past it are zeros
template <int DP, bool BF16>
__global__ __launch_bounds__(256) void cross_attn_kernel(const CrossAttn p, int qtiles) {
    typedef Half<BF16> T;
    typedef typename T::x8 x8;
    constexpr int CH = DP / 8, RL = 64 / CH, NL = KT / RL, TILE = KT * DP;     // 16-byte pieces a row, rows and loads of 1 KB
    constexpr int FAR = (int) 0x80000000u;
    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];           // [2][K tile, V tile]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int qt = (int) (blockIdx.x % qtiles), hk = (int) (blockIdx.x / qtiles % p.Hkv), b = (int) (blockIdx.x / qtiles / p.Hkv);
    const int G = p.H / p.Hkv;
    const int64_t R = (int64_t) G * p.Nq;
    const int nkv = p.kv_len ? max(0, min(p.kv_len[b], p.Nkv)) : p.Nkv;
    const int nq = p.q_len ? max(0, min(p.q_len[b], p.Nq)) : p.Nq;
    const int64_t r0 = (int64_t) qt * 128 + wave * 32;
    if (nq == 0 || (G == 1 && (int64_t) qt * 128 >= nq)) return;
    const int64_t row = std::min<int64_t>(r0 + l32, R - 1);
    const int h = hk * G + (int) (row / p.Nq), iq = (int) (row % p.Nq);

    const char *qrow = (const char *) p.q + iq * p.q_nb1 + h * p.q_nb2 + b * p.q_nb3;
    x8 q[DP / 16];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = 16 * ks + 8 * hi;
        const u32x4 zero = {0, 0, 0, 0};
        q[ks] = __builtin_bit_cast(x8, d < p.D ? load_q8<BF16>(qrow, d, p.q_type) : zero);
    }

    const char *kp = (const char *) p.k + hk * p.k_nb2 + b * p.k_nb3, *vp = (const char *) p.v + hk * p.v_nb2 + b * p.v_nb3;
    const uint8_t *flags = p.kv_valid ? p.kv_valid + b * p.kv_valid_nb : nullptr;
    // Piece c of row t of a tile lies at slot c ^ key(t). K: 16 lanes of a 16-byte read take one piece
    // of 16 rows: keys that send them to 16 places; V: the four rows of a transposing read
    const int lr = lane / CH;
    const int kc = (lane % CH) ^ (DP == 128 ? 4 * (wave & 3) + (lane >> 4) : (4 * (wave & 1) + (lane >> 4)) & 7);
    const int vc = (lane % CH) ^ (DP == 128 ? 4 * (lr & 3) : 2 * (lr & 3));
    const int koff = kc * 8 < p.D ? (int) (lr * p.k_nb1) + kc * 16 : FAR, voff = vc * 8 < p.D ? (int) (lr * p.v_nb1) + vc * 16 : FAR;
    auto issue = [&](int tile, int buf) {
        uint16_t *dst = lds + buf * 2 * TILE;
        const int left = min(KT, nkv - tile * KT);
        const int64_t k0 = (int64_t) tile * KT;
        // rows past the last state that counts read as zeros
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void *) (kp + k0 * p.k_nb1), (short) 0,
                                                                            (int) ((left - 1) * p.k_nb1) + 2 * p.D, 0x00020000);
        const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void *) (vp + k0 * p.v_nb1), (short) 0,
                                                                            (int) ((left - 1) * p.v_nb1) + 2 * p.D, 0x00020000);
#pragma unroll
        for (int i = 0; i < NL / 4; ++i) {
            const int j = wave + 4 * i;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void *) (dst + j * 512), 16, koff, (int) (j * RL * p.k_nb1), 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void *) (dst + TILE + j * 512), 16, voff, (int) (j * RL * p.v_nb1), 0, 0);
        }
    };
    // bit s: state s of the tile counts
    auto counted = [&](int tile) -> uint64_t {
        const int left = nkv - tile * KT;
        uint64_t m = left >= KT ? ~(uint64_t) 0 : ((uint64_t) 1 << left) - 1;
        if (flags) m &= __ballot(lane < left && flags[(int64_t) tile * KT + lane]);
        return m;
    };

    f32x16 o[DP / 32];
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[db][e] = 0.0f;
    float m_run = -__builtin_inff(), l_run = 0.0f;
    const float c = p.c;
    const int l16 = lane & 15, grp = (lane >> 4) & 1, vrow = 4 * hi + (l16 >> 2), vkey = (DP == 128 ? 4 : 2) * (l16 >> 2);
    const int tiles = (nkv + KT - 1) / KT;
    if (tiles) issue(0, 0);
    for (int t = 0; t < tiles; ++t) {
        const uint64_t count = counted(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                                     // tile t is in LDS, every wave is done with the one before
        if (t + 1 < tiles) issue(t + 1, (t + 1) & 1);
        const uint16_t *kb = lds + (t & 1) * 2 * TILE, *vb = kb + TILE;
        if (count == 0) continue;
        const bool some = count != ~(uint64_t) 0;
        if (some && flags) {
            // a state that does not count may hold anything: 0 times it may not be 0
            const int s = tid >> 2;
            if (!(count >> s & 1))
                for (int i = 0; i < DP / 32; ++i) *(u32x4 *) (lds + (t & 1) * 2 * TILE + TILE + s * DP + (tid & 3) * (DP / 4) + i * 8) = u32x4{0, 0, 0, 0};
            __syncthreads();
        }
        f32x16 s[2];
#pragma unroll
        for (int kb2 = 0; kb2 < 2; ++kb2) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kb2][e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                const int r = 32 * kb2 + l32, key = DP == 128 ? r & 15 : (r >> 1) & 7;
                const x8 a = *(const x8 *) (kb + r * DP + (((2 * ks + hi) ^ key) << 3));
                s[kb2] = T::mfma(a, q[ks], s[kb2]);
            }
        }
        if (some) {
            const uint64_t mine = count >> 4 * hi;
#pragma unroll
            for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!(mine >> (32 * kb2 + 8 * (e >> 2) + (e & 3)) & 1)) s[kb2][e] = -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[0][e]);
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[1][e]);
        const float m_new = fmaxf(m_run, half_pair_max(top) * c);
        const float sub = m_new == -__builtin_inff() ? 0.0f : m_new, alpha = __builtin_amdgcn_exp2f(m_run - sub);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
        x8 pf[4];
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) {
#pragma unroll
            for (int e = 0; e < 8; ++e) T::set(pf[kg], e, __builtin_amdgcn_exp2f(__builtin_fmaf(s[kg >> 1][8 * (kg & 1) + e], c, -sub)));
#pragma unroll
            for (int e = 0; e < 8; e += 2) l_run = T::sum2(pf[kg], e, l_run);
        }
#pragma unroll
        for (int kg = 0; kg < 4; ++kg)
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
                const int ch = 4 * db + 2 * grp + ((l16 & 3) >> 1);
                const uint16_t *at = vb + (16 * kg + vrow) * DP + ((ch ^ vkey) << 3) + 4 * (l16 & 1);
                const s16x4 a = read_turned(at), a2 = read_turned(at + 8 * DP);
                const s16x8 a8 = {a[0], a[1], a[2], a[3], a2[0], a2[1], a2[2], a2[3]};
                o[db] = T::mfma(__builtin_bit_cast(x8, a8), pf[kg], o[db]);
            }
    }
    const float l = half_pair_sum(l_run), inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;   // (a NaN stays)
    if (r0 + l32 >= R || iq >= nq) return;
    char *orow = (char *) p.o + h * p.o_nb1 + iq * p.o_nb2 + b * p.o_nb3;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * db + 2 * e + 4 * hi;
            if (d >= p.D) continue;
            const float v[4] = {o[db][e] * inv, o[db][e + 1] * inv, o[db][e + 2] * inv, o[db][e + 3] * inv};
            if (p.o_type == TSK_TYPE_F32) {
                *(f32x4 *) (orow + d * 4) = f32x4{v[0], v[1], v[2], v[3]};
            } else if (p.o_type == TSK_TYPE_BF16) {
                *(u32x2 *) (orow + d * 2) = u32x2{f32_to_bf16_bits(v[0]) | (uint32_t) f32_to_bf16_bits(v[1]) << 16,
                                                 f32_to_bf16_bits(v[2]) | (uint32_t) f32_to_bf16_bits(v[3]) << 16};
            } else {
                *(u32x2 *) (orow + d * 2) = u32x2{f32_to_f16_bits(v[0]) | (uint32_t) f32_to_f16_bits(v[1]) << 16,
                                                 f32_to_f16_bits(v[2]) | (uint32_t) f32_to_f16_bits(v[3]) << 16};
            }
        }
}

template <int DP, bool BF16>
hipError_t launch_dp(const CrossAttn &p, hipStream_t s) {
    const int64_t R = (int64_t) (p.H / p.Hkv) * p.Nq, qtiles = (R + 127) / 128, units = qtiles * p.Hkv * p.B;
    constexpr size_t LDS = 2 * 2 * KT * DP * 2;
    if (units * 256 >= (int64_t) 1 << 32 || units > 0x7fffffff) return hipErrorInvalidValue;
    lds_opt_in((const void *) cross_attn_kernel<DP, BF16>, LDS);
    launch_kernel(cross_attn_kernel<DP, BF16>, dim3((unsigned) units), dim3(256), LDS, s, p, (int) qtiles);
    return hipGetLastError();
}

}  // namespace

int cross_attn_splits(int D, int64_t Nq, int64_t Nkv, int64_t H, int64_t Hkv, int64_t B, size_t *bytes) {
    *bytes = 0;
    return 1;
}

hipError_t launch_cross_attn(const CrossAttn &p, hipStream_t s) {
    if (p.D <= 64) return p.kv_bf16 ? launch_dp<64, true>(p, s) : launch_dp<64, false>(p, s);
    return p.kv_bf16 ? launch_dp<128, true>(p, s) : launch_dp<128, false>(p, s);
}

}  // namespace tsk
