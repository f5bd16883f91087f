// Differential attention (gfx950): two softmax maps of one head, their difference times the values.
//   A_i = softmax(q_i k_i^T / 8 + mask), i = 1, 2 (64 channels each);   O = A_1 V - lambda A_2 V  (V 128 channels)
//   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init;   with gamma: O <- O * gamma (1 - lambda_init) / sqrt(mean(O^2) + eps) over the head's 128 channels.
// Query i of sequence b sees keys j < k_len[b] and, causal, j <= q_start[b] + i.  A query that sees no key gives zeros.
//
// Both maps share one pass over keys and values: running maximum and sum per map and query, two accumulators.
//   S_i^T[key][query] = K_i Q_i^T      a lane owns ONE query (column lane % 32) and 16 of a 32-key tile's keys: the softmax is lane-local plus one exchange
//                                      between the halves of the wave;
//   O_i^T[channel][query] += V^T P_i^T  the accumulator registers 8 s .. 8 s + 7 of S_i^T are the B operand of step s as they stand, if the A operand holds
//                                      the same keys in the same order: half h holds keys 16 s + 4 h + (0..3) and 16 s + 8 + 4 h + (0..3).
// P is rounded to the 16-bit type for the matrix cores (at most half a step of the type relative to each weight, or in fp16 2^-32 of the row's largest); scores, maxima, sums and both accumulators
// are fp32, and the row sums add the unrounded weights.  The maps' difference makes these roundings weigh more than the result's own (lambda 0.8, scores of
// deviation 1: together 1.6 roundings of the result in the 2-norm), so what map 1's weights lose is rounded once more and multiplied as well: for all keys where the keys
// and values are what takes the time (1.1 to 1.2 roundings), for 16 of 32 where the products are (1.45 at most; none, half, all of them: 727, 804, 896 us for 2 x 9216 tokens when it was measured).
// The heads of a group that share a key / value head are rows of one product: row r = query * group + head, so a causal tile of rows spans few queries.
#include "svd_common.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr int PART = 260;                      // floats of one row's share: two accumulators, maximum and sum of each map
constexpr float C_EXP = 0.125f * LOG2E;        // score scale and base 2 in one factor
constexpr float M_NONE = -3.0e38f;            // running maximum before the first visible key: finite, so that no -inf - -inf appears

struct DiffArgs {
    const svd_bf16* Q; int64_t q_sb, q_st, q_sh;
    const svd_bf16* K; int64_t k_sb, k_st, k_sh;
    const svd_bf16* V; int64_t v_sb, v_st, v_sh;
    svd_bf16* O; int64_t o_sb, o_st, o_sh;
    const float* lam; float lambda_init;
    const float* gamma; float eps;
    const int32_t* k_len; const int32_t* q_start;
    int n_q, n_k, kv_heads, group, causal;
};

__device__ __forceinline__ float diff_lambda(const float* lam, float lambda_init, int lane) {
    const float d1 = wave_sum(lam[lane] * lam[64 + lane]), d2 = wave_sum(lam[128 + lane] * lam[192 + lane]);
    return expf(d1) - expf(d2) + lambda_init;
}

// the factor of the head's norm; zeros stay zeros with eps = 0 too
__device__ __forceinline__ float diff_norm(float square_sum, const DiffArgs& p, float eps) {
    const float d = square_sum * (1.f / 128.f) + eps;
    return d == 0.f ? 0.f : (1.f - p.lambda_init) / sqrtf(d);
}

// `num` over a map's sum of weights.  A sum of 0 is that of a query that sees no key, whose result is zeros -- or of one whose scores are all -inf: they
// have no softmax, and the result is NaN.  (The largest finite score has a weight of 1 or more.)
__device__ __forceinline__ float diff_over(float num, float sum, int seen) { return sum == 0.f ? (seen > 0 ? NAN : 0.f) : num / sum; }

// keys of sequence b, in [0, n_k] whatever the lengths' tensor holds
__device__ __forceinline__ int key_count(const DiffArgs& p, int b) { return p.k_len ? max(0, min(p.k_len[b], p.n_k)) : p.n_k; }
// number of keys query q sees
__device__ __forceinline__ int seen_by(const DiffArgs& p, int b, int len, int q) {
    if (!p.causal) return len;
    const int64_t end = (int64_t)(p.q_start ? p.q_start[b] : len - p.n_q) + q + 1;
    return (int)max((int64_t)0, min((int64_t)len, end));
}

// What a query does not see must not reach it, and a weight of 0 is no help against an Inf or NaN in V: 0 * NaN is NaN.  In a tile that some of the block's
// queries see further into than others (where all see the same keys, hidden places hold the last of them again), non-finite values are looked for; if there are any, the block starts over in a form that multiplies with V with zeros in
// their places, and counts with a second product -- of the places with the 0 / 1 mask -- the non-finite values that each (channel, query) does see: those
// results become NaN (what p * NaN, and inf - lambda inf, come to).  Starting over keeps the rare form's registers out of the loop that always runs.
template <class E> struct NonFinite {
    static constexpr uint32_t EXP = E::kId == SVD_DTYPE_F16 ? 0x7C00u : 0x7F80u, ONE = E::kId == SVD_DTYPE_F16 ? 0x3C00u : 0x3F80u;
    static __device__ __forceinline__ bool any(uint4 w) { return bad(w.x) | bad(w.y) | bad(w.z) | bad(w.w); }
    static __device__ __forceinline__ bool bad(uint32_t w) { return (w & EXP) == EXP || (w & (EXP << 16)) == (EXP << 16); }
    static __device__ __forceinline__ uint32_t places(uint32_t w) {
        return ((w & EXP) == EXP ? ONE : 0u) | ((w & (EXP << 16)) == (EXP << 16) ? ONE << 16 : 0u);
    }
    static __device__ __forceinline__ uint32_t cleared(uint32_t w) {
        return w & (((w & EXP) == EXP ? 0u : 0xffffu) | ((w & (EXP << 16)) == (EXP << 16) ? 0u : 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 places(uint4 w) { return make_uint4(places(w.x), places(w.y), places(w.z), places(w.w)); }
    static __device__ __forceinline__ uint4 cleared(uint4 w) { return make_uint4(cleared(w.x), cleared(w.y), cleared(w.z), cleared(w.w)); }
};

// ---- LDS tiles: KT keys of 256 bytes (k1 | k2, or v), 16-byte slots swizzled by the key, written by LDS-DMA (4 rows per instruction, lane = row * 16 + slot) ----
//   K: slot ^ (key & 15): 16 lanes that read one slot of 16 different keys (ds_read_b128, A operand: lane = key) touch all 64 banks once;
//   V: slot ^ (4 (key & 3)): a transposing read takes 4 keys x 16 channels per 16 lanes; 32 lanes touch 4 keys x 2 x 32 bytes, all 64 banks once.
constexpr int ROW_B = 256;
constexpr int Q_B = 3 * 64 * 16;          // three query fragments of a wave
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// maximum over the two halves of the wave, in both
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Q_LDS: three of map 2's four query fragments wait in the wave's 3 KiB of LDS instead of 12 registers
template <class E, bool Q_LDS = false> struct DiffWave {
    static constexpr int RESTS = Q_LDS ? 1 : 2;          // 16-key halves of a step whose weights' rests are multiplied
    static constexpr float LIFT = E::kId == SVD_DTYPE_F16 ? 7.f : 0.f;          // see follow
    uint4 qf[8];
    uint4* q_lds;
    f32x16_t o[2][4], s[2];
    uint32_t pk[2][8], rest[4 * RESTS];        // weights in 16 bits; what map 1's lost
    float m[2], l[2];                  // exponent that the weights are taken against, and their sum
    int l31, hi, seen, first;          // keys that this lane's query sees; the fewest that any query of the wave sees
    bool uneven;                       // some query sees less than what is staged: places behind the staged keys repeat the last, which all others see
    bool bad;                          // a value that is not finite in a tile with hidden places
    uint32_t ka, va;                   // byte offsets of the lane's first K and V^T fragment in a 32-key tile; the others differ in bits 5..7 (K) and 6, 7 (V)

    __device__ __forceinline__ void init(const svd_bf16* Qr, int lane, uint4* wave_lds = nullptr) {
        q_lds = wave_lds + lane;
        l31 = lane & 31; hi = lane >> 5; bad = false;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const uint4 f = *(const uint4*)(Qr + 64 * i + 16 * s + 8 * hi);
                if (Q_LDS && i == 1 && s < 3) q_lds[s * 64] = f;
                else qf[4 * i + s] = f;
            }
        ka = l31 * ROW_B + ((hi ^ (l31 & 15)) << 4);
        const int i16 = lane & 15, g = (lane >> 4) & 1;
        va = (4 * hi + (i16 >> 2)) * ROW_B + (((2 * g + ((i16 & 3) >> 1)) ^ ((i16 >> 2) << 2)) << 4) + (i16 & 1) * 8;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            m[i] = M_NONE; l[i] = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][t][r] = 0.f;
        }
    }
    static __device__ __forceinline__ uint4 k_frag(uint32_t addr) {
        return __builtin_bit_cast(uint4, *(const __attribute__((address_space(3))) u32x4_t*)addr);
    }
    // 8 keys of one channel: 16 s + 4 h + (0..3) and 8 further on
    static __device__ __forceinline__ uint4 v_frag(uint32_t addr) {
        typedef __attribute__((address_space(3))) s16x4_t lds_t;
        const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)addr));
        const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(addr + 8 * ROW_B)));
        return make_uint4(a.x, a.y, b.x, b.y);
    }
    __device__ __forceinline__ uint4 q_frag(int i, int ks) const {
        return Q_LDS && i == 1 && ks < 3 ? q_lds[ks * 64] : qf[4 * i + ks];
    }
    // ---- the parts of a step of 32 keys, per map ----
    // S_i^T = K_i Q_i^T, K rows at LDS address sK
    __device__ __forceinline__ void scores(int i, uint32_t sK) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) s[i] = E::mfma(k_frag((sK + ka) ^ ((4 * i + ks) << 5)), q_frag(i, ks), s[i]);
    }
    __device__ __forceinline__ void hide(int i, int k0) {
        asm volatile("");          // a branch, not 16 selections in every step
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = k0 + 8 * (r >> 2) + 4 * hi + (r & 3) >= seen ? -INFINITY : s[i][r];
    }
    __device__ __forceinline__ float top(int i) {          // the query's largest score of the step, times c
        float mx = fmaxf(s[i][0], s[i][1]);
#pragma unroll
        for (int r = 2; r < 16; ++r) mx = fmaxf(mx, s[i][r]);
        return halves_max(mx) * C_EXP;
    }
    // m is the exponent that the weights are taken against.  It is only there to keep them in range: it follows when some query of the wave has a score 2^8 beyond
    // what m last came from (weights that much larger are as exact as others), not at every new maximum, of which 64 rows have one in almost every tile of the first
    // 2000 keys.  64 multiplications each time.  fp16 weights stand 2^LIFT higher, between 2^7 and 2^15 for a row's largest: what fp16 (at most 65504) has no number for
    // begins at 2^-25, so beside a weight of 1 it would drop all below 2^-25 from the products and not from the sum (up to n_k 2^-25 of the largest value: 1e-3 at
    // 32768 keys), and so only what is below 2^-32.  Sums and accumulators are as much larger, and every join takes them relative to their m.
    __device__ __forceinline__ void follow(int i, float mx) {
        if (__builtin_expect_with_probability(__builtin_amdgcn_ballot_w64(mx > m[i] + (8.f + LIFT)) != 0, 0, 0.999)) {
            const float m_new = fmaxf(m[i], mx - LIFT), alpha = __builtin_amdgcn_exp2f(m[i] - m_new);
            m[i] = m_new;
            l[i] *= alpha;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][t][r] *= alpha;
        }
    }
    // weights of scores 2 e and 2 e + 1
    __device__ __forceinline__ void weigh(int i, int e) {
        weights(i, e, __builtin_amdgcn_exp2f(fmaf(s[i][2 * e], C_EXP, -m[i])), __builtin_amdgcn_exp2f(fmaf(s[i][2 * e + 1], C_EXP, -m[i])));
    }
    __device__ __forceinline__ void weights(int i, int e, float p0, float p1) {
        l[i] += p0 + p1;
        pk[i][e] = E::pack(p0, p1);
        if (i == 0 && e < 4 * RESTS) rest[e] = E::pack(fmaf(E::lo(pk[i][e]), -1.f, p0), fmaf(E::hi(pk[i][e]), -1.f, p1));
    }
    __device__ __forceinline__ uint4 p_frag(int i, int q) const { return make_uint4(pk[i][4 * q], pk[i][4 * q + 1], pk[i][4 * q + 2], pk[i][4 * q + 3]); }
    __device__ __forceinline__ uint4 r_frag(int q) const { return make_uint4(rest[4 * q], rest[4 * q + 1], rest[4 * q + 2], rest[4 * q + 3]); }
    // o_i^T += V^T P_i^T for 16 keys and 32 channels
    __device__ __forceinline__ void add(int i, int q, int t, uint4 vf) {
        o[i][t] = E::mfma(vf, p_frag(i, q), o[i][t]);
        if (i == 0 && q < RESTS) o[i][t] = E::mfma(vf, r_frag(q), o[i][t]);
    }
    __device__ __forceinline__ void values(int i, int q, int t, uint32_t sV) { add(i, q, t, v_frag(((sV + va) ^ (t << 6)) + q * 16 * ROW_B)); }
    __device__ __forceinline__ void look_for_bad(uint32_t sV) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int t = 0; t < 4; ++t) bad |= NonFinite<E>::any(v_frag(((sV + va) ^ (t << 6)) + q * 16 * ROW_B));
        asm volatile("" ::: "memory");          // the fragments are read again for the products: 64 registers less
    }
    // a step of 32 keys from k0 on as one piece
    template <bool CLEAR> __device__ __forceinline__ void tile(uint32_t sK, uint32_t sV, int k0) {
        const bool partial = k0 + 32 > first;          // some query of the wave does not see all of the tile
        scores(0, sK);
        scores(1, sK);
        if (partial) { hide(0, k0); hide(1, k0); }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            follow(i, top(i));
#pragma unroll
            for (int e = 0; e < 8; ++e) weigh(i, e);
        }
        if constexpr (!CLEAR) {
            if (partial && uneven) look_for_bad(sV);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint4 vf = v_frag(((sV + va) ^ (t << 6)) + q * 16 * ROW_B);
#pragma unroll
                    for (int i = 0; i < 2; ++i) add(i, q, t, vf);
                }
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f32x16_t hit;
#pragma unroll
                for (int r = 0; r < 16; ++r) hit[r] = 0.f;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint4 vf = v_frag(((sV + va) ^ (t << 6)) + q * 16 * ROW_B);
                    uint32_t see[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = k0 + 16 * q + 8 * (j >> 1) + 4 * hi + 2 * (j & 1);
                        see[j] = (key < seen ? NonFinite<E>::ONE : 0u) | (key + 1 < seen ? NonFinite<E>::ONE << 16 : 0u);
                    }
                    hit = E::mfma(NonFinite<E>::places(vf), make_uint4(see[0], see[1], see[2], see[3]), hit);
#pragma unroll
                    for (int i = 0; i < 2; ++i) add(i, q, t, NonFinite<E>::cleared(vf));
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) o[0][t][r] = hit[r] > 0.f ? NAN : o[0][t][r];
            }
        }
    }
    // Half of a step, pipelined: the weights of map i for the step at k0 (its scores are in s[i]) on the vector unit, and at the same time on the matrix unit
    // the other map's scores from the K rows at sK and its products of weights that are there with the V rows at sV.
    __device__ __forceinline__ void half(int i, int k0, uint32_t sK, uint32_t sV) {
        if (__builtin_expect_with_probability(k0 + 32 > first, 0, 0.99)) hide(i, k0);
        auto vf = [&](int e) { return v_frag(((sV + va) ^ ((e & 3) << 6)) + (e >> 2) * 16 * ROW_B); };
        auto kf = [&](int ks) { return k_frag((sK + ka) ^ ((4 * (1 - i) + ks) << 5)); };
        uint4 k[2], x[2], v[4];
        k[0] = kf(0); x[0] = q_frag(1 - i, 0);
        v[0] = vf(0); v[1] = vf(1);
        const float mx = top(i);
        k[1] = kf(1); x[1] = q_frag(1 - i, 1);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[1 - i][r] = 0.f;
        s[1 - i] = E::mfma(k[0], x[0], s[1 - i]);
        follow(i, mx);
        // A matrix instruction keeps its unit for 32 cycles and the wave, if the next one follows at once, waiting as long: two of them stand around half of the vector
        // instructions of two weights each.  The four score products are a chain on one accumulator and lie apart, and so do a product and its rest's.
        auto score = [&](int ks) { s[1 - i] = E::mfma(k[ks & 1], x[ks & 1], s[1 - i]); };
        constexpr int AT2[2] = {2, 5}, AT3[2] = {4, 6};          // where the third and fourth stand: map 1's half has the rests' products in between
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e + 2 < 8) v[(e + 2) % 4] = vf(e + 2);
            if (e == 0) { k[0] = kf(2); x[0] = q_frag(1 - i, 2); }
            if (e == 1) { k[1] = kf(3); x[1] = q_frag(1 - i, 3); }
            o[1 - i][e & 3] = E::mfma(v[e % 4], p_frag(1 - i, e >> 2), o[1 - i][e & 3]);
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i][2 * e], C_EXP, -m[i])), t1 = fmaf(s[i][2 * e + 1], C_EXP, -m[i]);
            __builtin_amdgcn_sched_barrier(0);
            if (e == 0) score(1);
            if (e == AT2[i]) score(2);
            if (e == AT3[i]) score(3);
            if (1 - i == 0 && e > 0 && e <= 4 * RESTS) o[0][(e - 1) & 3] = E::mfma(v[(e - 1) % 4], r_frag((e - 1) >> 2), o[0][(e - 1) & 3]);
            weights(i, e, p0, __builtin_amdgcn_exp2f(t1));
            if (i == 0 && e < 4 * RESTS) asm volatile("" : "+v"(rest[e]));
            asm volatile("" : "+v"(pk[i][e]), "+v"(l[i]));          // made here, not where the next half needs it
            __builtin_amdgcn_sched_barrier(0);                      // the reads stay where they are: two products ahead of their use
        }
    }
    __device__ __forceinline__ void join_halves() {
#pragma unroll
        for (int i = 0; i < 2; ++i) l[i] += __shfl_xor(l[i], 32, 64);
    }
    // (A_1 - lambda A_2) V, the head's norm, one rounding.  A lane holds 64 channels of one row in pieces of four: the rows go through 8 KiB of the wave's LDS (slots
    // swizzled by the row) and leave as whole rows, four to an instruction.
    __device__ __forceinline__ void finish(const DiffArgs& p, int b, int h, int row0, int rows, uint32_t buf, int lane, float lam) {
        join_halves();
        const float w0 = diff_over(1.f, l[0], seen), w1 = diff_over(lam, l[1], seen);
        float ss = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                o[0][t][r] = o[0][t][r] * w0 - o[1][t][r] * w1;
                ss = fmaf(o[0][t][r], o[0][t][r], ss);
            }
        // gamma is requested here, in front of the branch: behind it every piece would wait for its own (25 frames: 176 us, 128 like this)
        float g[64];
        if (p.gamma) {
#pragma unroll
            for (int e = 0; e < 64; ++e) g[e] = p.gamma[8 * (e >> 2) + 4 * hi + (e & 3)];
        } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) g[e] = 1.f;
        }
        ss += __shfl_xor(ss, 32, 64);
        const float f = p.gamma ? svd_rms_factor(ss, p.eps) : 1.f;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(f != 1.f) != 0, 0)) {          // (others' values times 1, the same sum again)
            ss = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    o[0][t][r] *= f;
                    ss = fmaf(o[0][t][r], o[0][t][r], ss);
                }
            ss += __shfl_xor(ss, 32, 64);
        }
        const float norm = p.gamma ? diff_norm(ss, p, p.eps * f * f) : 1.f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = 32 * t + 2 * r + 4 * hi;
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = o[0][t][r + j] * (norm * g[16 * t + r + j]);
                typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
                const u32x2_t v = {E::pack(y[0], y[1]), E::pack(y[2], y[3])};
                *(__attribute__((address_space(3))) u32x2_t*)(buf + l31 * ROW_B + (((d >> 3) ^ (l31 & 15)) << 4) + (d & 4) * 2) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const int r = j + (lane >> 4), row = row0 + r;
            const uint4 v = k_frag(buf + r * ROW_B + (((lane & 15) ^ (r & 15)) << 4));
            if (row < rows) {
                const int q = p.group == 1 ? row : row / p.group;
                *(uint4*)(p.O + b * p.o_sb + q * p.o_st + (h * p.group + row - q * p.group) * p.o_sh + (lane & 15) * 8) = v;
            }
        }
    }
};

// Many queries: a workgroup of four waves holds 4 x 32 rows and walks the keys in steps of 32, staged once for all four.
// A step's exponentials keep the vector unit busy for longer (2 x 16 exponentials of 16 cycles and 118 other instructions a lane, 1000 cycles) than its products the
// matrix unit (24 instructions of 32 cycles), so the two have to run at once inside a wave.  The maps take turns: while map 1's weights of step j are made, the matrix unit
// does map 2's scores of step j and its products with V of step j - 1; while map 2's weights are made, map 1's scores of step j + 1 and its products with V of step j.
// So K is read a step ahead and V a step behind: rings of four 8-KiB slots each, requests two steps ahead, one barrier a step.
// 2 x 9216 tokens, 5 heads, fp16: 780 us (0.84 PFLOP/s of the one-pass work, 0.97 with the rests' products; the clock falls to 1.9 GHz under it; 720 workgroups on 512
// places leave the second round half empty).  Before the maps took turns: 828 us without the rests.  4 causal prompts of 1001 to 2001 tokens, 8 heads on 4: 80 us (104
// with long rows first everywhere).
template <class E> __global__ __launch_bounds__(256, 2) void attn_diff_rows_kernel(DiffArgs p, int row_blocks) {
    constexpr int SLOT_B = 32 * ROW_B, RING_B = 4 * SLOT_B;          // K ring, then V ring
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const uint32_t lds = lds_addr_of(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int wg;          // consecutive workgroups go round the 8 XCDs: give each XCD whole heads, whose keys and values stay in its L2
    {
        const int n = gridDim.x, x = blockIdx.x & 7, q = n >> 3, r = n & 7;
        wg = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (blockIdx.x >> 3);
    }
    // Causal rows differ in length.  Where all workgroups are on the chip at once (two to a CU), every other head runs from the short rows to the long ones, so that the two
    // of a CU are a long and a short one; else the long ones go first, for a short end.
    const int bh = wg / row_blocks, u = wg % row_blocks, h = bh % p.kv_heads, b = bh / p.kv_heads;
    const int rb = gridDim.x <= 512 && (bh & 1) ? u : row_blocks - 1 - u;
    const int rows = p.n_q * p.group, row0 = rb * 128 + wave * 32;
    const int rc = min(row0 + (lane & 31), rows - 1), q = rc / p.group, head = h * p.group + rc % p.group;
    const int len = key_count(p, b);
    const int last = seen_by(p, b, len, min(rows - 1, rb * 128 + 127) / p.group);                 // the workgroup's last row sees the most keys
    const int mine = row0 < rows ? seen_by(p, b, len, min(rows - 1, row0 + 31) / p.group) : 0;    // ... and the wave's
    DiffWave<E, true> w;
    w.init(p.Q + b * p.q_sb + q * p.q_st + head * p.q_sh, lane, (uint4*)(smem + 2 * RING_B + wave * Q_B));
    w.seen = seen_by(p, b, len, q);
    w.first = seen_by(p, b, len, min(rows - 1, row0) / p.group);
    w.uneven = w.first < last;
    const svd_bf16* Kb = p.K + b * p.k_sb + h * p.k_sh;
    const svd_bf16* Vb = p.V + b * p.v_sb + h * p.v_sh;
    // Requests: wave-uniform base in scalars, the lane's offset in 32 bits (32 rows of at most 2^26 bytes).  8 KiB by four waves: two instructions each.
    const int r0 = wave * 8 + (lane >> 4), c16 = lane & 15;
    const uint32_t k_row = (uint32_t)p.k_st * 2, v_row = (uint32_t)p.v_st * 2;
    uint32_t ko[2], vo[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        ko[u] = (r0 + 4 * u) * k_row + ((c16 ^ ((r0 + 4 * u) & 15)) << 4);
        vo[u] = (r0 + 4 * u) * v_row + ((c16 ^ ((r0 & 3) << 2)) << 4);
    }
    auto stage = [&](const svd_bf16* src, uint32_t row_b, const uint32_t* off, int j, uint32_t ring) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            uint32_t o = off[u];
            if (__builtin_expect_with_probability(j * 32 + 32 > last, 0, 0.99)) {          // rows behind the last visible key repeat it: they are masked, and hold nothing that is not seen
                const int row = r0 + 4 * u;
                o -= (row - min(row, last - 1 - j * 32)) * row_b;
            }
            glds16_saddr(o, src, __builtin_amdgcn_readfirstlane(ring + (j & 3) * SLOT_B + (wave * 8 + 4 * u) * ROW_B));
        }
    };
    auto stage_k = [&](int j) { stage(Kb + (int64_t)(j * 32) * p.k_st, k_row, ko, j, lds); };
    auto stage_v = [&](int j) { stage(Vb + (int64_t)(j * 32) * p.v_st, v_row, vo, j, lds + RING_B); };
    auto at_k = [&](int j) { return lds + (j & 3) * SLOT_B; };
    auto at_v = [&](int j) { return lds + RING_B + (j & 3) * SLOT_B; };
    const int steps = (last + 31) / 32, my_steps = (mine + 31) / 32;
    w.clear();
    if (steps > 0) {
        stage_k(0);
        if (steps > 1) stage_k(1);
        stage_v(0);
        if (steps > 2) { stage_k(2); stage_v(1); }
        else if (steps > 1) stage_v(1);
        svd_wait_dma();
        __syncthreads();
        w.scores(0, at_k(0));
#pragma unroll
        for (int e = 0; e < 8; ++e) w.pk[1][e] = 0;                       // no weights of step -1: nothing of V's first rows is added
        const svd_bf16* kp = Kb + (int64_t)96 * p.k_st;                   // the rows requested next: K of step j + 3, V of step j + 2
        const svd_bf16* vp = Vb + (int64_t)64 * p.v_st;
#pragma unroll 1
        for (int j = 0; j < steps; ++j) {
            // K of step j + 1 and V of step j: all but the last request, which is four instructions until the requests run out
            if (__builtin_expect_with_probability(j + 2 < steps, 1, 0.99)) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            else svd_wait_dma();
            __syncthreads();
            if (j + 3 < steps) stage(kp, k_row, ko, j + 3, lds);           // into the slots that step j - 1 was the last to read
            if (j + 2 < steps) stage(vp, v_row, vo, j + 2, lds + RING_B);
            kp += 32 * p.k_st; vp += 32 * p.v_st;
            if (j < my_steps) {
                if (__builtin_expect_with_probability(w.uneven && j * 32 + 32 > w.first, 0, 0.99)) w.look_for_bad(at_v(j));
                w.half(0, j * 32, at_k(j), at_v(j > 0 ? j - 1 : 0));
                w.half(1, j * 32, at_k(j + 1), at_v(j));
                if (__builtin_expect_with_probability(j == my_steps - 1, 0, 0.99)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w.values(1, e >> 2, e & 3, at_v(j));
                }
            }
        }
        if (__syncthreads_or(w.bad)) {          // once more, one step at a time, without what is not finite
            w.clear();
            for (int j = 0; j < steps; ++j) {
                stage_k(j);
                stage_v(j);
                svd_wait_dma();
                __syncthreads();
                if (j < my_steps) w.template tile<true>(at_k(j), at_v(j), j * 32);
                __syncthreads();
            }
        }
    }
    w.finish(p, b, h, row0, rows, lds + wave * SLOT_B, lane, diff_lambda(p.lam, p.lambda_init, lane));
}

// Few queries: one wave per (sequence, key / value head, 32 rows, share of the keys), no workgroup barrier; tiles of 32 keys, two in turn.  With one share
// the wave finishes the rows (2304 x 10 heads of 25 frames: 128 us, 4.6 TB/s; 16 KiB requested by each of 8 waves a CU); else it leaves maxima, sums and both accumulators in the scratch memory (fp32, [row][share][260]) for the join
// (8 caches of 16 to 32 k keys, 16 heads on 4: 90 us, 4.7 TB/s, and 5 for the join; one of 1025 keys, 8 heads: 6 and 3).
template <class E> __global__ __launch_bounds__(64, 2) void attn_diff_wave_kernel(DiffArgs p, int row_blocks, int shares, float* ws) {
    constexpr int KT = 32, TILE_B = KT * ROW_B, BUF_B = 2 * TILE_B;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const uint32_t lds = lds_addr_of(smem);
    const int lane = threadIdx.x;
    const int share = blockIdx.x % shares, u = blockIdx.x / shares, rb = u % row_blocks, bh = u / row_blocks, h = bh % p.kv_heads, b = bh / p.kv_heads;
    const int rows = p.n_q * p.group, row = rb * 32 + (lane & 31);
    const bool live = row < rows;
    const int rc = min(row, rows - 1), q = rc / p.group, head = h * p.group + rc % p.group;
    const int len = key_count(p, b);
    const int last = seen_by(p, b, len, min(rows - 1, rb * 32 + 31) / p.group);
    const int per = ((last + 31) / 32 + shares - 1) / shares * 32, begin = share * per, end = min(last, begin + per);      // shares of the keys there are, not of the capacity
    DiffWave<E> w;
    w.init(p.Q + b * p.q_sb + q * p.q_st + head * p.q_sh, lane);
    w.seen = seen_by(p, b, len, q);
    w.first = seen_by(p, b, len, rb * 32 / p.group);
    w.uneven = w.first < last;
    const svd_bf16* Kb = p.K + b * p.k_sb + h * p.k_sh;
    const svd_bf16* Vb = p.V + b * p.v_sb + h * p.v_sh;
    // requests as in the rows kernel; one wave requests all 8 + 8 KiB
    const int l4 = lane >> 4, c16 = lane & 15;
    const uint32_t k_row = (uint32_t)p.k_st * 2, v_row = (uint32_t)p.v_st * 2;
    auto stage = [&](int k0, int buf) {
        const svd_bf16 *ks = Kb + (int64_t)k0 * p.k_st, *vs = Vb + (int64_t)k0 * p.v_st;
        const int top = min(31, last - 1 - k0);                      // rows behind the last visible key repeat it: they are masked, and hold nothing that is not seen
#pragma unroll
        for (int r = 0; r < 32; r += 4) {
            const uint32_t dst = lds + buf * BUF_B + r * ROW_B, row = min(r + l4, top);
            glds16_saddr(row * k_row + ((c16 ^ l4 ^ (r & 12)) << 4), ks, dst);
            glds16_saddr(row * v_row + ((c16 ^ (l4 << 2)) << 4), vs, dst + TILE_B);
        }
    };
    if (begin < end) stage(begin, 0);
    // lambda while the first keys are on their way, not behind the last
    const float lam = shares == 1 ? __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, diff_lambda(p.lam, p.lambda_init, lane)))) : 0.f;
    auto walk = [&]<bool CLEAR>() {
        w.clear();
        if (CLEAR && begin < end) stage(begin, 0);
        int cur = 0;
        for (int k0 = begin; k0 < end; k0 += KT, cur ^= 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the reads of the tile that is overwritten next are done
            if (k0 + KT < end) {
                stage(k0 + KT, cur ^ 1);
                asm volatile("s_waitcnt vmcnt(16)" ::: "memory");         // all but the 16 just issued: this tile is there
            } else {
                svd_wait_dma();
            }
            w.template tile<CLEAR>(lds + cur * BUF_B, lds + cur * BUF_B + TILE_B, k0);
        }
    };
    walk.template operator()<false>();
    if (__builtin_amdgcn_ballot_w64(w.bad)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        walk.template operator()<true>();
    }
    if (shares == 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        w.finish(p, b, h, rb * 32, rows, lds, lane, lam);
        return;
    }
    w.join_halves();
    if (!live) return;
    float* part = ws + ((int64_t)(bh * rows + row) * shares + share) * PART;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 4) *(float4*)(part + 128 * i + 32 * t + 2 * r + 4 * w.hi) = make_float4(w.o[i][t][r], w.o[i][t][r + 1], w.o[i][t][r + 2], w.o[i][t][r + 3]);
    if (w.hi == 0) *(float4*)(part + 256) = make_float4(w.m[0], w.l[0], w.m[1], w.l[1]);
}

// Shares of a row's keys, joined one after the other: a lane holds two channels.
__device__ __forceinline__ float2 gamma_pair(const DiffArgs& p, int lane) { return p.gamma ? make_float2(p.gamma[2 * lane], p.gamma[2 * lane + 1]) : make_float2(1.f, 1.f); }
template <class E> struct Joined {
    float m[2] = {M_NONE, M_NONE}, l[2] = {0.f, 0.f}, o[2][2] = {};
    __device__ __forceinline__ void add(float4 ml, float2 x, float2 y) {          // maximum and sum of each map; the channels of each map's accumulator
        const float m0 = fmaxf(m[0], ml.x), m1 = fmaxf(m[1], ml.z);
        const float a0 = __builtin_amdgcn_exp2f(m[0] - m0), a1 = __builtin_amdgcn_exp2f(m[1] - m1), b0 = __builtin_amdgcn_exp2f(ml.x - m0), b1 = __builtin_amdgcn_exp2f(ml.z - m1);
        m[0] = m0; m[1] = m1;
        l[0] = fmaf(l[0], a0, ml.y * b0); l[1] = fmaf(l[1], a1, ml.w * b1);
        o[0][0] = fmaf(o[0][0], a0, x.x * b0); o[0][1] = fmaf(o[0][1], a0, x.y * b0);
        o[1][0] = fmaf(o[1][0], a1, y.x * b1); o[1][1] = fmaf(o[1][1], a1, y.y * b1);
    }
    // lam: diff_lambda, g: the lane's two channels of gamma, both requested before the wait for the shares
    __device__ __forceinline__ void finish(const DiffArgs& p, int b, int h, int row, int lane, float lam, float2 g) const {
        int seen = 0;
        if (l[0] == 0.f || l[1] == 0.f) seen = seen_by(p, b, key_count(p, b), row / p.group);
        const float w0 = diff_over(1.f, l[0], seen), w1 = diff_over(lam, l[1], seen);
        float y0 = o[0][0] * w0 - o[1][0] * w1, y1 = o[0][1] * w0 - o[1][1] * w1;
        if (p.gamma) {
            float ss = wave_sum(fmaf(y0, y0, y1 * y1));
            const float f = svd_rms_factor(ss, p.eps);          // the same in all lanes
            if (f != 1.f) {
                y0 *= f; y1 *= f;
                ss = wave_sum(fmaf(y0, y0, y1 * y1));
            }
            const float norm = diff_norm(ss, p, p.eps * f * f);
            y0 *= norm * g.x; y1 *= norm * g.y;
        }
        *(uint32_t*)(p.O + b * p.o_sb + (row / p.group) * p.o_st + (h * p.group + row % p.group) * p.o_sh + 2 * lane) = E::pack(y0, y1);
    }
};

// One workgroup per row: lane = two channels, the four waves take the shares in turn, four requested at once, and meet in LDS.  The order of the sums is fixed, so the result
// does not depend on which share finished first.  (One wave and one share at a time: 11.6 us for 128 rows of 32 shares, 7.8 for 8 of 17.)
template <class E> __global__ __launch_bounds__(256) void attn_diff_join_kernel(DiffArgs p, int shares, const float* ws) {
    __shared__ float4 s_ml[4];
    __shared__ float2 s_o[4][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rows = p.n_q * p.group, row = blockIdx.x % rows, bh = blockIdx.x / rows, h = bh % p.kv_heads, b = bh / p.kv_heads;
    const float* part = ws + (int64_t)blockIdx.x * shares * PART;
    const float lam = diff_lambda(p.lam, p.lambda_init, lane);
    const float2 g = gamma_pair(p, lane);
    Joined<E> sum;
    for (int s0 = wave; s0 < shares; s0 += 16) {
        float4 ml[4];
        float2 x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float* at = part + (int64_t)min(s0 + 4 * u, shares - 1) * PART;
            ml[u] = *(const float4*)(at + 256);
            x[u] = *(const float2*)(at + 2 * lane);
            y[u] = *(const float2*)(at + 128 + 2 * lane);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (s0 + 4 * u >= shares) break;
            sum.add(ml[u], x[u], y[u]);
        }
    }
    if (lane == 0) s_ml[wave] = make_float4(sum.m[0], sum.l[0], sum.m[1], sum.l[1]);
    s_o[wave][0][lane] = make_float2(sum.o[0][0], sum.o[0][1]); s_o[wave][1][lane] = make_float2(sum.o[1][0], sum.o[1][1]);
    __syncthreads();
    if (wave) return;
    Joined<E> all;
#pragma unroll
    for (int w = 0; w < 4; ++w) all.add(s_ml[w], s_o[w][0][lane], s_o[w][1][lane]);
    all.finish(p, b, h, row, lane, lam, g);
}

// A few rows and at most 256 keys: one workgroup per (sequence, key / value head), 32 keys to each of its eight waves, joined in LDS: one launch and no scratch memory.
// 8 heads, 100 / 256 keys: 6.4 / 7.8 us in a graph, 11.3 called one by one; shares and join 9.7 / 9.1 and 15.5.  It takes all 256 registers and spills 14 (60 bytes a lane).  (More keys, as a loop over tiles: 513 keys 11.6 against 9.7 us.)
constexpr int GROUP_WAVES = 8, GROUP_ROWS = 16, GROUP_KEYS = GROUP_WAVES * 32, GROUP_LDS = GROUP_WAVES * (64 * ROW_B + GROUP_ROWS * 16);
template <class E> __global__ __launch_bounds__(GROUP_WAVES * 64, 2) void attn_diff_group_kernel(DiffArgs p) {
    constexpr int TILE_B = 32 * ROW_B;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float4* s_ml = (float4*)(smem + GROUP_WAVES * 2 * TILE_B);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads, rows = p.n_q * p.group, row = lane & 31;
    const int rc = min(row, rows - 1), q = rc / p.group, head = h * p.group + rc % p.group;
    const int len = key_count(p, b), last = seen_by(p, b, len, p.n_q - 1), k0 = wave * 32;
    const uint32_t sK = lds_addr_of(smem) + wave * 2 * TILE_B, sV = sK + TILE_B;
    if (k0 < last) {          // requests as in the wave kernel; the keys, the values, the queries and lambda come in one wait
        const svd_bf16* ks = p.K + b * p.k_sb + h * p.k_sh + k0 * p.k_st;
        const svd_bf16* vs = p.V + b * p.v_sb + h * p.v_sh + k0 * p.v_st;
        const int l4 = lane >> 4, c16 = lane & 15, top = min(31, last - 1 - k0);
        const uint32_t k_row = (uint32_t)p.k_st * 2, v_row = (uint32_t)p.v_st * 2;
#pragma unroll
        for (int r = 0; r < 32; r += 4) {
            const uint32_t at = min(r + l4, top);
            glds16_saddr(at * k_row + ((c16 ^ l4 ^ (r & 12)) << 4), ks, sK + r * ROW_B);
            glds16_saddr(at * v_row + ((c16 ^ (l4 << 2)) << 4), vs, sV + r * ROW_B);
        }
    }
    DiffWave<E> w;
    w.init(p.Q + b * p.q_sb + q * p.q_st + head * p.q_sh, lane);
    w.seen = seen_by(p, b, len, q);
    w.first = seen_by(p, b, len, 0);
    w.uneven = w.first < last;
    const float lam = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, diff_lambda(p.lam, p.lambda_init, lane))));          // one register less
    w.clear();
    if (k0 < last) {
        svd_wait_dma();
        w.template tile<false>(sK, sV, k0);
        if (__builtin_amdgcn_ballot_w64(w.bad)) {
            w.clear();
            w.template tile<true>(sK, sV, k0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    const float2 g = gamma_pair(p, lane);
    w.join_halves();
    // 16 rows of 1 KiB in the wave's own tiles, pieces of 16 bytes swizzled by the row
    if (row < rows) {
        float4* part = (float4*)(smem + wave * 2 * TILE_B) + row * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    part[((128 * i + 32 * t + 2 * r + 4 * w.hi) >> 2) ^ row] = make_float4(w.o[i][t][r], w.o[i][t][r + 1], w.o[i][t][r + 2], w.o[i][t][r + 3]);
        if (w.hi == 0) s_ml[wave * GROUP_ROWS + row] = make_float4(w.m[0], w.l[0], w.m[1], w.l[1]);
    }
    __syncthreads();
    for (int r = wave; r < rows; r += GROUP_WAVES) {
        Joined<E> sum;
#pragma unroll
        for (int s = 0; s < GROUP_WAVES; ++s) {
            const float* part = (const float*)(smem + s * 2 * TILE_B) + r * 256 + (lane & 1) * 2;
            sum.add(s_ml[s * GROUP_ROWS + r], *(const float2*)(part + ((lane >> 1) ^ r) * 4), *(const float2*)(part + ((32 + (lane >> 1)) ^ r) * 4));
        }
        sum.finish(p, b, h, r, lane, lam, g);
    }
}

// Which form.  Both sides measured, us a call in a graph, fp16, 128 channels, all keys | causal:
//   many rows (128 to a workgroup, keys staged once for four waves) with more than 64 rows and 128 blocks of 128, else waves of 32 rows with the keys in shares: with fewer rows half
//     of a block's waves have none, with fewer blocks half of the CUs have none, and shares fill them.
//     64 rows, 2048 keys, 128 blocks (16 x 64 tokens, 8 heads): many-row form 67.6 | 69.7, waves 62.6 | 62.8; 65 rows: 68.1 | 70.7, 99.9 | 101; 128 rows 71.7 | 74.2, 106 | 106.
//     1 x 2000 tokens: 4 heads (64 blocks) 67.6 | 69.5, 67.8 | 50.3; 6 (96) 69.7 | 69.8, 95.8 | 67.2; 8 (128) 68.4 | 69.7, 107 | 79.5; 1 x 4096 tokens: 2 heads (64) 128 | 132, 84.0 | 70.7;
//     4 (128) 129 | 133, 148 | 128.  With few keys the border lies lower than the rule has it: 4 x 300 tokens, 8 heads (96 blocks) 17.7 | 19.8, 40.3 | 33.7.
//   one workgroup for up to 16 rows on up to 256 keys: see attn_diff_group_kernel.
enum { ROWS, WAVES, GROUP };
struct Plan { int form, row_blocks, shares; int64_t ws; };
Plan plan_for(int64_t batch, int64_t n_q, int64_t n_k, int64_t heads, int64_t kv_heads) {
    const int64_t rows = n_q * (heads / kv_heads), bh = batch * kv_heads;
    Plan r = {WAVES, (int)((rows + 31) / 32), 1, 0};
    if (rows > 64 && (rows + 127) / 128 * bh >= 128) return {ROWS, (int)((rows + 127) / 128), 1, 0};
    const int64_t units = r.row_blocks * bh;
    if (units > 0) {
        int64_t shares = (1024 + units - 1) / units;          // four waves on each CU (8 caches of 16-32k keys: 100 us with 640 to 1280 waves, 105 with 2048, 130 with 4096)
        if (shares > (n_k + 63) / 64) shares = (n_k + 63) / 64;
        // one launch where the keys fit one workgroup and there is a CU for each
        if (shares > 1 && rows <= GROUP_ROWS && bh <= 256 && n_k <= GROUP_KEYS) return {GROUP, 1, 1, 0};
        if (shares > 1) { r.shares = (int)shares; r.ws = rows * bh * shares * PART * 4; }
    }
    return r;
}

}  // namespace

extern "C" int64_t svd_attn_diff_ws_bytes(int32_t batch, int32_t n_q, int32_t n_k, int32_t heads, int32_t kv_heads) {
    if (batch < 0 || n_q < 0 || n_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return SVD_EINVAL;
    return plan_for(batch, n_q, n_k, heads, kv_heads).ws;
}

extern "C" int svd_attn_diff(const svd_bf16* Q, int64_t q_sb, int64_t q_st, int64_t q_sh, const svd_bf16* K, int64_t k_sb, int64_t k_st, int64_t k_sh,
                             const svd_bf16* V, int64_t v_sb, int64_t v_st, int64_t v_sh, svd_bf16* O, int64_t o_sb, int64_t o_st, int64_t o_sh,
                             const float* lam, float lambda_init, const float* gamma, float eps, const int32_t* k_len, const int32_t* q_start,
                             int32_t batch, int32_t n_q, int32_t n_k, int32_t heads, int32_t kv_heads, int32_t causal, void* ws, int64_t ws_bytes,
                             int32_t dtype, svd_stream_t stream) {
    if (batch < 0 || n_q < 0 || n_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return SVD_EINVAL;
    const Plan plan = plan_for(batch, n_q, n_k, heads, kv_heads);
    if (ws_bytes < plan.ws || (plan.ws > 0 && !ws) || ((uintptr_t)ws & 15)) return SVD_EINVAL;
    if (dtype != SVD_DTYPE_BF16 && dtype != SVD_DTYPE_F16) return SVD_EINVAL;
    if (!(eps >= 0.f) || (q_start && !causal)) return SVD_EINVAL;
    if ((q_sb | q_st | q_sh | k_sb | k_st | k_sh | v_sb | v_st | v_sh | o_sb | o_st | o_sh) & 7) return SVD_EINVAL;
    if (batch == 0 || n_q == 0) return SVD_OK;
    if (!Q || !O || !lam || (n_k > 0 && (!K || !V))) return SVD_EINVAL;
    if (((uintptr_t)Q | (uintptr_t)K | (uintptr_t)V | (uintptr_t)O) & 15 || ((uintptr_t)lam | (uintptr_t)gamma | (uintptr_t)k_len | (uintptr_t)q_start) & 3) return SVD_EINVAL;
    if (k_st < 0 || v_st < 0 || k_st > (1 << 25) || v_st > (1 << 25)) return SVD_EINVAL;          // a tile's rows are addressed with 32-bit offsets
    const int group = heads / kv_heads;
    // positions are 32-bit numbers, and the last shares of a wave's keys may begin and end up to 1024 tiles behind the last key
    if ((int64_t)n_q * group > 0x7fffff00 || n_k > 0x7fff0000) return SVD_EINVAL;
    const DiffArgs p = {Q, q_sb, q_st, q_sh, K, k_sb, k_st, k_sh, V, v_sb, v_st, v_sh, O, o_sb, o_st, o_sh, lam, lambda_init, gamma, eps, k_len, q_start,
                        n_q, n_k, kv_heads, group, causal};
    const int64_t grid = (int64_t)plan.row_blocks * batch * kv_heads * plan.shares;
    const int threads = plan.form == ROWS ? 256 : plan.form == GROUP ? GROUP_WAVES * 64 : 64;
    if (grid > 0xffffffff / threads || (int64_t)batch * heads * n_q > 0x7fffffff) return SVD_EINVAL;          // (a launch has less than 2^32 threads)
    if (plan.form == ROWS) {
        constexpr int LDS = 8 * 32 * ROW_B + 4 * Q_B;          // rings and map 2's queries: 76 KiB, two workgroups on a CU (two of 80 do not fit)
        SVD_DISPATCH_DTYPE(dtype, {
            SVD_ALLOW_LDS(attn_diff_rows_kernel<E>, LDS);
            hipLaunchKernelGGL((attn_diff_rows_kernel<E>), dim3((unsigned)grid), dim3(256), LDS, (hipStream_t)stream, p, plan.row_blocks);
        });
    } else if (plan.form == GROUP) {
        SVD_DISPATCH_DTYPE(dtype, {
            SVD_ALLOW_LDS(attn_diff_group_kernel<E>, GROUP_LDS);
            hipLaunchKernelGGL((attn_diff_group_kernel<E>), dim3((unsigned)grid), dim3(GROUP_WAVES * 64), GROUP_LDS, (hipStream_t)stream, p);
        });
    } else {
        const int LDS = (n_k > 32 ? 4 : 2) * 32 * ROW_B;          // one tile needs no second buffer: 8 waves on a CU instead of 5 (25 keys x 23040 heads: 128 us; 174 when it was measured, 300 with two and rows written 8 bytes at a time)
        SVD_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((attn_diff_wave_kernel<E>), dim3((unsigned)grid), dim3(64), LDS, (hipStream_t)stream, p, plan.row_blocks, plan.shares, (float*)ws));
        SVD_CHECK_LAUNCH("attn_diff");
        if (plan.shares > 1)
            SVD_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((attn_diff_join_kernel<E>), dim3((unsigned)((int64_t)batch * heads * n_q)), dim3(256), 0, (hipStream_t)stream, p, plan.shares, (const float*)ws));
    }
    SVD_CHECK_LAUNCH("attn_diff");
    return SVD_OK;
}
