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
// P is rounded to the 16-bit type for the matrix cores (at most half a step of the type relative to each weight); scores, maxima, sums and both accumulators
// are fp32, and the row sums add the unrounded weights.
// The heads of a group that share a key / value head are rows of one product: row r = query * group + head, so a causal tile of rows spans few queries.
#include "svd_common.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;
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

// keys of sequence b, in [0, n_k] whatever the lengths' tensor holds
__device__ __forceinline__ int key_count(const DiffArgs& p, int b) { return p.k_len ? max(0, min(p.k_len[b], p.n_k)) : p.n_k; }
// number of keys query q sees
__device__ __forceinline__ int seen_by(const DiffArgs& p, int b, int len, int q) {
    if (!p.causal) return len;
    const int64_t end = (int64_t)(p.q_start ? p.q_start[b] : len - p.n_q) + q + 1;
    return (int)max((int64_t)0, min((int64_t)len, end));
}

// What a query does not see must not reach it, and a weight of 0 is no help against an Inf or NaN in V: 0 * NaN is NaN.  In a tile that some of the block's
// queries see further into than others, non-finite values are looked for; if there are any, the products run on V with zeros in their places, and a second product
// -- of the places with the 0 / 1 mask -- counts for each (channel, query) the non-finite values that it does see: those results become NaN (what p * NaN, and
// inf - lambda inf, come to).  Rare, so it is a branch of its own.
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

// One wave per (sequence, key / value head, 32 rows).
template <class E> __global__ __launch_bounds__(64) void attn_diff_kernel(DiffArgs p, int row_blocks) {
    __shared__ __attribute__((aligned(16))) uint16_t sV[32][128 + 8];
    const int lane = threadIdx.x, l31 = lane & 31, hi = lane >> 5;
    const int rb = blockIdx.x % row_blocks, bh = blockIdx.x / row_blocks, h = bh % p.kv_heads, b = bh / p.kv_heads;
    const int rows = p.n_q * p.group, row = rb * 32 + l31;
    const bool live = row < rows;
    const int q = (live ? row : rows - 1) / p.group, head = h * p.group + (live ? row : rows - 1) % p.group;
    const int len = key_count(p, b), seen = seen_by(p, b, len, q);
    const int last = seen_by(p, b, len, min(rows - 1, rb * 32 + 31) / p.group);         // causal or not, the block's last row sees the most keys
    const int first = p.causal ? seen_by(p, b, len, rb * 32 / p.group) : last;          // ... and its first row the fewest
    const svd_bf16* Qr = p.Q + b * p.q_sb + q * p.q_st + head * p.q_sh;
    const svd_bf16* Kb = p.K + b * p.k_sb + h * p.k_sh;
    const svd_bf16* Vb = p.V + b * p.v_sb + h * p.v_sh;
    uint4 qf[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) qf[i][s] = *(const uint4*)(Qr + 64 * i + 16 * s + 8 * hi);
    f32x16_t o[2][4];
    float m[2] = {M_NONE, M_NONE}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][t][r] = 0.f;
    const float c = 0.125f * LOG2E;
    for (int k0 = 0; k0 < last; k0 += 32) {
        __syncthreads();
        for (int e = lane; e < 32 * 16; e += 64) {
            const int key = k0 + (e >> 4);          // rows behind the last visible key are zeros: nothing of them can reach a product
            *(uint4*)&sV[e >> 4][(e & 15) * 8] = key < last ? *(const uint4*)(Vb + (int64_t)key * p.v_st + (e & 15) * 8) : make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        const svd_bf16* Kr = Kb + (int64_t)min(k0 + l31, last - 1) * p.k_st;
        uint32_t pk[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f32x16_t s;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) s = E::mfma(*(const uint4*)(Kr + 64 * i + 16 * ks + 8 * hi), qf[i][ks], s);
            float mx = M_NONE;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = k0 + 8 * (r >> 2) + 4 * hi + (r & 3);
                s[r] = key < seen ? s[r] * c : -INFINITY;
                mx = fmaxf(mx, s[r]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float m_new = fmaxf(m[i], mx), alpha = __builtin_amdgcn_exp2f(m[i] - m_new);
            m[i] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float p0 = __builtin_amdgcn_exp2f(s[r] - m_new), p1 = __builtin_amdgcn_exp2f(s[r + 1] - m_new);
                sum += p0 + p1;
                pk[i][r >> 1] = E::pack(p0, p1);
            }
            l[i] = l[i] * alpha + sum;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][t][r] *= alpha;
        }
        auto v_frag = [&](int s, int t) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 16 * s + 8 * (j >> 1) + 4 * hi + 2 * (j & 1);
                w[j] = sV[key][32 * t + l31] | ((uint32_t)sV[key + 1][32 * t + l31] << 16);
            }
            return make_uint4(w[0], w[1], w[2], w[3]);
        };
        auto p_frag = [&](int i, int s) { return make_uint4(pk[i][4 * s], pk[i][4 * s + 1], pk[i][4 * s + 2], pk[i][4 * s + 3]); };
        bool bad = false;
        if (k0 + 32 > first) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < 4; ++t) bad |= NonFinite<E>::any(v_frag(s, t));
        }
        if (__builtin_amdgcn_ballot_w64(bad) == 0) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint4 vf = v_frag(s, t);
#pragma unroll
                    for (int i = 0; i < 2; ++i) o[i][t] = E::mfma(vf, p_frag(i, s), o[i][t]);
                }
        } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f32x16_t hit;
#pragma unroll
                for (int r = 0; r < 16; ++r) hit[r] = 0.f;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint4 vf = v_frag(s, t);
                    uint32_t see[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = k0 + 16 * s + 8 * (j >> 1) + 4 * hi + 2 * (j & 1);
                        see[j] = (key < seen ? NonFinite<E>::ONE : 0u) | (key + 1 < seen ? NonFinite<E>::ONE << 16 : 0u);
                    }
                    hit = E::mfma(NonFinite<E>::places(vf), make_uint4(see[0], see[1], see[2], see[3]), hit);
#pragma unroll
                    for (int i = 0; i < 2; ++i) o[i][t] = E::mfma(NonFinite<E>::cleared(vf), p_frag(i, s), o[i][t]);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (hit[r] > 0.f) o[0][t][r] = NAN;
            }
        }
    }
    const float lam = diff_lambda(p.lam, p.lambda_init, lane);
    float w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor(l[i], 32, 64);
        w[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    }
    w[1] *= lam;
    float ss = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[0][t][r] = o[0][t][r] * w[0] - o[1][t][r] * w[1];
            ss = fmaf(o[0][t][r], o[0][t][r], ss);
        }
    ss += __shfl_xor(ss, 32, 64);
    const float norm = p.gamma ? (1.f - p.lambda_init) / sqrtf(ss * (1.f / 128.f) + p.eps) : 1.f;
    if (!live) return;
    svd_bf16* Or = p.O + b * p.o_sb + q * p.o_st + head * p.o_sh;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * t + 2 * r + 4 * hi;
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = o[0][t][r + j] * (p.gamma ? norm * p.gamma[d + j] : 1.f);
            *(uint2*)(Or + d) = make_uint2(E::pack(y[0], y[1]), E::pack(y[2], y[3]));
        }
}

}  // namespace

extern "C" int64_t svd_attn_diff_ws_bytes(int32_t batch, int32_t n_q, int32_t n_k, int32_t heads, int32_t kv_heads) {
    if (batch < 0 || n_q < 0 || n_k < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads) return SVD_EINVAL;
    return 0;
}

extern "C" int svd_attn_diff(const svd_bf16* Q, int64_t q_sb, int64_t q_st, int64_t q_sh, const svd_bf16* K, int64_t k_sb, int64_t k_st, int64_t k_sh,
                             const svd_bf16* V, int64_t v_sb, int64_t v_st, int64_t v_sh, svd_bf16* O, int64_t o_sb, int64_t o_st, int64_t o_sh,
                             const float* lam, float lambda_init, const float* gamma, float eps, const int32_t* k_len, const int32_t* q_start,
                             int32_t batch, int32_t n_q, int32_t n_k, int32_t heads, int32_t kv_heads, int32_t causal, void* ws, int64_t ws_bytes,
                             int32_t dtype, svd_stream_t stream) {
    const int64_t need = svd_attn_diff_ws_bytes(batch, n_q, n_k, heads, kv_heads);
    if (need < 0 || ws_bytes < need || (need > 0 && !ws)) return SVD_EINVAL;
    if (dtype != SVD_DTYPE_BF16 && dtype != SVD_DTYPE_F16) return SVD_EINVAL;
    if (!(eps >= 0.f) || (q_start && !causal)) return SVD_EINVAL;
    if ((q_sb | q_st | q_sh | k_sb | k_st | k_sh | v_sb | v_st | v_sh | o_sb | o_st | o_sh) & 7) return SVD_EINVAL;
    if (batch == 0 || n_q == 0) return SVD_OK;
    if (!Q || !O || !lam || (n_k > 0 && (!K || !V))) return SVD_EINVAL;
    if (((uintptr_t)Q | (uintptr_t)K | (uintptr_t)V | (uintptr_t)O) & 15 || ((uintptr_t)lam | (uintptr_t)gamma | (uintptr_t)k_len | (uintptr_t)q_start) & 3) return SVD_EINVAL;
    const int group = heads / kv_heads;
    if ((int64_t)n_q * group > 0x7fffff00 || n_k > 0x7fffff00) return SVD_EINVAL;
    const DiffArgs p = {Q, q_sb, q_st, q_sh, K, k_sb, k_st, k_sh, V, v_sb, v_st, v_sh, O, o_sb, o_st, o_sh, lam, lambda_init, gamma, eps, k_len, q_start,
                        n_q, n_k, kv_heads, group, causal};
    const int row_blocks = (n_q * group + 31) / 32;
    const int64_t grid = (int64_t)row_blocks * batch * kv_heads;
    if (grid > 0x7fffffff) return SVD_EINVAL;
    SVD_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((attn_diff_kernel<E>), dim3((unsigned)grid), dim3(64), 0, (hipStream_t)stream, p, row_blocks));
    SVD_CHECK_LAUNCH("attn_diff");
    return SVD_OK;
}
