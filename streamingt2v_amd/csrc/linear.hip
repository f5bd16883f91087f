// Matrix product with bias, activation and residual in its epilogue, operands fp16 | bf16 | e4m3 (gfx950).
//   Y[m, n] = act( xs[m] ws[n] sum_k X[m, k] W[n, k] + bias[n] ) + R[m, n]
// Products accumulate in fp32; the scales, the bias, the activation and the residual act on the fp32 value, which is rounded once, to Y's type.
// A K step is 128 BYTES of a row for every operand type (64 fp16 / bf16 values, 128 e4m3 values): one staging and one LDS layout serve all of them, and
// v_mfma_f32_32x32x16 (16 bit) and v_mfma_f32_32x32x64_f8f6f4 (e4m3, twice the rate) do the same number of cycles of work on the same bytes.
//
// e4m3 operands have two forms.  The e4m3 matrix instruction adds the products of 8 consecutive k to a sum whose last bit is 2^-13 of the largest of them
// (measured: next to 2^16, 2^3 counts and 2^2 does not; across groups of 8 it adds in fp32): up to 7 * 2^-13 of a group's largest product is cut off, 1e-5 to
// 5e-5 of a result in the 2-norm.  A result rounded to 16 bits (2^-11, 2^-8) does not show that; an fp32 result does, so for fp32 results the values are
// widened to fp16 (exact: e4m3's 448 .. 2^-9 lie inside it) and multiplied by the fp16 instruction, at its rate.
#include "svd_common.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

struct InF8 { static constexpr int kBytes = 1; static constexpr bool kWiden = false; };
struct InF8Wide { static constexpr int kBytes = 1; static constexpr bool kWiden = true; };
struct InF16 { static constexpr int kBytes = 2; static constexpr bool kWiden = false; using E = ElemF16; };
struct InBF16 { static constexpr int kBytes = 2; static constexpr bool kWiden = false; using E = ElemBF16; };

struct LinArgs {
    const char* X; int64_t ldx;              // leading dimensions of X and W in bytes
    const char* W; int64_t ldw;
    const float* xs; const float* ws; const float* bias;
    const void* R; int64_t ldr;
    void* Y; int64_t ldy;
    int M, N, kbytes, act, res_f32, out_f32, pair;          // pair: two adjacent columns of Y (and R) are one aligned access
};

// 64 bytes of K of 32 rows: lane l holds row l % 32.  Which k a lane's bytes are does not matter to a sum as long as both operands agree: half h of the wave holds
// chunks 4 s + 2 h and 4 s + 2 h + 1 of 16 bytes.
template <class In> struct Frag {
    uint4 v[In::kWiden ? 4 : 2];
    __device__ __forceinline__ void set(uint4 c0, uint4 c1) {
        if constexpr (In::kWiden) { widen(c0, v[0], v[1]); widen(c1, v[2], v[3]); }
        else { v[0] = c0; v[1] = c1; }
    }
    static __device__ __forceinline__ uint32_t two(uint32_t w, bool high) {
        return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))
                    : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    }
    static __device__ __forceinline__ void widen(uint4 c, uint4& a, uint4& b) {
        a = make_uint4(two(c.x, false), two(c.x, true), two(c.y, false), two(c.y, true));
        b = make_uint4(two(c.z, false), two(c.z, true), two(c.w, false), two(c.w, true));
    }
};
template <class In> __device__ __forceinline__ f32x16_t mma64(const Frag<In>& a, const Frag<In>& b, f32x16_t c) {
    if constexpr (In::kWiden) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = ElemF16::mfma(a.v[i], b.v[i], c);
        return c;
    } else if constexpr (In::kBytes == 1) {
        const i32x8_t x = {(int)a.v[0].x, (int)a.v[0].y, (int)a.v[0].z, (int)a.v[0].w, (int)a.v[1].x, (int)a.v[1].y, (int)a.v[1].z, (int)a.v[1].w};
        const i32x8_t y = {(int)b.v[0].x, (int)b.v[0].y, (int)b.v[0].z, (int)b.v[0].w, (int)b.v[1].x, (int)b.v[1].y, (int)b.v[1].z, (int)b.v[1].w};
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);     // block scales 2^0: the rows' scales are applied in the epilogue
    } else {
        c = In::E::mfma(a.v[0], b.v[0], c);
        return In::E::mfma(a.v[1], b.v[1], c);
    }
}

// tanh form of GELU: 0.5 v (1 + tanh u) = v / (1 + exp(-2 u)),  u = sqrt(2 / pi) (v + 0.044715 v^3)
__device__ __forceinline__ float gelu_tanh_f(float v) {
    const float u = 0.7978845608028654f * fmaf(0.044715f * v * v, v, v);
    return v * __builtin_amdgcn_rcpf(1.f + __expf(-2.f * u));
}
__device__ __forceinline__ float act_f(float v, int act) {
    switch (act) {
        case SVD_ACT_RELU: return v < 0.f ? 0.f : v;          // keeps a NaN
        case SVD_ACT_GELU: return gelu_erf_f(v);
        case SVD_ACT_GELU_TANH: return gelu_tanh_f(v);
        case SVD_ACT_SILU: return silu_f(v);
        default: return v;
    }
}

template <class Eo> __device__ __forceinline__ void epilogue(const LinArgs& p, int m, int n, float acc) {
    float v = acc;
    if (p.xs) v *= p.xs[m];
    if (p.ws) v *= p.ws[n];
    if (p.bias) v += p.bias[n];
    v = act_f(v, p.act);
    if (p.R) v += p.res_f32 ? ((const float*)p.R)[m * p.ldr + n] : Eo::to_f32(((const uint16_t*)p.R)[m * p.ldr + n]);
    if (p.out_f32) ((float*)p.Y)[m * p.ldy + n] = v;
    else ((uint16_t*)p.Y)[m * p.ldy + n] = Eo::from_f32(v);
}

// 16 bytes at k-byte `kb` of a row of `kbytes` bytes, zeros behind its end; rows of any alignment
template <int EB> __device__ __forceinline__ uint4 load_chunk(const char* row, int kb, int kbytes) {
    struct __attribute__((packed, aligned(EB))) U { uint32_t x, y, z, w; };
    uint4 r = make_uint4(0, 0, 0, 0);
    if (kb + 16 <= kbytes) {
        const U u = *(const U*)(row + kb);
        r = make_uint4(u.x, u.y, u.z, u.w);
    } else if (kb < kbytes) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; i += EB)
            if (kb + i < kbytes) {
                const uint32_t v = EB == 1 ? *(const uint8_t*)(row + kb + i) : *(const uint16_t*)(row + kb + i);
                w[i >> 2] |= v << (8 * (i & 3));
            }
        r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}

// ---- large products: BM x BN outputs per workgroup of WM x WN waves, each TM x TN tiles of 32 x 32; rows 16-byte aligned ----
// K goes in steps of 128 bytes (whole cache lines: with 64 the L2 has twice the requests to serve) through two LDS slots, rows of 128 bytes with 16-byte chunks
// swizzled by (row >> 1) & 7: 16 lanes that read one chunk of 16 rows touch all 64 banks once.  A half step of 64 bytes multiplies fragments that the half before has read
// and reads the next half's between its matrix instructions.  So a slot is free when the first half of its step is done, and is filled then, by LDS-DMA, for the
// step after the next: two halves of a step (2000 cycles of matrix work) ahead of its use, one barrier a step.
// W's rows lie in LDS as even, then odd columns of each 64: a lane's two tiles of such a block are two adjacent columns, so results leave (and residuals come) as
// pairs, 32 lanes a contiguous 128 (fp32: 256) bytes of a row.
// Measured, 256 x 256: bf16 28800 x 1280 x 5120 onto an fp32 stream 390 us (0.97 PFLOP/s; two whole rounds 320 us, the split third 43, the join 17), e4m3
// 28800 x 5120 x 1280 with GELU 260 us (1.45 PFLOP/s), 226 without scales, bias and activation; e4m3 to fp32 (widened, 128 x 128) 374.  The same loop without its requests and LDS
// reads takes 232 of the 320 us (1.47 PFLOP/s, what a large library product reaches), without either of them 286; one workgroup fills a CU, so nothing runs beside its epilogue.
// The whole-tile kernel takes all 256 registers and spills 32 (68 bytes a lane; 74 MB of the 369 that the e4m3 product writes); the kernel of the shares, the same loop
// without the epilogue, 248 to 254 and none.
template <int WM_, int WN_, int TM_, int TN_> struct Tile {
    static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, WAVES = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32, SLOT = (BM + BN) * 128, REQ = (BM + BN) / 8 / WAVES;
};
__device__ const uint4 g_zeros = {0, 0, 0, 0};

template <int ACT, int N> __device__ __forceinline__ void act_all(f32x16_t (&acc)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            if constexpr (ACT == SVD_ACT_GELU) {
                const svd_f32x2 y = gelu_erf_f2(svd_f32x2{acc[i][r], acc[i + 1][r]});
                acc[i][r] = y[0]; acc[i + 1][r] = y[1];
            } else {
                acc[i][r] = act_f(acc[i][r], ACT); acc[i + 1][r] = act_f(acc[i + 1][r], ACT);
            }
        }
}

// TM x TN finished tiles of a wave: scales and bias, activation, residual, one rounding.  m0, n0: the wave's first row and column; xs: its rows' scales (LDS).
// Columns come and go as pairs; `whole`: all its rows exist.
template <class Eo, int TM, int TN> __device__ __forceinline__ void finish_tiles(const LinArgs& p, f32x16_t (&acc)[TM * TN], int m0, int n0, const float* xs, bool whole, int l31, int hi) {
#pragma unroll
    for (int b = 0; b < TN / 2; ++b) {
        const int c0 = min(n0 + 64 * b + 2 * l31, p.N - 1), c1 = min(c0 + 1, p.N - 1);
        const float w0 = p.ws ? p.ws[c0] : 1.f, w1 = p.ws ? p.ws[c1] : 1.f, b0 = p.bias ? p.bias[c0] : 0.f, b1 = p.bias ? p.bias[c1] : 0.f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x4 = *(const float4*)(xs + 32 * i + 8 * g + 4 * hi);
                const float x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = 4 * g + k;
                    acc[i * TN + 2 * b][r] = fmaf(acc[i * TN + 2 * b][r] * x[k], w0, b0);
                    acc[i * TN + 2 * b + 1][r] = fmaf(acc[i * TN + 2 * b + 1][r] * x[k], w1, b1);
                }
            }
    }
    if (p.act == SVD_ACT_RELU) act_all<SVD_ACT_RELU>(acc);
    else if (p.act == SVD_ACT_GELU) act_all<SVD_ACT_GELU>(acc);
    else if (p.act == SVD_ACT_GELU_TANH) act_all<SVD_ACT_GELU_TANH>(acc);
    else if (p.act == SVD_ACT_SILU) act_all<SVD_ACT_SILU>(acc);
    // Addresses: the row is the wave's (scalars), a lane adds its column pair and, in the upper half, four rows, in 32 bits.
    const int ey = p.out_f32 ? 4 : 2, er = p.res_f32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int b = 0; b < TN / 2; ++b) {
            const int n = n0 + 64 * b + 2 * l31, mb = m0 + 32 * i;
            f32x16_t &v0 = acc[i * TN + 2 * b], &v1 = acc[i * TN + 2 * b + 1];
            if (n >= p.N) continue;
            if (!p.pair) {          // odd widths or strides: element by element
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int m = mb + 8 * (r >> 2) + (r & 3) + 4 * hi;
                    if (m >= p.M) continue;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (n + c >= p.N) continue;
                        float v = c ? v1[r] : v0[r];
                        if (p.R) v += p.res_f32 ? ((const float*)p.R)[m * p.ldr + n + c] : Eo::to_f32(((const uint16_t*)p.R)[m * p.ldr + n + c]);
                        if (p.out_f32) ((float*)p.Y)[m * p.ldy + n + c] = v;
                        else ((uint16_t*)p.Y)[m * p.ldy + n + c] = Eo::from_f32(v);
                    }
                }
                continue;
            }
            if (p.R) {
                const char* base = (const char*)p.R + ((int64_t)mb * p.ldr + n0 + 64 * b) * er;
                const uint32_t lane_off = (4 * hi * (uint32_t)p.ldr + 2 * l31) * er;
#pragma unroll
                for (int half = 0; half < 16; half += 8) {          // eight rows' residuals in flight
                    float2 res[16];
#pragma unroll
                    for (int r = half; r < half + 8; ++r) {
                        const int row = 8 * (r >> 2) + (r & 3);
                        const char* at = whole ? base + (int64_t)row * p.ldr * er + lane_off
                                               : (const char*)p.R + ((int64_t)min(mb + row + 4 * hi, p.M - 1) * p.ldr + n) * er;
                        if (p.res_f32) res[r] = *(const float2*)at;
                        else { const uint32_t w = *(const uint32_t*)at; res[r] = make_float2(Eo::lo(w), Eo::hi(w)); }
                    }
#pragma unroll
                    for (int r = half; r < half + 8; ++r) { v0[r] += res[r].x; v1[r] += res[r].y; }
                }
            }
            char* base = (char*)p.Y + ((int64_t)mb * p.ldy + n0 + 64 * b) * ey;
            const uint32_t lane_off = (4 * hi * (uint32_t)p.ldy + 2 * l31) * ey;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 8 * (r >> 2) + (r & 3);
                char* at = base + (int64_t)row * p.ldy * ey + lane_off;
                if (whole || mb + row + 4 * hi < p.M) {
                    if (p.out_f32) *(float2*)at = make_float2(v0[r], v1[r]);
                    else *(uint32_t*)at = Eo::pack(v0[r], v1[r]);
                }
            }
        }
}

// Rows of any alignment laid out anew, 16-byte aligned, zeros behind their end: a copy of X and W is cheap next to a product that needs tiles (the same tiles filled through
// registers from unaligned rows: 543 us instead of 258 + 20 at 28800 x 5120 x 1280 e4m3).
template <int EB> __global__ __launch_bounds__(256) void linear_align_kernel(const char* src, int64_t ld, char* dst, int64_t rows, int kbytes) {
    const int chunks = (kbytes + 15) >> 4;
    const int64_t n = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / chunks;
        const int c = (int)(i - row * chunks);
        ((uint4*)dst)[i] = load_chunk<EB>(src + row * ld, c * 16, kbytes);
    }
}

// Place of tile `w` of the list: 8 tiles of M by all tiles of N, then the next 8: the 32 workgroups that an XCD runs at once share 8 bands of X and 4 of W.
__device__ __forceinline__ void tile_place(int w, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int g = w / (8 * tiles_n), gm = min(8, tiles_m - g * 8), u = w - g * 8 * tiles_n;
    tm = g * 8 + u % gm;
    tn = u / gm;
}
// Split of a product's last, incomplete round of workgroups: the first `whole` tiles have a workgroup each, the others `shares` of K each, whose sums meet in
// scratch memory (fp32, [share][wave][tile][4 rows of 4][lane]) and are finished by linear_join_kernel in the order of the shares.
struct Rounds { int whole, shares; float* ws; };

// SHARE: the launch over the shares of K of the tiles behind the whole ones
template <class In, class Eo, class T, bool SHARE> __global__ __launch_bounds__(T::WAVES * 64, 2) void linear_tile_kernel(LinArgs p, int tiles_m, int tiles_n, Rounds rd) {
    constexpr int TM = T::TM, TN = T::TN, NF = TM + TN;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const uint32_t lds = lds_addr_of(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    int m0, n0, k_from = 0, steps = (p.kbytes + 127) >> 7;          // steps of 128 bytes of K
    {
        int w;
        if constexpr (!SHARE) {          // consecutive workgroups go round the 8 XCDs: each gets a contiguous piece of the list
            const int n = rd.whole, x = blockIdx.x & 7, q = n >> 3, r = n & 7;
            w = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (blockIdx.x >> 3);
        } else {
            w = rd.whole + blockIdx.x / rd.shares;
            const int share = blockIdx.x % rd.shares, per = (steps + rd.shares - 1) / rd.shares;
            k_from = min(share * per, steps);
            steps = min(per, steps - k_from);
        }
        tile_place(w, tiles_m, tiles_n, m0, n0);
        m0 *= T::BM; n0 *= T::BN;
    }
    const int wm = (wave / T::WN) * TM * 32, wn = (wave % T::WN) * TN * 32;
    // requests: 8 rows of 128 bytes each; a wave's are all of X or all of W
    const bool is_x = wave * T::REQ < T::BM / 8;
    const char* src = (is_x ? p.X + (int64_t)m0 * p.ldx : p.W + (int64_t)n0 * p.ldw) + (int64_t)k_from * 128;
    const int kbytes = p.kbytes - k_from * 128;
    const int chunk = (lane & 7) ^ (lane >> 4);          // of the even requests; the odd ones' differs in bit 2
    uint32_t off[T::REQ];
#pragma unroll
    for (int u = 0; u < T::REQ; ++u) {
        const int r = (wave * T::REQ + u) * 8 + (lane >> 3) - (is_x ? 0 : T::BM);
        const int n = (r & ~63) | ((r & 31) << 1) | ((r >> 5) & 1);
        const int row = is_x ? min(r, p.M - 1 - m0) : min(n, p.N - 1 - n0);          // rows behind the last repeat it; their results are not stored
        off[u] = (uint32_t)row * (uint32_t)(is_x ? p.ldx : p.ldw) + (chunk ^ (u & 1) << 2) * 16;
    }
    auto request = [&](int j) {
        const uint32_t dst = lds + (j & 1) * T::SLOT + wave * T::REQ * 1024;
        if (__builtin_expect(j * 128 + 128 <= kbytes, 1)) {
#pragma unroll
            for (int u = 0; u < T::REQ; ++u) glds16_saddr(off[u], src + (int64_t)j * 128, __builtin_amdgcn_readfirstlane(dst + u * 1024));
        } else {          // the last step's chunks behind K are zeros
#pragma unroll
            for (int u = 0; u < T::REQ; ++u)
                glds16_asm(j * 128 + (chunk ^ (u & 1) << 2) * 16 < kbytes ? src + (int64_t)j * 128 + off[u] : (const char*)&g_zeros, __builtin_amdgcn_readfirstlane(dst + u * 1024));
        }
    };
    f32x16_t acc[TM * TN];
#pragma unroll
    for (int i = 0; i < TM * TN; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    uint4 f[2][NF][2];
    const uint32_t la = l31 * 128 + (((2 * hi) ^ ((l31 >> 1) & 7)) << 4);
    auto read = [&](int j, int half, int e) {          // fragment e of half a step: X tiles 0 .. TM - 1, then W tiles
        const uint32_t at = (lds + (j & 1) * T::SLOT + (e < TM ? (wm + 32 * e) * 128 : (T::BM + wn + 32 * (e - TM)) * 128) + la) ^ (half * 64);
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        f[half][e][0] = __builtin_bit_cast(uint4, *(const __attribute__((address_space(3))) u32x4_t*)at);
        f[half][e][1] = __builtin_bit_cast(uint4, *(const __attribute__((address_space(3))) u32x4_t*)(at ^ 16));
    };
    // the order in which a step's fragments are read for the next: first those that its first products take
    auto nth = [](int e) { return e == 0 ? 0 : e <= TN ? TM + e - 1 : e - TN; };
    if (steps > 0) request(0);
    if (steps > 1) request(1);
    svd_wait_dma();
    __syncthreads();
#pragma unroll
    for (int e = 0; e < NF; ++e) read(0, 0, e);
    auto half_step = [&]<int SET>(int j) {
        if constexpr (SET == 1) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");          // step j + 1 is there; this wave's reads of step j are done
            __syncthreads();
            if (j + 2 < steps) request(j + 2);
        }
        constexpr int PASSES = In::kWiden ? 4 : In::kBytes == 1 ? 1 : 2;          // matrix instructions per tile and step
        int e = 0;
#pragma unroll
        for (int h = 0; h < PASSES; ++h)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int n = 0; n < TN; ++n) {
                    if (e < NF) read(j + SET, SET ^ 1, nth(e));
                    ++e;
                    const uint4 *a = f[SET][i], *b = f[SET][TM + n];
                    f32x16_t& c = acc[i * TN + n];
                    if constexpr (In::kWiden) {
                        uint4 x[2], y[2];
                        Frag<In>::widen(a[h >> 1], x[0], x[1]);
                        Frag<In>::widen(b[h >> 1], y[0], y[1]);
                        c = ElemF16::mfma(x[h & 1], y[h & 1], c);
                    } else if constexpr (In::kBytes == 1) {
                        Frag<In> x, y;
                        x.set(a[0], a[1]); y.set(b[0], b[1]);
                        c = mma64<In>(x, y, c);
                    } else {
                        c = In::E::mfma(a[h], b[h], c);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
    };
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
        half_step.template operator()<0>(j);
        half_step.template operator()<1>(j);
    }

    if constexpr (SHARE) {          // the sums, as they lie
        float4* out = (float4*)rd.ws + ((int64_t)blockIdx.x * T::WAVES + wave) * (TM * TN * 4 * 64) + lane;
#pragma unroll
        for (int i = 0; i < TM * TN; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) out[(i * 4 + g) * 64] = make_float4(acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]);
    } else {
        float* s_xs = (float*)smem;
        __syncthreads();          // the ring's last reads are done
        for (int r = tid; r < T::BM; r += T::WAVES * 64) s_xs[r] = p.xs ? p.xs[min(m0 + r, p.M - 1)] : 1.f;
        __syncthreads();
        finish_tiles<Eo, TM, TN>(p, acc, m0 + wm, n0 + wn, s_xs + wm, m0 + T::BM <= p.M, l31, hi);
    }
}

// One workgroup per split tile and band of 32 rows of its waves: the shares' sums in their order, then the epilogue.
template <class Eo, class T> __global__ __launch_bounds__(T::WAVES * 64) void linear_join_kernel(LinArgs p, int tiles_m, int tiles_n, Rounds rd) {
    __shared__ float s_xs[T::WAVES][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), t = blockIdx.x / T::TM, i = blockIdx.x % T::TM;
    int m0, n0;
    tile_place(rd.whole + t, tiles_m, tiles_n, m0, n0);
    m0 = m0 * T::BM + (wave / T::WN) * T::TM * 32 + 32 * i;
    n0 = n0 * T::BN + (wave % T::WN) * T::TN * 32;
    f32x16_t acc[T::TN];
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[j][r] = 0.f;
    for (int s = 0; s < rd.shares; ++s) {
        const float4* in = (const float4*)rd.ws + ((int64_t)(t * rd.shares + s) * T::WAVES + wave) * (T::TM * T::TN * 4 * 64) + i * T::TN * 4 * 64 + lane;
#pragma unroll
        for (int j = 0; j < T::TN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 v = in[(j * 4 + g) * 64];
                acc[j][4 * g] += v.x; acc[j][4 * g + 1] += v.y; acc[j][4 * g + 2] += v.z; acc[j][4 * g + 3] += v.w;
            }
    }
    if (lane < 32) s_xs[wave][lane] = p.xs ? p.xs[min(m0 + lane, p.M - 1)] : 1.f;
    __syncthreads();
    finish_tiles<Eo, 1, T::TN>(p, acc, m0, n0, s_xs[wave], m0 + 32 <= p.M, lane & 31, lane >> 5);
}

// ---- few rows: 32 columns x 32 TM rows per workgroup, its waves take 64-byte steps of K in turn and add up through LDS.  No staging: the weights are read once, straight
// into fragments; rows of any alignment.  What bounds it is latency and the rate at which a CU takes requests of 64 lanes, so the work is spread: 16 or 8 columns to a
// workgroup while all of them are on the chip at once, sixteen waves for long rows.  A tile of 8 (16) columns and at most as many rows multiplies 4 (2) steps of K at once: the
// 32 rows and columns of the matrix instruction are its rows and columns in `groups` different places of K, and only the products of the same place count.
// us, before and after: 1 x 1280 x 5120 bf16 13.3 -> 6.0, e4m3 8.0 -> 4.5 (6.6 MB); 64 x 1280 x 5120 bf16 29 -> 17; 77 x 1001 x 515 fp16 11 -> 6.7; one row of 1280 by
// 5120 columns, e4m3 4.2. ----
template <class In, class Eo, int TM, int NW> __global__ __launch_bounds__(NW * 64) void linear_rows_kernel(LinArgs p, int tiles_n, int log_cols, int groups) {
    const int cols = 1 << log_cols;
    __shared__ __attribute__((aligned(16))) float part[NW][TM * 16][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, hi = lane >> 5;
    const int m0 = (blockIdx.x / tiles_n) * (groups > 1 ? cols : 32 * TM), n0 = (blockIdx.x % tiles_n) * cols;
    const int kg = groups > 1 ? l31 >> log_cols : 0, lr = l31 - kg * cols;          // the lane's share of K and its row and column of the tile
    const int wb = lr < cols && n0 + lr < p.N ? p.kbytes : 0;          // rows that do not count are zeros and cost no requests
    const char* wr = p.W + (int64_t)min(n0 + lr, p.N - 1) * p.ldw;
    const char* xr[TM];
    int xb[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) xb[i] = m0 + 32 * i + lr < p.M ? p.kbytes : 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) xr[i] = p.X + (int64_t)min(m0 + 32 * i + lr, p.M - 1) * p.ldx;
    f32x16_t acc[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    constexpr int U = TM == 1 ? 4 : 2;          // steps in flight
    const int steps = (p.kbytes + 64 * groups - 1) / (64 * groups);
    for (int j0 = wave; j0 < steps; j0 += NW * U) {
        uint4 w[U][2], x[U][TM][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = ((j0 + u * NW) * groups + kg) * 64 + 32 * hi;          // behind K: zeros
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                w[u][c] = load_chunk<In::kBytes>(wr, kb + 16 * c, wb);
#pragma unroll
                for (int i = 0; i < TM; ++i) x[u][i][c] = load_chunk<In::kBytes>(xr[i], kb + 16 * c, xb[i]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Frag<In> a, b;
            b.set(w[u][0], w[u][1]);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                a.set(x[u][i][0], x[u][i][1]);
                acc[i] = mma64<In>(a, b, acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) part[wave][i * 16 + r][lane] = acc[i][r];
    __syncthreads();
    const int log_w = groups > 1 ? log_cols : 5;
    for (int o = tid; o < TM << 2 * log_w; o += NW * 64) {
        const int c = o & ((1 << log_w) - 1), row = o >> log_w, m = m0 + row, n = n0 + c;
        if (m >= p.M || n >= p.N || c >= cols) continue;
        float v = 0.f;
        for (int g = 0; g < groups; ++g) {          // of the tile, the blocks whose row and column have the same share of K
            const int x = row + g * cols, r = (x >> 3) * 4 + (x & 3), ln = ((x >> 2) & 1) * 32 + c + g * cols;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += part[w][r][ln];
        }
        epilogue<Eo>(p, m, n, v);
    }
}

using Big = Tile<2, 4, 4, 2>;              // 256 x 256, eight waves, 128 KiB: one workgroup on a CU
using Small = Tile<2, 2, 2, 2>;            // 128 x 128, four waves, 64 KiB: two
constexpr int CUS = 256;
constexpr int ROWS_TWO = 256;

// Which form, from sizes alone.  Both sides measured, us a call in a graph, bf16 | e4m3 to 16 bits:
//   rows kernel below 64 tiles of 128 x 128, because such tiles leave most CUs without one, and shares of K cost a join:
//     K = 1280, rows kernel against tiles: 20 tiles (256 x 1280) 10.8 | 7.5 against 12.9 | 9.9; 40 (512 x 1280) 18.0 | 10.8, 16.4 | 10.8; 60 (768 x 1280) 17.7 | 11.0, 17.1 | 12.1;
//     64 (1024 x 1024) 17.7 | 11.0, 17.8 | 12.0; 70 (896 x 1280) 24.1 | 14.4, 18.6 | 12.5; 80 (1024 x 1280) 24.1 | 14.7, 19.1 | 13.1.
//     With K = 5120 the border lies lower than the rule has it: 10 tiles (128 x 1280) 21.1 | 12.5, 16.7 | 14.3; 20 (256 x 1280) 33.5 | 17.2, 20.0 | 17.1; 60 (768 x 1280) 62.9 | 33.2, 25.4 | 25.5.
//   256 x 256 from 128 of them on (a workgroup for every other CU), because they read half the operand bytes a product: K = 1280, 256 x 256 against 128 x 128:
//     160 tiles (5120 x 2048) 36.0 | 24.9, 44.4 | 30.5; 300 (5120 x 3840) 72.0 | 47.9, 69.6 | 45.3; 2260 (28800 x 5120) e4m3 with GELU 260, 266; 565 (28800 x 1280 x 5120) bf16 390, 454.
//     At 128 tiles (4096 x 2048) the rule begins too early: 41.1 | 34.0, 24.8 | 15.7, all of them split in two shares of K here and 512 places filled once there.
enum { ROWS, BIG, SMALL };
struct LinPlan { int form, whole, shares; int64_t ws; };
template <class T> LinPlan rounds_of(int form, int64_t tm, int64_t tn, int64_t kbytes, int slots) {
    const int64_t tiles = tm * tn, rest = tiles % slots, steps = (kbytes + 127) / 128;
    LinPlan r = {form, (int)tiles, 1, 0};
    int64_t shares = rest ? slots / rest : 1;
    if (shares > steps / 4) shares = steps / 4;          // a share of at least 4 steps
    if (shares > 8) shares = 8;
    if (shares > 1) { r.whole = (int)(tiles - rest); r.shares = (int)shares; r.ws = rest * shares * T::BM * T::BN * 4; }
    return r;
}
LinPlan lin_plan(int64_t M, int64_t N, int64_t kbytes, bool wide) {
    auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    const int64_t small = up(M, 128) * up(N, 128), big = up(M, 256) * up(N, 256);
    if (M <= 64 || small < 64) return {ROWS, 0, 1, 0};
    if (!wide && big >= 128) return rounds_of<Big>(BIG, up(M, 256), up(N, 256), kbytes, CUS);          // (widened fragments do not leave registers for the large tile)
    return rounds_of<Small>(SMALL, up(M, 128), up(N, 128), kbytes, 2 * CUS);
}

template <class In, class Eo, class T> int launch_tiles(const LinArgs& p, const LinPlan& plan, float* ws, hipStream_t stream) {
    const int tm = (p.M + T::BM - 1) / T::BM, tn = (p.N + T::BN - 1) / T::BN, rest = tm * tn - plan.whole;
    const Rounds rd = {plan.whole, plan.shares, ws};
    constexpr int LDS = 2 * T::SLOT;
    if (plan.whole) {
        if (LDS > 65536) SVD_ALLOW_LDS((linear_tile_kernel<In, Eo, T, false>), LDS);
        hipLaunchKernelGGL((linear_tile_kernel<In, Eo, T, false>), dim3((unsigned)plan.whole), dim3(T::WAVES * 64), LDS, stream, p, tm, tn, rd);
        SVD_CHECK_LAUNCH("linear_act");
    }
    if (rest) {
        if (LDS > 65536) SVD_ALLOW_LDS((linear_tile_kernel<In, Eo, T, true>), LDS);
        hipLaunchKernelGGL((linear_tile_kernel<In, Eo, T, true>), dim3((unsigned)(rest * plan.shares)), dim3(T::WAVES * 64), LDS, stream, p, tm, tn, rd);
        SVD_CHECK_LAUNCH("linear_act");
        hipLaunchKernelGGL((linear_join_kernel<Eo, T>), dim3((unsigned)(rest * T::TM)), dim3(T::WAVES * 64), 0, stream, p, tm, tn, rd);
    }
    SVD_CHECK_LAUNCH("linear_act");
    return SVD_OK;
}

int64_t aligned_copy_bytes(int64_t M, int64_t N, int64_t kbytes) { return (M + N) * ((kbytes + 15) & ~15ll); }

template <class In, class Eo> int launch(LinArgs p, void* ws, int64_t ws_bytes, hipStream_t stream) {
    const LinPlan plan = lin_plan(p.M, p.N, p.kbytes, In::kWiden);
    if (plan.form == ROWS) {
        // Columns to a workgroup: halved while every one still has a CU; two tiles of rows share the weights' fragments once there are more than that
        // (64 x 1280 x 5120: 29 us with two, 17 without; 256 x 1280 x 5120: 33 and 42).
        int log_cols = 5;
        const int64_t tm = (p.M + 31) / 32;
        while (log_cols > 3 && (((int64_t)p.N - 1 >> (log_cols - 1)) + 1) * tm <= CUS) --log_cols;
        const int cols = 1 << log_cols;
        const int groups = p.M <= cols && p.kbytes < 1 << 30 ? 32 / cols : 1;          // (positions in K stay 32-bit numbers)
        const int64_t tn = (p.N + cols - 1) / cols, ones = tm * tn;
        const bool two = p.M > 32 && ones > ROWS_TWO, many = p.kbytes > 2048 * groups && ones <= ROWS_TWO;
        const int64_t grid = two ? (p.M + 63) / 64 * tn : ones;
        if (grid > 0x7fffff) return SVD_EINVAL;          // 2^32 threads
        const dim3 g((unsigned)grid);
        if (two) hipLaunchKernelGGL((linear_rows_kernel<In, Eo, 2, 8>), g, dim3(512), 0, stream, p, (int)tn, log_cols, groups);
        else if (many) hipLaunchKernelGGL((linear_rows_kernel<In, Eo, 1, 16>), g, dim3(1024), 0, stream, p, (int)tn, log_cols, groups);
        else hipLaunchKernelGGL((linear_rows_kernel<In, Eo, 1, 8>), g, dim3(512), 0, stream, p, (int)tn, log_cols, groups);
        SVD_CHECK_LAUNCH("linear_act");
        return SVD_OK;
    }
    constexpr int64_t FAR = 1 << 23;          // tiles are addressed with 32-bit offsets
    const bool anew = (((uintptr_t)p.X | (uintptr_t)p.W | p.ldx | p.ldw | p.kbytes) & 15) || p.ldx >= FAR || p.ldw >= FAR;
    if (ws_bytes < plan.ws + (anew ? aligned_copy_bytes(p.M, p.N, p.kbytes) : 0) || ((plan.ws || anew) && !ws) || ((uintptr_t)ws & 15)) return SVD_EINVAL;
    if ((int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128) * 8 > 0x7fffffff) return SVD_EINVAL;
    if (anew) {
        const int kp = (p.kbytes + 15) & ~15;
        if (kp >= FAR) return SVD_EINVAL;
        char *x = (char*)ws + plan.ws, *w = x + (int64_t)p.M * kp;
        auto copy = [&](const char* src, int64_t ld, char* dst, int64_t rows) {
            const int64_t blocks = (rows * (kp >> 4) + 255) / 256;
            hipLaunchKernelGGL((linear_align_kernel<In::kBytes>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, stream, src, ld, dst, rows, p.kbytes);
        };
        copy(p.X, p.ldx, x, p.M);
        SVD_CHECK_LAUNCH("linear_act");
        copy(p.W, p.ldw, w, p.N);
        SVD_CHECK_LAUNCH("linear_act");
        p.X = x; p.W = w; p.ldx = p.ldw = p.kbytes = kp;
    }
    p.pair = !((p.out_f32 ? (uintptr_t)p.Y & 7 : (uintptr_t)p.Y & 3) | (!p.R ? 0 : p.res_f32 ? (uintptr_t)p.R & 7 : (uintptr_t)p.R & 3) | ((p.ldy | (p.R ? p.ldr : 0) | p.N) & 1)) &&
             p.ldy < (1 << 26) && p.ldr < (1 << 26);
    if constexpr (!In::kWiden)
        if (plan.form == BIG) return launch_tiles<In, Eo, Big>(p, plan, (float*)ws, stream);
    return launch_tiles<In, Eo, Small>(p, plan, (float*)ws, stream);
}

}  // namespace

extern "C" int64_t svd_linear_act_ws_bytes(int64_t M, int32_t N, int32_t K, int32_t flags, int32_t in_dtype, int32_t aligned) {
    if (M < 0 || M > 0x7fffff00 || N < 1 || N > 0x7fffff00 || K < 1 || K > 0x3fffefff) return SVD_EINVAL;
    const bool f8 = in_dtype == SVD_DTYPE_F8;
    const int64_t kbytes = (int64_t)K * (f8 ? 1 : 2);
    const LinPlan plan = lin_plan(M, N, kbytes, f8 && (flags & SVD_LIN_OUT_F32));
    return plan.ws + (plan.form != ROWS && !aligned ? aligned_copy_bytes(M, N, kbytes) : 0);
}

extern "C" int svd_linear_act(const void* X, int64_t ldx, const void* W, int64_t ldw, const float* xscale, const float* wscale, const float* bias,
                              const void* R, int64_t ldr, void* Y, int64_t ldy, int64_t M, int32_t N, int32_t K, int32_t act, int32_t flags,
                              void* ws, int64_t ws_bytes, int32_t in_dtype, int32_t dtype, svd_stream_t stream) {
    const int es = in_dtype == SVD_DTYPE_F8 ? 1 : 2;
    if (!X || !W || !Y || M < 0 || M > 0x7fffff00 || N < 1 || N > 0x7fffff00 || K < 1 || K > 0x3fffefff || ldx < K || ldw < K || ldy < N || (R && ldr < N)) return SVD_EINVAL;
    if (act < SVD_ACT_NONE || act > SVD_ACT_SILU || (flags & ~(SVD_LIN_RES_F32 | SVD_LIN_OUT_F32)) || (!R && (flags & SVD_LIN_RES_F32))) return SVD_EINVAL;
    if (dtype != SVD_DTYPE_BF16 && dtype != SVD_DTYPE_F16) return SVD_EINVAL;
    if (in_dtype != SVD_DTYPE_F8 && in_dtype != dtype) return SVD_EINVAL;
    if (in_dtype != SVD_DTYPE_F8 && (xscale || wscale)) return SVD_EINVAL;
    const uintptr_t f4 = (uintptr_t)xscale | (uintptr_t)wscale | (uintptr_t)bias | ((flags & SVD_LIN_RES_F32) ? (uintptr_t)R : 0) | ((flags & SVD_LIN_OUT_F32) ? (uintptr_t)Y : 0);
    const uintptr_t f2 = (es == 2 ? (uintptr_t)X | (uintptr_t)W : 0) | (uintptr_t)R | (uintptr_t)Y;
    if ((f4 & 3) || (f2 & 1)) return SVD_EINVAL;
    if (M == 0) return SVD_OK;
    const LinArgs p = {(const char*)X, ldx * es, (const char*)W, ldw * es, xscale, wscale, bias, R, ldr, Y, ldy, (int)M, N, K * es, act,
                       !!(flags & SVD_LIN_RES_F32), !!(flags & SVD_LIN_OUT_F32), 0};
    if (in_dtype == SVD_DTYPE_F16) return launch<InF16, ElemF16>(p, ws, ws_bytes, (hipStream_t)stream);
    if (in_dtype == SVD_DTYPE_BF16) return launch<InBF16, ElemBF16>(p, ws, ws_bytes, (hipStream_t)stream);
    if (p.out_f32) return dtype == SVD_DTYPE_F16 ? launch<InF8Wide, ElemF16>(p, ws, ws_bytes, (hipStream_t)stream) : launch<InF8Wide, ElemBF16>(p, ws, ws_bytes, (hipStream_t)stream);
    return dtype == SVD_DTYPE_F16 ? launch<InF8, ElemF16>(p, ws, ws_bytes, (hipStream_t)stream) : launch<InF8, ElemBF16>(p, ws, ws_bytes, (hipStream_t)stream);
}
