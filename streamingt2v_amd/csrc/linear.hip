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
    int M, N, kbytes, act, res_f32, out_f32;
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

// 128 x 128 outputs per workgroup of four waves (64 x 64 each); operands of any alignment, staged through registers.
template <class In, class Eo> __global__ __launch_bounds__(256) void linear_any_kernel(LinArgs p, int tiles_n) {
    __shared__ __attribute__((aligned(16))) char smem[2 * 128 * 128];
    char* sA = smem; char* sB = smem + 128 * 128;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l31 = lane & 31, hi = lane >> 5;
    const int m0 = (blockIdx.x / tiles_n) * 128, n0 = (blockIdx.x % tiles_n) * 128;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    f32x16_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    for (int k0 = 0; k0 < p.kbytes; k0 += 128) {
        uint4 ra[4], rb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = j * 32 + (tid >> 3), ch = tid & 7;
            ra[j] = load_chunk<In::kBytes>(p.X + (int64_t)min(m0 + row, p.M - 1) * p.ldx, k0 + ch * 16, p.kbytes);
            rb[j] = load_chunk<In::kBytes>(p.W + (int64_t)min(n0 + row, p.N - 1) * p.ldw, k0 + ch * 16, p.kbytes);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = j * 32 + (tid >> 3), slot = (tid & 7) ^ ((row >> 1) & 7);
            *(uint4*)(sA + row * 128 + slot * 16) = ra[j];
            *(uint4*)(sB + row * 128 + slot * 16) = rb[j];
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Frag<In> a[2], b[2];
            const int ch = 4 * s + 2 * hi;
            auto chunk = [&](const char* base, int row, int c) { return *(const uint4*)(base + row * 128 + ((c ^ ((row >> 1) & 7)) << 4)); };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i].set(chunk(sA, wm + 32 * i + l31, ch), chunk(sA, wm + 32 * i + l31, ch + 1));
                b[i].set(chunk(sB, wn + 32 * i + l31, ch), chunk(sB, wn + 32 * i + l31, ch + 1));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma64<In>(a[i], b[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + wm + 32 * i + 8 * (r >> 2) + 4 * hi + (r & 3), n = n0 + wn + 32 * j + l31;
                if (m < p.M && n < p.N) epilogue<Eo>(p, m, n, acc[i][j][r]);
            }
}

template <class In, class Eo> int launch(const LinArgs& p, hipStream_t stream) {
    const int64_t tm = (p.M + 127) / 128, tn = (p.N + 127) / 128;
    if (tm * tn > 0x7fffffff) return SVD_EINVAL;
    hipLaunchKernelGGL((linear_any_kernel<In, Eo>), dim3((unsigned)(tm * tn)), dim3(256), 0, stream, p, (int)tn);
    SVD_CHECK_LAUNCH("linear_act");
    return SVD_OK;
}

}  // namespace

extern "C" int svd_linear_act(const void* X, int64_t ldx, const void* W, int64_t ldw, const float* xscale, const float* wscale, const float* bias,
                              const void* R, int64_t ldr, void* Y, int64_t ldy, int64_t M, int32_t N, int32_t K, int32_t act, int32_t flags,
                              int32_t in_dtype, int32_t dtype, svd_stream_t stream) {
    const int es = in_dtype == SVD_DTYPE_F8 ? 1 : 2;
    if (!X || !W || !Y || M < 0 || M > 0x7fffff00 || N < 1 || N > 0x7fffff00 || K < 1 || K > 0x3fffff00 || ldx < K || ldw < K || ldy < N || (R && ldr < N)) return SVD_EINVAL;
    if (act < SVD_ACT_NONE || act > SVD_ACT_SILU || (flags & ~(SVD_LIN_RES_F32 | SVD_LIN_OUT_F32)) || (!R && (flags & SVD_LIN_RES_F32))) return SVD_EINVAL;
    if (dtype != SVD_DTYPE_BF16 && dtype != SVD_DTYPE_F16) return SVD_EINVAL;
    if (in_dtype != SVD_DTYPE_F8 && in_dtype != dtype) return SVD_EINVAL;
    if (in_dtype != SVD_DTYPE_F8 && (xscale || wscale)) return SVD_EINVAL;
    const uintptr_t f4 = (uintptr_t)xscale | (uintptr_t)wscale | (uintptr_t)bias | ((flags & SVD_LIN_RES_F32) ? (uintptr_t)R : 0) | ((flags & SVD_LIN_OUT_F32) ? (uintptr_t)Y : 0);
    const uintptr_t f2 = (es == 2 ? (uintptr_t)X | (uintptr_t)W : 0) | (uintptr_t)R | (uintptr_t)Y;
    if ((f4 & 3) || (f2 & 1)) return SVD_EINVAL;
    if (M == 0) return SVD_OK;
    const LinArgs p = {(const char*)X, ldx * es, (const char*)W, ldw * es, xscale, wscale, bias, R, ldr, Y, ldy, (int)M, N, K * es, act,
                       !!(flags & SVD_LIN_RES_F32), !!(flags & SVD_LIN_OUT_F32)};
    if (in_dtype == SVD_DTYPE_F16) return launch<InF16, ElemF16>(p, (hipStream_t)stream);
    if (in_dtype == SVD_DTYPE_BF16) return launch<InBF16, ElemBF16>(p, (hipStream_t)stream);
    if (p.out_f32) return dtype == SVD_DTYPE_F16 ? launch<InF8Wide, ElemF16>(p, (hipStream_t)stream) : launch<InF8Wide, ElemBF16>(p, (hipStream_t)stream);
    return dtype == SVD_DTYPE_F16 ? launch<InF8, ElemF16>(p, (hipStream_t)stream) : launch<InF8, ElemBF16>(p, (hipStream_t)stream);
}
