// RMS norm with the residual's addition, 16-bit or e4m3 output (gfx950).
//   s = x (+ r);   y = s * gamma / sqrt(mean(s^2) + eps);   e4m3: a = max |y| / 448 per row, q = rn8(y / a).
// The sum, the mean square and the row maximum are fp32; s is rounded once (to the stream's type), y once (to 16 bits or to e4m3 after the division by a).
#include "svd_common.h"

namespace {

constexpr float F8_MAX = 448.f;              // largest finite e4m3

// The row's scale.  A row of zeros has scale 0 and values 0; a row with an Inf or NaN in it (or whose sum s overflows) has scale NaN
// and values NaN, so that it cannot pass for numbers.  |y * inv| <= 448 (1 + 2^-22) rounds to at most 448: no clamp (which would swallow a NaN).
// The scale of any other row is at least 2^-126: 1 / a of a smaller one would be infinite.
__device__ __forceinline__ float f8_scale(float row_max, float square_sum) {
    return !(square_sum < INFINITY) ? NAN : row_max == 0.f ? 0.f : fmaxf(row_max / F8_MAX, 0x1p-126f);
}
__device__ __forceinline__ float f8_inv(float a) { return a == 0.f ? 0.f : 1.f / a; }

// Rows wider than 10240 channels, and fp32 x with a 16-bit residual.  One workgroup per row, any width: three passes over the row (square sum, maximum, result); the second and third read from the L2.
// r and s may be the same rows: a thread reads the elements it writes, in every pass, and writes them last.
template <class E, bool X32, bool R32, bool F8>
__global__ __launch_bounds__(256) void rmsnorm_row_kernel(const void* X, int64_t ldx, const void* R, int64_t ldr, const float* __restrict__ gamma, float eps,
                                                          void* Y, int64_t ldy, float* __restrict__ scale, void* S, int64_t lds, int64_t rows, int channels) {
    __shared__ float red[8];
    const int tid = threadIdx.x, wave = tid >> 6;
    auto at = [&](int64_t row, int c) {
        float v = X32 ? ((const float*)X)[row * ldx + c] : E::to_f32(((const uint16_t*)X)[row * ldx + c]);
        if (R) v += R32 ? ((const float*)R)[row * ldr + c] : E::to_f32(((const uint16_t*)R)[row * ldr + c]);
        return v;
    };
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        float sq = 0.f;
        for (int c = tid; c < channels; c += 256) { const float v = at(row, c); sq = fmaf(v, v, sq); }
        sq = wave_sum(sq);
        if ((tid & 63) == 0) red[wave] = sq;
        __syncthreads();
        float ss = red[0] + red[1] + red[2] + red[3];
        const float f = svd_rms_factor(ss, eps);
        if (f != 1.f) {
            __syncthreads();
            sq = 0.f;
            for (int c = tid; c < channels; c += 256) { const float v = at(row, c) * f; sq = fmaf(v, v, sq); }
            sq = wave_sum(sq);
            if ((tid & 63) == 0) red[wave] = sq;
            __syncthreads();
            ss = red[0] + red[1] + red[2] + red[3];
        }
        const float rstd = svd_rms_inv(ss, (float)channels, eps * f * f);
        float inv = 1.f;
        if constexpr (F8) {
            float mx = 0.f;
            for (int c = tid; c < channels; c += 256) mx = fmaxf(mx, fabsf(at(row, c) * f * (gamma ? gamma[c] * rstd : rstd)));
            mx = wave_max(mx);
            if ((tid & 63) == 0) red[4 + wave] = mx;
            __syncthreads();
            mx = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
            const float a = f8_scale(mx, ss);
            inv = f8_inv(a);
            if (tid == 0) scale[row] = a;
        }
        for (int c = tid; c < channels; c += 256) {
            const float v = at(row, c);
            const float y = v * f * (gamma ? gamma[c] * rstd : rstd);
            if constexpr (F8) {
                const float q = y * inv;
                ((uint8_t*)Y)[row * ldy + c] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
            } else {
                ((uint16_t*)Y)[row * ldy + c] = E::from_f32(y);
            }
            if (S) {
                if constexpr (R32) ((float*)S)[row * lds + c] = v;
                else ((uint16_t*)S)[row * lds + c] = E::from_f32(v);
            }
        }
        __syncthreads();
    }
}

// Rows in registers: TPR threads to a row, 8 channels at a time, at most 5 pieces a thread; one read and one write of everything.  x and r are all requested before
// the first is used (up to 240 bytes a thread in flight).  A row of 16 or 64 threads is reduced inside a wave, one of 256 through LDS.
// What bounds it is memory: 115200 x 640, fp16 x onto an fp32 stream, e4m3 out: 152 us, 5.3 TB/s (a large copy: 5.1); 9217 x 1277 bf16 rows of odd width 26 us, 3.6 TB/s.
// One row of 1280 takes 3.3 us, all of it latency.  (The one-row kernel's three passes: 604 and 43 us.)
// AL: 16-byte aligned rows of whole pieces; else pieces of any alignment (the memory pipe takes them, at more lines per access) and a last one element by element.
template <class E, bool F32, bool AL> __device__ __forceinline__ void load8(const void* row, int c, int n, float (&v)[8]) {
    constexpr int EB = F32 ? 4 : 2;
    struct __attribute__((packed, aligned(AL ? 16 : EB))) U { uint32_t w[4]; };
    const char* p = (const char*)row + (int64_t)c * EB;
    if (AL || c + 8 <= n) {
        if constexpr (F32) {
            const U a = *(const U*)p, b = *(const U*)(p + 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = __uint_as_float(a.w[i]); v[4 + i] = __uint_as_float(b.w[i]); }
        } else {
            const U a = *(const U*)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = E::lo(a.w[i]); v[2 * i + 1] = E::hi(a.w[i]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = c + i < n ? (F32 ? ((const float*)row)[c + i] : E::to_f32(((const uint16_t*)row)[c + i])) : 0.f;
    }
}
// KIND 0: 16 bit, 1: fp32, 2: e4m3
template <class E, int KIND, bool AL> __device__ __forceinline__ void store8(void* row, int c, int n, const float (&v)[8]) {
    constexpr int EB = KIND == 1 ? 4 : KIND == 0 ? 2 : 1, W = 2 * EB;
    struct __attribute__((packed, aligned(AL ? (W < 4 ? 8 : 16) : EB))) U { uint32_t w[W < 4 ? W : 4]; };
    char* p = (char*)row + (int64_t)c * EB;
    uint32_t w[W];
    if constexpr (KIND == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (KIND == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = E::pack(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false), true);
    }
    if (AL || c + 8 <= n) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            U u;
#pragma unroll
            for (int j = 0; j < (W < 4 ? W : 4); ++j) u.w[j] = w[i + j];
            *(U*)(p + 4 * i) = u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < n) {
                if constexpr (KIND == 1) ((float*)row)[c + i] = v[i];
                else if constexpr (KIND == 0) ((uint16_t*)row)[c + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
                else ((uint8_t*)row)[c + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
            }
    }
}
// over the TPR threads of a row; red: 4 floats of LDS of their own
template <int TPR, bool MAX> __device__ __forceinline__ float row_reduce(float v, float* red) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) { const float u = __shfl_xor(v, o, 64); v = MAX ? fmaxf(v, u) : v + u; }
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = MAX ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}
template <class E, bool X32, int RM /* 0 no residual, 1 16 bit, 2 fp32 */, bool F8, int TPR, bool AL>
__global__ __launch_bounds__(256) void rmsnorm_vec_kernel(const void* X, int64_t ldx, const void* R, int64_t ldr, const float* __restrict__ gamma, float eps,
                                                          void* Y, int64_t ldy, float* __restrict__ scale, void* S, int64_t lds, int64_t rows, int channels) {
    constexpr int MAXV = 5;
    __shared__ float red[8];
    const int sub = threadIdx.x % TPR;
    const int64_t row0 = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR, row = row0 < rows ? row0 : rows - 1;          // rows behind the last compute it again and store nothing
    const char* xr = (const char*)X + row * ldx * (X32 ? 4 : 2);
    const char* rr = RM ? (const char*)R + row * ldr * (RM == 2 ? 4 : 2) : nullptr;
    float v[MAXV][8], r[MAXV][8];
#pragma unroll
    for (int k = 0; k < MAXV; ++k) {
        const int c = (sub + TPR * k) * 8;
        if (c < channels) {
            load8<E, X32, AL>(xr, c, channels, v[k]);
            if constexpr (RM != 0) load8<E, RM == 2, AL>(rr, c, channels, r[k]);
        }
    }
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < MAXV; ++k)
        if ((sub + TPR * k) * 8 < channels) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (RM != 0) v[k][i] += r[k][i];
                sq = fmaf(v[k][i], v[k][i], sq);
            }
        }
    const bool live = row0 < rows;
    if constexpr (RM != 0)
        if (S && live) {
#pragma unroll
            for (int k = 0; k < MAXV; ++k) {
                const int c = (sub + TPR * k) * 8;
                if (c < channels) store8<E, RM == 2, AL>((char*)S + row * lds * (RM == 2 ? 4 : 2), c, channels, v[k]);
            }
        }
    float ss = row_reduce<TPR, false>(sq, red);
    const float f = svd_rms_factor(ss, eps);
    if (__builtin_expect(f != 1.f, 0)) {          // all threads of the row
        if (TPR > 64) __syncthreads();
        sq = 0.f;
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
            if ((sub + TPR * k) * 8 < channels) {
#pragma unroll
                for (int i = 0; i < 8; ++i) { v[k][i] *= f; sq = fmaf(v[k][i], v[k][i], sq); }
            }
        ss = row_reduce<TPR, false>(sq, red);
    }
    const float rstd = svd_rms_inv(ss, (float)channels, eps * f * f);
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < MAXV; ++k) {
        const int c = (sub + TPR * k) * 8;
        if (c < channels) {
            float g[8];
            if (gamma) load8<E, true, AL>(gamma, c, channels, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[k][i] *= gamma ? g[i] * rstd : rstd;
                if constexpr (F8) mx = fmaxf(mx, fabsf(v[k][i]));
            }
        }
    }
    if constexpr (F8) {
        mx = row_reduce<TPR, true>(mx, red + 4);
        const float a = f8_scale(mx, ss), inv = f8_inv(a);
        if (sub == 0 && live) scale[row] = a;
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] *= inv;
    }
    if (!live) return;
#pragma unroll
    for (int k = 0; k < MAXV; ++k) {
        const int c = (sub + TPR * k) * 8;
        if (c < channels) store8<E, F8 ? 2 : 0, AL>((char*)Y + row * ldy * (F8 ? 1 : 2), c, channels, v[k]);
    }
}

struct NormCall {
    const void* X; int64_t ldx; const void* R; int64_t ldr; const float* gamma; float eps; void* Y; int64_t ldy; float* yscale; void* S; int64_t lds; int64_t rows;
    int channels;
    hipStream_t stream;
};
template <class E, bool X32, int RM, bool F8, int TPR> void launch_vec(const NormCall& n, bool al) {
    const dim3 grid((unsigned)((n.rows + 256 / TPR - 1) / (256 / TPR)));
    if (al) hipLaunchKernelGGL((rmsnorm_vec_kernel<E, X32, RM, F8, TPR, true>), grid, dim3(256), 0, n.stream, n.X, n.ldx, n.R, n.ldr, n.gamma, n.eps, n.Y, n.ldy, n.yscale, n.S, n.lds, n.rows, n.channels);
    else hipLaunchKernelGGL((rmsnorm_vec_kernel<E, X32, RM, F8, TPR, false>), grid, dim3(256), 0, n.stream, n.X, n.ldx, n.R, n.ldr, n.gamma, n.eps, n.Y, n.ldy, n.yscale, n.S, n.lds, n.rows, n.channels);
}
// Threads to a row from its width alone: five pieces a thread at most.  Wider rows, and fp32 x with a 16-bit residual, take the one-row kernel; so do rows whose threads
// would be 2^32 or more, which a launch cannot have.
template <class E, bool X32, int RM, bool F8> bool try_vec(const NormCall& n, bool al) {
    const int tpr = n.channels <= 640 ? 16 : n.channels <= 2560 ? 64 : 256;
    if (n.channels > 10240 || n.rows > 0xffffff00ll / tpr) return false;
    if (tpr == 16) launch_vec<E, X32, RM, F8, 16>(n, al);
    else if (tpr == 64) launch_vec<E, X32, RM, F8, 64>(n, al);
    else launch_vec<E, X32, RM, F8, 256>(n, al);
    return true;
}
template <class E, bool F8> bool try_all(const NormCall& n, bool x32, bool r32, bool al) {
    if (!n.R) return x32 ? try_vec<E, true, 0, F8>(n, al) : try_vec<E, false, 0, F8>(n, al);
    if (x32) return r32 && try_vec<E, true, 2, F8>(n, al);
    return r32 ? try_vec<E, false, 2, F8>(n, al) : try_vec<E, false, 1, F8>(n, al);
}

}  // namespace

extern "C" int svd_rmsnorm(const void* X, int64_t ldx, const void* R, int64_t ldr, const float* gamma, float eps, void* Y, int64_t ldy, float* yscale,
                           void* S, int64_t lds, int64_t rows, int32_t channels, int32_t flags, int32_t dtype, svd_stream_t stream) {
    const bool x32 = flags & SVD_RMS_X_F32, r32 = flags & SVD_RMS_R_F32, f8 = flags & SVD_RMS_OUT_F8;
    if (!X || !Y || rows < 0 || channels < 1 || channels > 0x7fffff00 || ldx < channels || ldy < channels || (flags & ~7) || !(eps >= 0.f)) return SVD_EINVAL;
    if ((R && ldr < channels) || (S && (!R || lds < channels)) || (!R && r32) || (f8 && !yscale)) return SVD_EINVAL;
    if (((uintptr_t)X & (x32 ? 3 : 1)) || ((uintptr_t)R & (r32 ? 3 : 1)) || ((uintptr_t)S & (r32 ? 3 : 1)) || (!f8 && ((uintptr_t)Y & 1)) || ((uintptr_t)gamma & 3) || ((uintptr_t)yscale & 3)) return SVD_EINVAL;
    if (dtype != SVD_DTYPE_BF16 && dtype != SVD_DTYPE_F16) return SVD_EINVAL;
    if (rows == 0) return SVD_OK;
    const NormCall n = {X, ldx, R, ldr, gamma, eps, Y, ldy, yscale, S, lds, rows, channels, (hipStream_t)stream};
    const int64_t by = (ldx * (x32 ? 4 : 2)) | (R ? ldr * (r32 ? 4 : 2) : 0) | (S ? lds * (r32 ? 4 : 2) : 0) | ldy * 2;          // (e4m3 pieces of 8 bytes: ldy * 2 a multiple of 16)
    const bool al = !(channels & 7) && !(by & 15) && !(((uintptr_t)X | (uintptr_t)R | (uintptr_t)S | (uintptr_t)gamma) & 15) && !((uintptr_t)Y & (f8 ? 7 : 15));
    bool done = false;
    SVD_DISPATCH_DTYPE(dtype, done = f8 ? try_all<E, true>(n, x32, r32, al) : try_all<E, false>(n, x32, r32, al));
    if (done) {
        SVD_CHECK_LAUNCH("rmsnorm");
        return SVD_OK;
    }
    const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
#define LAUNCH(X32, R32, F8) hipLaunchKernelGGL((rmsnorm_row_kernel<E, X32, R32, F8>), dim3(grid), dim3(256), 0, (hipStream_t)stream, X, ldx, R, ldr, gamma, eps, Y, ldy, yscale, S, lds, rows, channels)
#define LAUNCH_F8(X32, R32) do { if (f8) LAUNCH(X32, R32, true); else LAUNCH(X32, R32, false); } while (0)
    SVD_DISPATCH_DTYPE(dtype, {
        if (x32 && r32) LAUNCH_F8(true, true);
        else if (x32) LAUNCH_F8(true, false);
        else if (r32) LAUNCH_F8(false, true);
        else LAUNCH_F8(false, false);
    });
#undef LAUNCH_F8
#undef LAUNCH
    SVD_CHECK_LAUNCH("rmsnorm");
    return SVD_OK;
}
