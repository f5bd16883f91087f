// RMS norm with the residual's addition, 16-bit or e4m3 output (gfx950).
//   s = x (+ r);   y = s * gamma / sqrt(mean(s^2) + eps);   e4m3: a = max |y| / 448 per row, q = rn8(y / a).
// The sum, the mean square and the row maximum are fp32; s is rounded once (to the stream's type), y once (to 16 bits or to e4m3 after the division by a).
#include "svd_common.h"

namespace {

constexpr float F8_MAX = 448.f;              // largest finite e4m3

// The row's scale.  A row of zeros has scale 0 and values 0; a row whose square sum is not finite (an Inf or NaN in it, or |s| beyond 1e19) has scale NaN
// and values NaN, so that it cannot pass for numbers.  |y * inv| <= 448 (1 + 2^-22) rounds to at most 448: no clamp (which would swallow a NaN).
__device__ __forceinline__ float f8_scale(float row_max, float square_sum) { return square_sum < INFINITY ? row_max / F8_MAX : NAN; }
__device__ __forceinline__ float f8_inv(float a) { return a == 0.f ? 0.f : 1.f / a; }

// One workgroup per row, any width: three passes over the row (square sum, maximum, result); the second and third read from the L2.
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
        const float ss = red[0] + red[1] + red[2] + red[3];
        const float rstd = 1.f / sqrtf(ss / (float)channels + eps);
        float inv = 1.f;
        if constexpr (F8) {
            float mx = 0.f;
            for (int c = tid; c < channels; c += 256) mx = fmaxf(mx, fabsf(at(row, c) * (gamma ? gamma[c] * rstd : rstd)));
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
            const float y = v * (gamma ? gamma[c] * rstd : rstd);
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

}  // namespace

extern "C" int svd_rmsnorm(const void* X, int64_t ldx, const void* R, int64_t ldr, const float* gamma, float eps, void* Y, int64_t ldy, float* yscale,
                           void* S, int64_t lds, int64_t rows, int32_t channels, int32_t flags, int32_t dtype, svd_stream_t stream) {
    const bool x32 = flags & SVD_RMS_X_F32, r32 = flags & SVD_RMS_R_F32, f8 = flags & SVD_RMS_OUT_F8;
    if (!X || !Y || rows < 0 || channels < 1 || ldx < channels || ldy < channels || (flags & ~7) || !(eps >= 0.f)) return SVD_EINVAL;
    if ((R && ldr < channels) || (S && (!R || lds < channels)) || (!R && r32) || (f8 && !yscale)) return SVD_EINVAL;
    if (((uintptr_t)X & (x32 ? 3 : 1)) || ((uintptr_t)R & (r32 ? 3 : 1)) || ((uintptr_t)S & (r32 ? 3 : 1)) || (!f8 && ((uintptr_t)Y & 1)) || ((uintptr_t)gamma & 3) || ((uintptr_t)yscale & 3)) return SVD_EINVAL;
    if (dtype != SVD_DTYPE_BF16 && dtype != SVD_DTYPE_F16) return SVD_EINVAL;
    if (rows == 0) return SVD_OK;
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
