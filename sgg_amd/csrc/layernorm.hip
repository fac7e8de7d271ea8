// Layer normalisation over the last axis, forward and backward (f32 / bf16 / f16 rows, fp32 weight, bias, statistics and sums).
//   mu = sum_j x_j / C,  v = sum_j (x_j - mu)^2 / C,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean_j g - xh mean_j(g xh)),  dw_j = sum_i dy_ij xh_ij,  db_j = sum_i dy_ij
// The variance is summed from the centred values (x - mu), never as E[x^2] - mu^2: rows far from zero lose nothing.
#include "common.h"

namespace {

constexpr int LN_ROWS = 256;        // rows of one partial sum of dw / db

template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w, const float* __restrict__ b,
                                                     T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, long M, int C, float eps) {
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    const T* xr = x + row * ldx;
    float s = 0.f;
    for (int c = lane; c < C; c += 64) s += Elem<T>::ld(xr + c);
    const float mu = wave_sum(s) / (float)C;
    s = 0.f;
    for (int c = lane; c < C; c += 64) {
        const float d = Elem<T>::ld(xr + c) - mu;
        s = fmaf(d, d, s);
    }
    const float r = 1.0f / sqrtf(wave_sum(s) / (float)C + eps);
    for (int c = lane; c < C; c += 64) {
        const float xh = (Elem<T>::ld(xr + c) - mu) * r;
        Elem<T>::st(y + row * C + c, fmaf(xh, w ? w[c] : 1.f, b ? b[c] : 0.f));
    }
    if (lane == 0 && mean) {
        mean[row] = mu;
        rstd[row] = r;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_dx_kernel(const T* __restrict__ dy, long ld_dy, const T* __restrict__ x, long ldx, const float* __restrict__ w,
                                                    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx, long M, int C) {
    const int lane = threadIdx.x & 63;
    const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    const T *xr = x + row * ldx, *gr = dy + row * ld_dy;
    const float mu = mean[row], r = rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int c = lane; c < C; c += 64) {
        const float g = Elem<T>::ld(gr + c) * (w ? w[c] : 1.f), xh = (Elem<T>::ld(xr + c) - mu) * r;
        s1 += g;
        s2 = fmaf(g, xh, s2);
    }
    s1 = wave_sum(s1) / (float)C;
    s2 = wave_sum(s2) / (float)C;
    for (int c = lane; c < C; c += 64) {
        const float g = Elem<T>::ld(gr + c) * (w ? w[c] : 1.f), xh = (Elem<T>::ld(xr + c) - mu) * r;
        Elem<T>::st(dx + row * C + c, r * (g - s1 - xh * s2));
    }
}

// partial sums of dw / db over LN_ROWS rows: thread = (column of 64, every 4th row)
template <typename T>
__global__ __launch_bounds__(256) void ln_dw_kernel(const T* __restrict__ dy, long ld_dy, const T* __restrict__ x, long ldx, const float* __restrict__ mean,
                                                    const float* __restrict__ rstd, float* __restrict__ ws, long M, int C) {
    __shared__ float red[2][256];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63);
    const long r0 = (long)blockIdx.y * LN_ROWS, r1 = min(M, r0 + LN_ROWS);
    float a = 0.f, b = 0.f;
    if (c < C)
        for (long row = r0 + (threadIdx.x >> 6); row < r1; row += 4) {
            const float g = Elem<T>::ld(dy + row * ld_dy + c);
            a = fmaf(g, (Elem<T>::ld(x + row * ldx + c) - mean[row]) * rstd[row], a);
            b += g;
        }
    red[0][threadIdx.x] = a;
    red[1][threadIdx.x] = b;
    __syncthreads();
    if (threadIdx.x < 64 && c < C) {
        float* o = ws + (long)blockIdx.y * 2 * C;
        const int t = threadIdx.x;
        o[c] = (red[0][t] + red[0][t + 64]) + (red[0][t + 128] + red[0][t + 192]);
        o[C + c] = (red[1][t] + red[1][t + 64]) + (red[1][t + 128] + red[1][t + 192]);
    }
}

__global__ __launch_bounds__(256) void ln_dw_sum_kernel(const float* __restrict__ ws, int parts, int C, float* __restrict__ dw, float* __restrict__ db) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= 2 * C) return;
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += ws[(long)p * 2 * C + c];
    float* o = c < C ? dw : db;
    if (o) o[c < C ? c : c - C] = s;
}

bool ln_args_ok(int64_t M, int C, int64_t ld) { return M >= 0 && C >= 1 && C <= SGG_LAYER_NORM_MAX && ld >= C && M < (int64_t)1 << 31; }

}  // namespace

extern "C" int sgg_layer_norm_fwd(const void* x, int64_t ldx, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t M, int C,
                                  float eps, int dtype, void* stream) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (!ln_args_ok(M, C, ldx) || !(eps > 0.f) || !mean != !rstd) return SGG_ERR_ARG;
    if (M == 0) return SGG_OK;
    if (!x || !y) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL(ln_fwd_kernel<T>, dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, (const T*)x, (long)ldx, w, b, (T*)y, mean,
                                            rstd, (long)M, C, eps));
    SGG_CHECK_LAUNCH();
    return SGG_OK;
}

extern "C" int sgg_layer_norm_bwd_parts(int64_t M, int C, int dtype) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (!ln_args_ok(M, C, C)) return SGG_ERR_ARG;
    return (int)((M + LN_ROWS - 1) / LN_ROWS);
}

extern "C" int sgg_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ldx, const float* w, const float* mean, const float* rstd, void* dx,
                                  float* dw, float* db, float* ws, int64_t M, int C, int dtype, void* stream) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (!ln_args_ok(M, C, ldx) || ld_dy < C) return SGG_ERR_ARG;
    const bool want_w = dw || db;
    if (M > 0 && (!dy || !x || !mean || !rstd || (want_w && !ws))) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    const int parts = sgg_layer_norm_bwd_parts(M, C, dtype);
    if (M > 0 && dx) {
        SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL(ln_dx_kernel<T>, dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, (const T*)dy, (long)ld_dy, (const T*)x,
                                                (long)ldx, w, mean, rstd, (T*)dx, (long)M, C));
        SGG_CHECK_LAUNCH();
    }
    if (want_w) {
        if (M > 0) {
            SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL(ln_dw_kernel<T>, dim3((C + 63) / 64, parts), dim3(256), 0, s, (const T*)dy, (long)ld_dy, (const T*)x,
                                                    (long)ldx, mean, rstd, ws, (long)M, C));
            SGG_CHECK_LAUNCH();
        }
        hipLaunchKernelGGL(ln_dw_sum_kernel, dim3((2 * C + 255) / 256), dim3(256), 0, s, ws, parts, C, dw, db);
        SGG_CHECK_LAUNCH();
    }
    return SGG_OK;
}
