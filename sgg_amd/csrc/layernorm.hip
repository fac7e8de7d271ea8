// Layer normalisation over the last axis, forward and backward (f32 / bf16 / f16 rows, fp32 weight, bias, statistics and sums).
//   mu = sum_j x_j / C,  v = sum_j (x_j - mu)^2 / C,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean_j g - xh mean_j(g xh)),  dw_j = sum_i dy_ij xh_ij,  db_j = sum_i dy_ij
// The variance is summed from the centred values (x - mu), never as E[x^2] - mu^2: rows far from zero lose nothing.
//
// Memory-bound both ways (8 .. 24 operations per element against 4 .. 12 bytes), so every row is read once and stays in registers between its
// sums and its result, and a workgroup walks many rows: w, b -- 8 bytes per column, twice a 16-bit row's -- and the column sums of dw, db live in
// registers over all of them, and the next row's loads are in flight while this one is reduced.  A lane owns pieces of 8 consecutive columns.  How many
// lanes share a row follows from C alone (LnShape): 8 .. 64 lanes of one wave up to 512 columns (several rows per wave: short rows would
// leave lanes idle), then 1 .. 16 waves with two pieces per lane, which is what the registers of the backward hold.
// Measured (a copy reaches 4.9 TB/s): 65536 x 4096 bf16 forward 194 us (5.5 TB/s), backward 334 us (4.8); 12345 x 1001 f32 20 and 27 us (4.9, 5.4);
// 7936 x 512 f16, 8 MB, 7 and 9 us; the join of the column sums 4 .. 7 us; one row of 512 2 us.
// Rows of any alignment are loaded 16 bytes at a time (this chip's global loads need no alignment); only a row's last, partial piece goes
// element by element.
#include "common.h"

namespace {

typedef u32x4 u32x4_any __attribute__((aligned(2)));       // 16 bytes at the alignment of an element
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// 8 elements as they lie; n of them are there
template <typename T> struct Piece {
    u32x4 r;
    __device__ __forceinline__ void load(const T* p, int n) {
        if (n == 8) {
            r = *reinterpret_cast<const u32x4_any*>(p);
        } else {
            unsigned h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = j < n ? (unsigned)reinterpret_cast<const unsigned short*>(p)[j] : 0u;
            r = u32x4{h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16};
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { unpack8<T>(r, v); }
    static __device__ __forceinline__ void store(T* p, const float (&v)[8], int n) {
        const u32x4 q = pack8<T>(v);
        if (n == 8) {
            *reinterpret_cast<u32x4_any*>(p) = q;
        } else {
            const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) reinterpret_cast<unsigned short*>(p)[j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
        }
    }
};
template <> struct Piece<float> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* p, int n) {
        if (n == 8) {
            a = *reinterpret_cast<const f32x4_any*>(p);
            b = *reinterpret_cast<const f32x4_any*>(p + 4);
        } else {
            float h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = j < n ? p[j] : 0.f;
            a = f32x4{h[0], h[1], h[2], h[3]};
            b = f32x4{h[4], h[5], h[6], h[7]};
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&v)[8], int n) {
        if (n == 8) {
            *reinterpret_cast<f32x4_any*>(p) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_any*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) p[j] = v[j];
        }
    }
};

// LPR lanes of a wave (a power of two) and WPR waves share a row (WPR > 1: LPR = 64), NV pieces per lane
template <int LPR_, int WPR_, int NV_>
struct LnShape {
    static constexpr int LPR = LPR_, WPR = WPR_, NV = NV_;
    static constexpr int WAVES = WPR > 4 ? WPR : 4, THREADS = 64 * WAVES;
    static constexpr int GROUPS = WPR > 1 ? WAVES / WPR : WAVES * (64 / LPR);       // rows a workgroup works on at a time
    static constexpr int CAP = LPR * WPR * NV * 8;                                  // columns
};

// the lane's columns of a per-column vector (fill where there is none)
template <typename L, int NV>
__device__ __forceinline__ void load_columns(const float* p, const L& at, float fill, float (&v)[NV][8]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (p && at.n[i] > 0) {
            Piece<float> q;
            q.load(p + at.col[i], at.n[i]);
            q.get(v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = fill;
        }
    }
}

// sum over the lanes of a row; every lane of the row gets it.  red: WAVES floats of LDS, a set of its own per call inside one row (no lane can be two
// calls ahead of another: the barriers in between)
template <typename S>
__device__ __forceinline__ float row_sum(float v, float* red) {
    if constexpr (S::LPR == 64) {
        v = wave_sum(v);
        if constexpr (S::WPR > 1) {
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) red[wave] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int i = 0; i < S::WPR; ++i) v += red[wave / S::WPR * S::WPR + i];
        }
    } else {
#pragma unroll
        for (int o = S::LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    }
    return v;
}

template <typename S> struct LnLane {
    int group, slot, n[S::NV], col[S::NV];
    __device__ __forceinline__ LnLane(int C) {
        const int t = threadIdx.x;
        group = S::WPR > 1 ? t / (64 * S::WPR) : t / S::LPR;
        slot = S::WPR > 1 ? t % (64 * S::WPR) : t % S::LPR;
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            col[i] = (i * S::LPR * S::WPR + slot) * 8;
            n[i] = min(8, max(0, C - col[i]));
        }
    }
};

template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS) void ln_fwd_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w, const float* __restrict__ b,
                                                            T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, long M, int C, float eps) {
    __shared__ float red[2][S::WAVES];
    const LnLane<S> at(C);
    float wv[S::NV][8], bv[S::NV][8];
    load_columns(w, at, 1.f, wv);
    load_columns(b, at, 0.f, bv);
    const long step = (long)gridDim.x * S::GROUPS;
    const float invC = 1.f / (float)C;
    Piece<T> p[S::NV];
    // every workgroup's trip count is uniform (barriers inside): a group past the last row works on row M - 1 again and stores nothing
    long row0 = (long)blockIdx.x * S::GROUPS;
    if (row0 >= M) return;
    {
        const T* xr = x + min(row0 + at.group, M - 1) * ldx;
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
            if (at.n[i] > 0) p[i].load(xr + at.col[i], at.n[i]);
    }
    for (; row0 < M; row0 += step) {
        const long row = row0 + at.group;
        float v[S::NV][8];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            if (at.n[i] > 0) p[i].get(v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] = j < at.n[i] ? v[i][j] : 0.f;
                s += v[i][j];
            }
        }
        if (row0 + step < M) {                                    // the next row's loads
            const T* xr = x + min(row + step, M - 1) * ldx;
#pragma unroll
            for (int i = 0; i < S::NV; ++i)
                if (at.n[i] > 0) p[i].load(xr + at.col[i], at.n[i]);
        }
        const float mu = row_sum<S>(s, red[0]) * invC;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] = j < at.n[i] ? v[i][j] - mu : 0.f;
                s = fmaf(v[i][j], v[i][j], s);
            }
        const float r = 1.0f / sqrtf(row_sum<S>(s, red[1]) * invC + eps);
        if (row < M) {
#pragma unroll
            for (int i = 0; i < S::NV; ++i) {
                float o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = fmaf(v[i][j] * r, wv[i][j], bv[i][j]);
                if (at.n[i] > 0) Piece<T>::store(y + row * C + at.col[i], o, at.n[i]);
            }
            if (at.slot == 0 && mean) {
                mean[row] = mu;
                rstd[row] = r;
            }
        }
    }
}

// dx and this workgroup's column sums of dw, db (ws[block][2][C]); DX / DW: which of the two are wanted
template <typename T, typename S, bool DX, bool DW>
__global__ __launch_bounds__(S::THREADS) void ln_bwd_kernel(const T* __restrict__ dy, long ld_dy, const T* __restrict__ x, long ldx,
                                                            const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            T* __restrict__ dx, float* __restrict__ ws, long M, int C) {
    __shared__ float red[2][S::WAVES];
    __shared__ float fold[DW && S::GROUPS > 1 ? S::GROUPS * S::CAP : 1];
    const LnLane<S> at(C);
    float wv[S::NV][8], aw[S::NV][8] = {}, ab[S::NV][8] = {};
    load_columns(w, at, 1.f, wv);
    const long step = (long)gridDim.x * S::GROUPS;
    const float invC = 1.f / (float)C;
    Piece<T> px[S::NV], pg[S::NV];
    float mu_n, r_n;
    auto fetch = [&](long row) {
        row = min(row, M - 1);
        const T *xr = x + row * ldx, *gr = dy + row * ld_dy;
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
            if (at.n[i] > 0) {
                px[i].load(xr + at.col[i], at.n[i]);
                pg[i].load(gr + at.col[i], at.n[i]);
            }
        mu_n = mean[row];
        r_n = rstd[row];
    };
    long row0 = (long)blockIdx.x * S::GROUPS;
    if (row0 < M) fetch(row0 + at.group);
    for (; row0 < M; row0 += step) {
        const long row = row0 + at.group;
        const float mu = mu_n, r = r_n;
        float xh[S::NV][8], g[S::NV][8];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            if (at.n[i] > 0) {
                px[i].get(xh[i]);
                pg[i].get(g[i]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = j < at.n[i] && row < M;             // (a row past the end adds nothing)
                xh[i][j] = in ? (xh[i][j] - mu) * r : 0.f;
                const float d = in ? g[i][j] : 0.f;
                if constexpr (DW) {
                    aw[i][j] = fmaf(d, xh[i][j], aw[i][j]);
                    ab[i][j] += d;
                }
                if constexpr (DX) {
                    g[i][j] = d * wv[i][j];
                    s1 += g[i][j];
                    s2 = fmaf(g[i][j], xh[i][j], s2);
                }
            }
        }
        if (row0 + step < M) fetch(row + step);
        if constexpr (DX) {
            s1 = row_sum<S>(s1, red[0]) * invC;
            s2 = row_sum<S>(s2, red[1]) * invC;
            if (row < M) {
#pragma unroll
                for (int i = 0; i < S::NV; ++i) {
                    float o[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] = r * (g[i][j] - s1 - xh[i][j] * s2);
                    if (at.n[i] > 0) Piece<T>::store(dx + row * C + at.col[i], o, at.n[i]);
                }
            }
        }
    }
    if constexpr (DW) {
        float* part = ws + (long)blockIdx.x * 2 * C;
#pragma unroll
        for (int h = 0; h < 2; ++h) {                             // dw, then db
            if constexpr (S::GROUPS == 1) {
#pragma unroll
                for (int i = 0; i < S::NV; ++i)
                    if (at.n[i] > 0) Piece<float>::store(part + h * C + at.col[i], h ? ab[i] : aw[i], at.n[i]);
            } else {                                              // the row groups of the workgroup meet in LDS, added in group order
                __syncthreads();
#pragma unroll
                for (int i = 0; i < S::NV; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) fold[at.group * S::CAP + at.col[i] + j] = h ? ab[i][j] : aw[i][j];
                __syncthreads();
                for (int c = threadIdx.x; c < C; c += S::THREADS) {
                    float s = 0.f;
#pragma unroll
                    for (int q = 0; q < S::GROUPS; ++q) s += fold[q * S::CAP + c];
                    part[h * C + c] = s;
                }
            }
        }
    }
}

// column sums of the partials: 16 columns x 16 strided shares of the parts per workgroup, both levels in a fixed order
__global__ __launch_bounds__(256) void ln_dw_sum_kernel(const float* __restrict__ ws, int parts, int C, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float red[16][17];
    const int cl = threadIdx.x & 15, share = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
    float s = 0.f;
    if (c < 2 * C)
#pragma unroll 8
        for (int p = share; p < parts; p += 16) s += ws[(long)p * 2 * C + c];
    red[share][cl] = s;
    __syncthreads();
    if (share == 0 && c < 2 * C) {
#pragma unroll
        for (int p = 1; p < 16; ++p) s += red[p][cl];
        float* o = c < C ? dw : db;
        if (o) o[c < C ? c : c - C] = s;
    }
}

// C -> shape: BODY with S the shape
#define LN_FOR_SHAPE(C, ...)                                                   \
    if ((C) <= 64) { using S = LnShape<8, 1, 1>; __VA_ARGS__; }                \
    else if ((C) <= 128) { using S = LnShape<16, 1, 1>; __VA_ARGS__; }         \
    else if ((C) <= 256) { using S = LnShape<32, 1, 1>; __VA_ARGS__; }         \
    else if ((C) <= 512) { using S = LnShape<64, 1, 1>; __VA_ARGS__; }         \
    else if ((C) <= 1024) { using S = LnShape<64, 1, 2>; __VA_ARGS__; }        \
    else if ((C) <= 2048) { using S = LnShape<64, 2, 2>; __VA_ARGS__; }        \
    else if ((C) <= 4096) { using S = LnShape<64, 4, 2>; __VA_ARGS__; }        \
    else if ((C) <= 8192) { using S = LnShape<64, 8, 2>; __VA_ARGS__; }        \
    else { using S = LnShape<64, 16, 2>; __VA_ARGS__; }

// workgroups: enough rows for all, at most `waves` waves per CU
template <typename S>
int ln_blocks(int64_t M, int waves) {
    const int64_t most = 256 * (int64_t)(waves / S::WAVES > 0 ? waves / S::WAVES : 1);
    const int64_t need = (M + S::GROUPS - 1) / S::GROUPS;
    return (int)(need < most ? need : most);
}
constexpr int LN_FWD_WAVES = 16, LN_BWD_WAVES = 8;

bool ln_args_ok(int64_t M, int C, int64_t ld) { return M >= 0 && C >= 1 && C <= SGG_LAYER_NORM_MAX && ld >= C && M < (int64_t)1 << 31; }

}  // namespace

extern "C" int sgg_layer_norm_fwd(const void* x, int64_t ldx, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t M, int C,
                                  float eps, int dtype, void* stream) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (!ln_args_ok(M, C, ldx) || !(eps > 0.f) || !mean != !rstd) return SGG_ERR_ARG;
    if (M == 0) return SGG_OK;
    if (!x || !y) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    LN_FOR_SHAPE(C, SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL((ln_fwd_kernel<T, S>), dim3(ln_blocks<S>(M, LN_FWD_WAVES)), dim3(S::THREADS), 0, s, (const T*)x,
                                                            (long)ldx, w, b, (T*)y, mean, rstd, (long)M, C, eps)));
    SGG_CHECK_LAUNCH();
    return SGG_OK;
}

extern "C" int sgg_layer_norm_bwd_parts(int64_t M, int C, int dtype) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (!ln_args_ok(M, C, C)) return SGG_ERR_ARG;
    LN_FOR_SHAPE(C, return ln_blocks<S>(M, LN_BWD_WAVES));
}

extern "C" int sgg_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ldx, const float* w, const float* mean, const float* rstd, void* dx,
                                  float* dw, float* db, float* ws, int64_t M, int C, int dtype, void* stream) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (!ln_args_ok(M, C, ldx) || ld_dy < C) return SGG_ERR_ARG;
    const bool want_w = dw || db;
    if (M > 0 && (!dy || !x || !mean || !rstd || (want_w && !ws))) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    const int parts = sgg_layer_norm_bwd_parts(M, C, dtype);
    if (M > 0 && (dx || want_w)) {
#define LN_BWD(DX_, DW_)                                                                                                                              \
    LN_FOR_SHAPE(C, SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL((ln_bwd_kernel<T, S, DX_, DW_>), dim3(parts), dim3(S::THREADS), 0, s, (const T*)dy,          \
                                                            (long)ld_dy, (const T*)x, (long)ldx, w, mean, rstd, (T*)dx, ws, (long)M, C)))
        if (dx && want_w) { LN_BWD(true, true); } else if (dx) { LN_BWD(true, false); } else { LN_BWD(false, true); }
#undef LN_BWD
        SGG_CHECK_LAUNCH();
    }
    if (want_w) {
        hipLaunchKernelGGL(ln_dw_sum_kernel, dim3((2 * C + 15) / 16), dim3(256), 0, s, ws, parts, C, dw, db);
        SGG_CHECK_LAUNCH();
    }
    return SGG_OK;
}
