// Layer normalisation over the last axis, forward and backward (f32 / bf16 / f16 rows, fp32 weight, bias, statistics and sums).
//   mu = sum_j x_j / C,  v = sum_j (x_j - mu)^2 / C,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean_j g - xh mean_j(g xh)),  dw_j = sum_i dy_ij xh_ij,  db_j = sum_i dy_ij
// Rows far from zero lose nothing: the mean comes from a sum without fp32's rounding (LnSum) and is subtracted as two floats -- an fp32 sum's error, a
// few 2^-24 of the MEAN, would enter every x - mu and be multiplied by r, up to 316: constant rows of 1e6 came out 1.0 from 0 --, the variance
// is summed from the centred values, never as E[x^2] - mu^2, and the backward, which gets the mean as one float, centres once more by the mean of what is left.
//
// Memory-bound both ways (8 .. 24 operations per element against 4 .. 12 bytes), so every row is read once and stays in registers between its
// sums and its result, and a workgroup walks many rows: w, b -- 8 bytes per column, twice a 16-bit row's -- and the column sums of dw, db live in
// registers over all of them, and the next row's loads are in flight while this one is reduced.  A lane owns pieces of 8 consecutive columns.  How many
// lanes share a row follows from C alone (LnShape): 8 .. 64 lanes of one wave up to 512 columns (several rows per wave: short rows would
// leave lanes idle), then 1 .. 16 waves with two pieces per lane, which is what the registers of the backward hold.
// Measured (a copy reaches 4.9 TB/s), the backward with the join of its column sums, 4 .. 7 us: 65536 x 4096 bf16 forward 197 us (5.5 TB/s), backward 308 us
// (5.2); 12345 x 1001 f32 19 and 35 us (5.2, 4.3); 7936 x 512 f16, 8 MB, 5.6 and 11.7 us; one row of 512 2 us.
// Rows of any alignment are loaded 16 bytes at a time (this chip's global loads need no alignment); only a row's last, partial piece goes
// element by element.
#include <type_traits>

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

// v of another lane, by DPP (lanes that `rmask` leaves out get 0)
template <int CTRL, int RMASK = 0xF> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, RMASK, 0xF, false));
}
template <int CTRL, int RMASK = 0xF> __device__ __forceinline__ double dpp(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, RMASK, 0xF, false),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, RMASK, 0xF, false));
}
__device__ __forceinline__ float lane63(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ __forceinline__ double lane63(double v) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}
// sum over each W neighbouring lanes (a power of two); every one of them gets it
template <int W, typename F> __device__ __forceinline__ F lanes_sum(F v) {
    if constexpr (W >= 2) v += dpp<0xB1>(v);                     // quad_perm [1,0,3,2]
    if constexpr (W >= 4) v += dpp<0x4E>(v);                     // quad_perm [2,3,0,1]
    if constexpr (W >= 8) v += dpp<0x141>(v);                    // row_half_mirror
    if constexpr (W >= 16) v += dpp<0x140>(v);                   // row_mirror
    if constexpr (W == 32) v += __shfl_xor(v, 16, 64);
    if constexpr (W == 64) {
        v += dpp<0x142, 0xA>(v);                                 // row_bcast15 into rows 1, 3
        v += dpp<0x143, 0xC>(v);                                 // row_bcast31 into rows 2, 3: lane 63 holds the sum
        v = lane63(v);
    }
    return v;
}

// N sums at once over the lanes of a row; every lane of the row gets them.  red: N x WAVES values of LDS that no call one barrier earlier or later uses (no
// lane can be two barriers ahead of another)
template <typename S, int N, typename F>
__device__ __forceinline__ void row_sums(F (&v)[N], F* red) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lanes_sum<S::LPR>(v[k]);
    if constexpr (S::WPR > 1) {                                  // (LPR = 64: one value per wave)
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) red[k * S::WAVES + wave] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = lanes_sum<S::WPR>(red[k * S::WAVES + wave / S::WPR * S::WPR + lane % S::WPR]);
    }
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

// The type a row's sum is held in.  Values of 16 bits that lie within a factor 4 add up in fp32 without any rounding: 8 (bf16) or 11 significand bits,
// 2 for the factor, 14 or 11 for as many columns, 24 in all; and where a row is wider than a factor 4, its spread is max|x| / sqrt(2 C) or more and
// fp32's rounding, 6e-7 max|x|, nothing beside it.  All others take 64 bits (65536 x 4096 bf16 in 64 bits: 201 us, 197 this way;
// 100000 x 200 f16 20.3 and 17.7).
template <typename T, int CAP> struct LnSum { using type = double; };
template <int CAP> struct LnSum<bf16_t, CAP> { using type = float; };
template <int CAP> struct LnSum<f16_t, CAP> { using type = std::conditional_t<(CAP <= 2048), float, double>; };
constexpr float LN_TINY = 0x1p-80f;

// the mean as two floats from the sum: the quotient itself (of a constant row the constant), and what its rounding leaves
__device__ __forceinline__ void ln_mean(double s, double C, double invC, float& mu, float& rest) {
    double m = s * invC;
    m = fma(fma(-m, C, s), invC, m);
    mu = (float)m;
    rest = (float)(m - (double)mu);
}
__device__ __forceinline__ void ln_mean(float s, float C, float invC, float& mu, float& rest) {
    mu = s * invC;
    mu = fmaf(fmaf(-mu, C, s), invC, mu);
    rest = fmaf(-mu, C, s) * invC;
}

template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS) void ln_fwd_kernel(const T* __restrict__ x, long ldx, const float* __restrict__ w, const float* __restrict__ b,
                                                            T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd, long M, int C, float eps) {
    using Sum = typename LnSum<T, S::CAP>::type;
    __shared__ Sum red_mean[S::WAVES];
    __shared__ float red_var[2][S::WAVES];
    const LnLane<S> at(C);
    float wv[S::NV][8], bv[S::NV][8];
    load_columns(w, at, 1.f, wv);
    load_columns(b, at, 0.f, bv);
    const long step = (long)gridDim.x * S::GROUPS;
    const Sum invC = (Sum)1 / (Sum)C;
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
        Sum sum[1] = {};
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            if (at.n[i] > 0) p[i].get(v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] = j < at.n[i] ? v[i][j] : 0.f;
                sum[0] += (Sum)v[i][j];
            }
        }
        if (row0 + step < M) {                                    // the next row's loads
            const T* xr = x + min(row + step, M - 1) * ldx;
#pragma unroll
            for (int i = 0; i < S::NV; ++i)
                if (at.n[i] > 0) p[i].load(xr + at.col[i], at.n[i]);
        }
        row_sums<S>(sum, red_mean);
        float mu, rest;
        ln_mean(sum[0], (Sum)C, invC, mu, rest);
        float sq[1] = {0.f};
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] = j < at.n[i] ? (v[i][j] - mu) - rest : 0.f;
                sq[0] = fmaf(v[i][j], v[i][j], sq[0]);
            }
        row_sums<S>(sq, red_var[0]);
        float r = 1.0f / sqrtf(sq[0] * (float)invC + eps);
        if constexpr (!std::is_same_v<T, f16_t>) {
            // differences past 2^57 or so, whose squares fp32 does not hold: once more, scaled (eps is nothing beside them).  Every lane of a wave, and of
            // a workgroup whose waves share rows, has to come along
            bool again = __any(r == 0.f);
            if constexpr (S::WPR > 1 && S::GROUPS > 1)
#pragma unroll
                for (int g = 0; g < S::WAVES; g += S::WPR) {
                    float t = 0.f;
#pragma unroll
                    for (int i = 0; i < S::WPR; ++i) t += red_var[0][g + i];
                    again = again || __builtin_isinf(t);
                }
            if (again) {
                float tq[1] = {0.f};
#pragma unroll
                for (int i = 0; i < S::NV; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) tq[0] = fmaf(v[i][j] * LN_TINY, v[i][j] * LN_TINY, tq[0]);
                row_sums<S>(tq, red_var[1]);
                if (r == 0.f) r = LN_TINY / sqrtf(tq[0] * (float)invC);
            }
        }
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

// dx and this workgroup's column sums of dw, db (ws[block][2][C]); DX / DW: which of the two are wanted.  With u = (x - mean) r and a = mean_j u (what the
// mean's rounding to a float has left): xh = u - a, mean_j(g xh) = mean_j(g u) - a mean_j g, all of a row's sums in one go
template <typename T, typename S, bool DX, bool DW>
__global__ __launch_bounds__(S::THREADS) void ln_bwd_kernel(const T* __restrict__ dy, long ld_dy, const T* __restrict__ x, long ldx,
                                                            const float* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            T* __restrict__ dx, float* __restrict__ ws, long M, int C) {
    __shared__ float red[2][3 * S::WAVES];                    // (rows in turn: one barrier per row)
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
    int odd = 0;
    for (; row0 < M; row0 += step, odd ^= 1) {
        const long row = row0 + at.group;
        const float mu = mu_n, r = r_n;
        float u[S::NV][8], d[S::NV][8];
        float s[DX ? 3 : 1] = {};
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
            if (at.n[i] > 0) {
                px[i].get(u[i]);
                pg[i].get(d[i]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = j < at.n[i] && row < M;             // (a row past the end adds nothing)
                u[i][j] = in ? (u[i][j] - mu) * r : 0.f;
                d[i][j] = in ? d[i][j] : 0.f;
                s[0] += u[i][j];
                if constexpr (DX) {
                    const float g = d[i][j] * wv[i][j];
                    s[1] += g;
                    s[2] = fmaf(g, u[i][j], s[2]);
                }
            }
        }
        if (row0 + step < M) fetch(row + step);
        row_sums<S>(s, red[odd]);
        const float a = s[0] * invC;
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                u[i][j] -= a;
                asm("" : "+v"(d[i][j]));                          // (d w is multiplied again below: kept over the sums, it would spill at 1024 threads)
                if constexpr (DW) {
                    aw[i][j] = fmaf(d[i][j], u[i][j], aw[i][j]);
                    ab[i][j] += d[i][j];
                }
            }
        if constexpr (DX) {
            const float s1 = s[1] * invC, s2 = s[2] * invC - a * s1;
            if (row < M) {
#pragma unroll
                for (int i = 0; i < S::NV; ++i) {
                    float o[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] = r * (d[i][j] * wv[i][j] - s1 - u[i][j] * s2);
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

// workgroups: enough rows for all, at most `waves` waves per CU.  Forward 16 (65536 x 4096 bf16 197 us; 8 waves: 245, 32: 205; f32 496, 492, 417),
// backward 8, whose workgroups each leave a row of partial column sums to join (308 us; 4 waves: 482, 16: 330; 7936 x 512 f16 11.7, 12.2, 13.9)
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
