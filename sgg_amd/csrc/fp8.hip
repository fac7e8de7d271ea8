// Matrix products in 8-bit floating point (OCP e4m3) with a power-of-two scale for each block of 128 along the reduction.
//
// Operand form: row m of a matrix [M][K] is Kp = K rounded up to 128 values of e4m3 (zero past K), laid out in slabs of 64: byte k of row m lies at
// ((k / 64) * R + m) * 64 + k % 64, R = M rounded up to even (the row it adds is zero).  A tile's rows of one slab are one contiguous piece of memory,
// read in whole cache lines; rows Kp apart give half lines (7936 x 4096 x 25088, 16-bit output: 668 us in slabs, 714 in rows; 8192^3: 402 and 432).
// Block b of a row, columns 128 b .. 128 b + 127, has the scale 2^e, e the smallest exponent >= -126 with max|x| <= 448 * 2^e, and q = x 2^-e rounded
// to nearest even: |x - q 2^e| <= 2^-4 |x| down to e4m3's subnormals (2^-10 of the scale).  A power of two because the matrix instruction of this
// chip (v_mfma_scale_f32_*_f8f6f4) multiplies by an e8m0 scale per row and 32 columns itself: dividing by it rounds nothing and applying it costs
// nothing.  Non-finite elements become NaN and do not enter the maximum: the products they take part in are NaN, the rest of the block keeps its scale.
// Scales are bytes (e + 127), 128 rows to a group: byte ((b * G + m / 128) * 32 + m % 32) * 4 + (m / 32) % 4 with G = ceil(M / 128) -- one dword
// holds the rows r, r + 32, r + 64, r + 96 of a group, i.e. what a lane of the 32-row MFMA fragments needs, picked by the instruction's
// byte selector.
#include <atomic>

#include "gemm_args.h"

namespace {

constexpr int QB = 128;             // columns of a block

__host__ __device__ __forceinline__ long slab_rows(long rows) { return (rows + 1) & ~1L; }
__host__ __device__ __forceinline__ long scale_bytes(long rows, long blocks) { return blocks * ((rows + 127) / 128) * 128; }
__device__ __forceinline__ long scale_at(long m, long blk, long groups) { return ((blk * groups + (m >> 7)) * 32 + (m & 31)) * 4 + ((m >> 5) & 3); }

// biased exponent byte of the block whose largest finite magnitude is `top`:  top = 1.f * 2^E; 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_byte(float top) {
    const unsigned t = __float_as_uint(top);
    return max(1, (int)(t >> 23) - 8 + ((t & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ float scale_inv(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }        // 2^-(byte - 127)
__device__ __forceinline__ bool is_inf(float v) { return (__float_as_uint(v) & 0x7fffffffu) == 0x7f800000u; }
__device__ __forceinline__ float not_inf(float v) { return is_inf(v) ? 0.f : fabsf(v); }
__device__ __forceinline__ unsigned pack_fp8x4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// 8 values times inv -> 8 codes; infinities go as NaN (a NaN stays one by itself)
__device__ __forceinline__ u32x2 pack_fp8x8(const float (&v)[8], float inv, bool inf) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = v[j] * inv;
    if (inf) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = is_inf(v[j]) ? __uint_as_float(0x7fc00000u) : q[j];
    }
    return u32x2{pack_fp8x4(q[0], q[1], q[2], q[3]), pack_fp8x4(q[4], q[5], q[6], q[7])};
}
// max over the 16 lanes of a DPP row (values >= 0)
__device__ __forceinline__ float row16_max(float v) {
#define FP8_DPP_MAX(ctrl) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, false)));
    FP8_DPP_MAX(0xB1)   // quad_perm [1,0,3,2]
    FP8_DPP_MAX(0x4E)   // quad_perm [2,3,0,1]
    FP8_DPP_MAX(0x141)  // row_half_mirror
    FP8_DPP_MAX(0x140)  // row_mirror
#undef FP8_DPP_MAX
    return v;
}

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
// 8 elements at any alignment (this chip's 16-byte loads need none)
template <typename T> __device__ __forceinline__ void load8_any(const T* p, float (&v)[8]) {
    const u32x4 q = *reinterpret_cast<const u32x4_any*>(p);
    unpack8<T>(q, v);
}
template <> __device__ __forceinline__ void load8_any<float>(const float* p, float (&v)[8]) {
    const f32x4 a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// One workgroup = a tile of 128 x 128 values; thread (tr, tc) holds rows 8 tr .. 8 tr + 7, columns 8 tc .. 8 tc + 7.  The row form needs the largest
// magnitude of each row of the tile (16 lanes meet), the transposed form that of each column (LDS), the column sums (a bias gradient) one number per
// column: all out of one reading, which is what bounds it (8-byte and 16-byte stores, every line of both outputs written whole).
// Measured: 7936 x 25088 f16 to the row form 115 .. 125 us (600 MB, 4.8 .. 5.2 TB/s: a copy's rate); 7936 x 4096 bf16 to both forms 27 us warm, 33 cold
// (130 MB, 4.8 and 3.9 TB/s); 1985 x 333 f32, rows of no alignment, to both 7 us (element by element 12); one row of 25088 3 us.
// max() drops NaN, so only infinities need a second look: a tile's rows (columns) are gone over again without them where the maximum is infinite.
template <typename T, bool ROWS, bool COLS, bool SUM>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const T* __restrict__ x, long ldx, long M, int K, unsigned char* __restrict__ rows,
                                                           unsigned char* __restrict__ rscale, unsigned char* __restrict__ cols,
                                                           unsigned char* __restrict__ cscale, float* __restrict__ sums, int tilesK) {
    __shared__ __attribute__((aligned(16))) unsigned char tile[COLS ? 128 * 128 : 16];
    __shared__ float cred[COLS ? 16 : 1][128];
    __shared__ unsigned char rbyte[128], cbyte[128], cinf[128];
    const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
    const long tm = blockIdx.x / tilesK;
    const int tk = (int)(blockIdx.x - tm * tilesK);
    const long m0 = tm * 128;
    const int k0 = tk * QB;
    const long RM = slab_rows(M);
    float v[8][8];
    const int left = min(8, K - k0 - tc * 8);
    const T* p0 = x + (m0 + tr * 8) * ldx + k0 + tc * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (m0 + tr * 8 + i < M && left == 8) {
            load8_any(p0 + i * ldx, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
            if (m0 + tr * 8 + i < M)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) v[i][j] = Elem<T>::ld(p0 + i * ldx + j);
        }
    }
    if constexpr (ROWS) {
        auto row_form = [&](int i) {
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[i][j]));
            top = row16_max(top);
            const bool inf = is_inf(top);
            if (inf) {                                            // (all 16 lanes of the row together)
                top = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, not_inf(v[i][j]));
                top = row16_max(top);
            }
            const int byte = scale_byte(top);
            if (m0 + tr * 8 + i < RM)
                *reinterpret_cast<u32x2*>(rows + ((2L * tk + (tc >> 3)) * RM + m0 + tr * 8 + i) * 64 + (tc & 7) * 8) = pack_fp8x8(v[i], scale_inv(byte), inf);
            if (tc == 0) rbyte[tr * 8 + i] = (unsigned char)byte;
        };
        if (COLS || m0 + 128 <= M) {
#pragma unroll
            for (int i = 0; i < 8; ++i) row_form(i);
        } else {                                                  // few rows: nothing done for those past the end, whose blocks are zeros (one row: 4.6 us against 5.2; no gain with COLS)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (m0 + tr * 8 + i < RM) row_form(i);
                else if (tc == 0) rbyte[tr * 8 + i] = (unsigned char)scale_byte(0.f);
        }
    }
    if constexpr (COLS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i][j]));
            cred[tr][tc * 8 + j] = top;
        }
    }
    if constexpr (ROWS || COLS) __syncthreads();
    if constexpr (ROWS)
        if (tid < 32) {
            const long groups = (M + 127) / 128;
            reinterpret_cast<unsigned*>(rscale)[((long)tk * groups + tm) * 32 + tid] =
                rbyte[tid] | (unsigned)rbyte[tid + 32] << 8 | (unsigned)rbyte[tid + 64] << 16 | (unsigned)rbyte[tid + 96] << 24;
        }
    if constexpr (COLS) {
        const long RK = slab_rows(K), groups = ((long)K + 127) / 128;
        if (tid < 128) {
            float top = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, cred[r][tid]);
            cinf[tid] = is_inf(top);
            cbyte[tid] = (unsigned char)scale_byte(top);
        }
        if (__syncthreads_or(tid < 128 && cinf[tid])) {           // some column holds an infinity: the columns' maxima again, without them
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, not_inf(v[i][j]));
                cred[tr][tc * 8 + j] = top;
            }
            __syncthreads();
            if (tid < 128) {
                float top = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, cred[r][tid]);
                cbyte[tid] = (unsigned char)scale_byte(top);
            }
            __syncthreads();
        }
        if (tid < 32)
            reinterpret_cast<unsigned*>(cscale)[(tm * groups + tk) * 32 + tid] =
                cbyte[tid] | (unsigned)cbyte[tid + 32] << 8 | (unsigned)cbyte[tid + 64] << 16 | (unsigned)cbyte[tid + 96] << 24;
        // transposed tile in LDS: column c's 128 bytes, their 8-byte pieces permuted by c / 8 so that neither side's accesses pile up on a bank
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = tc * 8 + j;
            const float t[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
            *reinterpret_cast<u32x2*>(tile + c * 128 + ((tr ^ tc) << 3)) = pack_fp8x8(t, scale_inv(cbyte[c]), cinf[c]);
        }
        if constexpr (SUM) {
#pragma unroll
            for (int j = 0; j < 8; ++j) cred[tr][tc * 8 + j] = ((v[0][j] + v[1][j]) + (v[2][j] + v[3][j])) + ((v[4][j] + v[5][j]) + (v[6][j] + v[7][j]));
        }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int c = p * 32 + (tid >> 3), h = tid & 7, key = c >> 3;               // 16 bytes: pieces 2h and 2h + 1
            const u32x2 a = *reinterpret_cast<const u32x2*>(tile + c * 128 + (((2 * h) ^ key) << 3));
            const u32x2 b = *reinterpret_cast<const u32x2*>(tile + c * 128 + (((2 * h + 1) ^ key) << 3));
            if (k0 + c < RK) *reinterpret_cast<u32x4*>(cols + ((2 * tm + (h >> 2)) * RK + k0 + c) * 64 + (h & 3) * 16) = u32x4{a.x, a.y, b.x, b.y};
        }
        if constexpr (SUM)
            if (tid < 128 && k0 + tid < K) {                      // this tile's 128 rows; the tiles' sums are added in order by the caller
                float t = cred[0][tid];
#pragma unroll
                for (int r = 1; r < 16; ++r) t += cred[r][tid];
                sums[tm * K + k0 + tid] = t;
            }
    }
}

// ---- product: C[m][n] = sum_k A[m][k] W[n][k] (+ bias, ReLU), operands in the form above
//
// Two matrix pipes.  The 8-bit one (v_mfma_scale_f32_32x32x64_f8f6f4, twice the 16-bit rate) adds products in groups of 8 neighbouring columns: each is cut
// (toward zero) at 2^-13 of the power of two at or below the group's largest, a code below e4m3's 2^-6 counting as 2^-6 there; the groups' sums join with
// 24 bits (seen bit by bit; the older 8-bit instructions do the same).  A cut is as large where the sum cancels: it is small beside the terms, not beside the
// output.  Measured against 64 bits for K = 128 .. 25088: 1.2e-5 of the outputs' rms for normal operands, 9e-6 behind a ReLU, 4e-5 for magnitudes spread by
// 2^N(0,1), 1.7e-4 of the root of the squared terms by 2^(3 N(0,1)).  Rounding the output costs up to 4.9e-4 (f16) or 3.9e-3 (bf16) of itself, and 16-bit outputs
// are what this pipe is used for: of 7936 x 4096 bf16 gradients 1.2 % go to the neighbouring value.  An fp32 output gets fp32 sums: e4m3 * 2^e is converted in
// registers to bf16 -- exactly, four significant bits and any exponent -- and multiplied on the bf16 pipe, whose products are whole and whose sums
// round at 2^-24 (2^e * e4m3 below 2^-133 or from 2^128 on leaves bf16's range: 0 / inf).  So do products of up to 32 rows, whatever their output.

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Fp8Args {
    const unsigned char *A, *As, *W, *Ws;
    const float* bias;
    char* C;
    long ldc, Kp;
    int M, N, act, out_dt;
};

__device__ __forceinline__ i32x8 join8(const u32x4& a, const u32x4& b) { return i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w}; }

// byte SEL of a scale dword -> 2^e as fp32 bits (the conversion uses its exponent)
template <int SEL>
__device__ __forceinline__ float scale_f32(unsigned word) { return __uint_as_float(((word >> (8 * SEL)) & 0xffu) << 23); }

// a fragment of the bf16 pipe from one of the 8-bit pipe: the lane's 32 values as 4 x 8
struct Wide { u32x4 c[4]; };
__device__ __forceinline__ Wide widen(const i32x8& v, float scale) {
    Wide w;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        w.c[c].x = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * c], scale, false));
        w.c[c].y = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * c], scale, true));
        w.c[c].z = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * c + 1], scale, false));
        w.c[c].w = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * c + 1], scale, true));
    }
    return w;
}
__device__ __forceinline__ void mma_wide(f32x16& acc, const Wide& w, const Wide& a) {
#pragma unroll
    for (int c = 0; c < 4; ++c) acc = mfma_32x32x16<SGG_BF16>(w.c[c], a.c[c], acc);
}

// ---- where results go: fp32 partial outputs of a K slice ([slice][M][N]), or act(sum + bias) in the output's type

__device__ __forceinline__ void out_st(char* C, long at, int dt, float v) {
    if (dt == SGG_F32) reinterpret_cast<float*>(C)[at] = v;
    else if (dt == SGG_BF16) reinterpret_cast<bf16_t*>(C)[at] = f32_to_bf16(v);
    else reinterpret_cast<f16_t*>(C)[at] = (f16_t)v;
}

// 8 consecutive outputs of a row, nv of them inside (any alignment: this chip's 16-byte stores need none)
__device__ __forceinline__ void out_row8(const Fp8Args& g, const float (&bias8)[8], float (&v)[8], long m, long n, int nv, float* part) {
    if (part) {
        float* o = part + m * g.N + n;
        if (nv == 8) {
            *reinterpret_cast<f32x4_any*>(o) = f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_any*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < nv) o[k] = v[k];
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v[k] += bias8[k];
        if (g.act == SGG_ACT_RELU) v[k] = v[k] < 0.f ? 0.f : v[k];                       // (keeps NaN)
    }
    const long at = m * g.ldc + n;
    if (nv < 8) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < nv) out_st(g.C, at + k, g.out_dt, v[k]);
    } else if (g.out_dt == SGG_F32) {
        float* o = reinterpret_cast<float*>(g.C) + at;
        *reinterpret_cast<f32x4_any*>(o) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_any*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<u32x4_any*>(g.C + at * 2) = g.out_dt == SGG_BF16 ? pack8<bf16_t>(v) : pack8<f16_t>(v);
    }
}

// a wave's 32 MI x 32 NI outputs, from fragments whose lanes hold one row m and 4 consecutive n per register quad, to rows of 8 consecutive n per lane
// through 8.5 KiB of LDS of its own (est; row stride 272 bytes)
constexpr int EST = 32 * 272;
template <int MI, int NI>
__device__ __forceinline__ void out_wave(const Fp8Args& g, f32x16 (&acc)[MI][NI], char* est, long m0, long n0, float* part) {
    constexpr int LN = 4 * NI, ROWS = 64 / LN;                // lanes along a row, rows at a time
    const int lane = threadIdx.x & 63, fr = lane & 31, fh = lane >> 5, rl = lane / LN, cl = (lane % LN) * 8;
    const long n = n0 + cl;
    const int nv = (int)min(8L, max(0L, (long)g.N - n));
    float bias8[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bias8[k] = g.bias && !part && k < nv ? g.bias[n + k] : 0.f;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<f32x4*>(est + fr * 272 + (ni * 32 + 8 * c + 4 * fh) * 4) =
                    f32x4{acc[mi][ni][4 * c], acc[mi][ni][4 * c + 1], acc[mi][ni][4 * c + 2], acc[mi][ni][4 * c + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                               // (its own writes: no other wave reads them)
#pragma unroll
        for (int it = 0; it < 32 / ROWS; ++it) {
            const long m = m0 + mi * 32 + rl + ROWS * it;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(est + (rl + ROWS * it) * 272 + cl * 4);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(est + (rl + ROWS * it) * 272 + cl * 4 + 16);
            float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            if (m < g.M && nv > 0) out_row8(g, bias8, v, m, n, nv, part);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// the K slices' partial outputs, added in slice order; then bias, activation and the output's rounding
__global__ __launch_bounds__(256) void fp8_join_kernel(const Fp8Args g, const float* __restrict__ ws, int slices) {
    const long n = ((long)blockIdx.x * 64 + (threadIdx.x & 63)) * 8;
    if (n >= g.N) return;
    const int nv = (int)min(8L, (long)g.N - n);
    float bias8[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bias8[k] = g.bias && k < nv ? g.bias[n + k] : 0.f;
    for (long m = (long)blockIdx.y * 4 + (threadIdx.x >> 6); m < g.M; m += (long)gridDim.y * 4) {
        float v[8] = {};
        const float* p = ws + m * g.N + n;
#pragma unroll 4
        for (int s = 0; s < slices; ++s, p += (long)g.M * g.N) {
            if (nv == 8) {
                const f32x4 a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w; v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < nv) v[k] += p[k];
            }
        }
        out_row8(g, bias8, v, m, n, nv, nullptr);
    }
}

// Workgroup -> (tile, K slice).  One-dimensional grid of tiles x slices; consecutive logical ids run on one XCD (its own L2): a slice's tiles together, so that
// the slice's columns of A are fetched into one L2 once and not into all eight.
__device__ __forceinline__ void tile_and_slice(int tilesM, int tilesN, int& tm, int& tn, int& slice) {
    const int tiles = tilesM * tilesN, logical = xcd_remap(blockIdx.x, gridDim.x);
    slice = logical / tiles;
    // inside a slice, columns of 4 tiles of M at a time (4, 6 and 8 within 1 %)
    constexpr int GM = 4;
    const int t = logical - slice * tiles, first = t / (GM * tilesN) * GM, h = min(GM, tilesM - first), in = t - first * tilesN;
    tm = first + in % h;
    tn = in / h;
}

// ---- (1) up to 32 rows of A: a stream of W.  Bound by reading W once (its bytes / the memory's rate); everything else hides behind that.  A workgroup
// owns 32 rows of W and a K slice, its 4 waves take the slice's blocks in turn (four neighbouring 128-byte pieces of every row are in flight together)
// straight into registers, DEPTH blocks ahead of their use; the waves' sums meet in LDS.  Always the bf16 pipe: the conversions are a tenth of the
// time W takes to arrive.  32 x 4096 x 25088: 22.1 us (4.7 TB/s of W) with its join.
template <int DEPTH>
__global__ __launch_bounds__(256) void fp8_few_rows_kernel(const Fp8Args g, float* __restrict__ ws, int per, int slices) {
    __shared__ float red[4][32 * 33];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 31, fh = lane >> 5;
    const int slice = blockIdx.x % slices;
    const long n0 = (long)(blockIdx.x / slices) * 32;
    const int blocks = (int)(g.Kp / 128), b0 = min(slice * per, blocks), b1 = min(b0 + per, blocks);
    const long gA = ((long)g.M + 127) / 128, gW = ((long)g.N + 127) / 128;
    const long RA = slab_rows(g.M) * 64, RW = slab_rows(g.N) * 64;
    const unsigned char* wp = g.W + min(n0 + fr, (long)g.N - 1) * 64 + fh * 16;
    const unsigned char* ap = g.A + (long)min(fr, g.M - 1) * 64 + fh * 16;
    const unsigned* sw = reinterpret_cast<const unsigned*>(g.Ws) + (n0 >> 7) * 32 + fr;
    const unsigned* sa = reinterpret_cast<const unsigned*>(g.As) + fr;
    const int shift = (int)(n0 >> 5 & 3) * 8;
    struct { u32x4 w[4], a[4]; unsigned ew, ea; } buf[DEPTH];
    auto fetch = [&](auto& t, int b) {
#pragma unroll
        for (int c = 0; c < 4; ++c) t.w[c] = *reinterpret_cast<const u32x4*>(wp + (2L * b + (c >> 1)) * RW + (c & 1) * 32);
#pragma unroll
        for (int c = 0; c < 4; ++c) t.a[c] = *reinterpret_cast<const u32x4*>(ap + (2L * b + (c >> 1)) * RA + (c & 1) * 32);
        t.ew = sw[(long)b * gW * 32];
        t.ea = sa[(long)b * gA * 32];
    };
    f32x16 acc = {};
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
        if (b0 + wave + 4 * u < b1) fetch(buf[u], b0 + wave + 4 * u);
    for (int b = b0 + wave; b < b1; b += 4 * DEPTH) {
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            if (b + 4 * u >= b1) continue;
            const float fw = scale_f32<0>(buf[u].ew >> shift), fa = scale_f32<0>(buf[u].ea);
            mma_wide(acc, widen(join8(buf[u].w[0], buf[u].w[1]), fw), widen(join8(buf[u].a[0], buf[u].a[1]), fa));
            mma_wide(acc, widen(join8(buf[u].w[2], buf[u].w[3]), fw), widen(join8(buf[u].a[2], buf[u].a[3]), fa));
            if (b + 4 * (u + DEPTH) < b1) fetch(buf[u], b + 4 * (u + DEPTH));
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) red[wave][fr * 33 + 8 * (r >> 2) + 4 * fh + (r & 3)] = acc[r];
    __syncthreads();
    float* part = slices > 1 ? ws + (long)slice * g.M * g.N : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = i * 8 + (tid >> 5);
        const long n = n0 + (tid & 31);
        if (m >= g.M || n >= g.N) continue;
        const int at = m * 33 + (tid & 31);
        float v = (red[0][at] + red[1][at]) + (red[2][at] + red[3][at]);
        if (part) {
            part[(long)m * g.N + n] = v;
        } else {
            v += g.bias ? g.bias[n] : 0.f;
            out_st(g.C, m * g.ldc + n, g.out_dt, g.act == SGG_ACT_RELU && v < 0.f ? 0.f : v);
        }
    }
}

// The same for up to 16 rows: 16 rows of W per workgroup and 16 waves over K, so that 4096 rows of W already occupy every CU without K slices whose
// partial outputs a second launch would have to add.  1 x 4096 x 25088: 17.9 us (5.7 TB/s of W, which the memory-side cache holds in part), 21.0 by the kernel above.
template <int DEPTH>
__global__ __launch_bounds__(1024) void fp8_few16_kernel(const Fp8Args g, float* __restrict__ ws, int per, int slices) {
    __shared__ float red[16][16 * 17];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int slice = blockIdx.x % slices;
    const long n0 = (long)(blockIdx.x / slices) * 16;
    const int blocks = (int)(g.Kp / 128), b0 = min(slice * per, blocks), b1 = min(b0 + per, blocks);
    const long gA = ((long)g.M + 127) / 128, gW = ((long)g.N + 127) / 128;
    const long n = min(n0 + fr, (long)g.N - 1);
    const long RA = slab_rows(g.M) * 64, RW = slab_rows(g.N) * 64;
    const unsigned char* wp = g.W + n * 64 + fq * 16;
    const unsigned char* ap = g.A + (long)min(fr, g.M - 1) * 64 + fq * 16;
    const unsigned* sw = reinterpret_cast<const unsigned*>(g.Ws) + (n >> 7) * 32 + (n & 31);
    const unsigned* sa = reinterpret_cast<const unsigned*>(g.As) + fr;
    const int shift = (int)(n >> 5 & 3) * 8;
    struct { u32x4 w[2], a[2]; unsigned ew, ea; } buf[DEPTH];
    auto fetch = [&](auto& t, int b) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            t.w[c] = *reinterpret_cast<const u32x4*>(wp + (2L * b + c) * RW);
            t.a[c] = *reinterpret_cast<const u32x4*>(ap + (2L * b + c) * RA);
        }
        t.ew = sw[(long)b * gW * 32];
        t.ea = sa[(long)b * gA * 32];
    };
    f32x4 acc = {};
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
        if (b0 + wave + 16 * u < b1) fetch(buf[u], b0 + wave + 16 * u);
    for (int b = b0 + wave; b < b1; b += 16 * DEPTH) {
#pragma unroll
        for (int u = 0; u < DEPTH; ++u) {
            if (b + 16 * u >= b1) continue;
            const Wide w = widen(join8(buf[u].w[0], buf[u].w[1]), scale_f32<0>(buf[u].ew >> shift)), a = widen(join8(buf[u].a[0], buf[u].a[1]), scale_f32<0>(buf[u].ea));
#pragma unroll
            for (int c = 0; c < 4; ++c)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w.c[c]), __builtin_bit_cast(bf16x8_t, a.c[c]), acc, 0, 0, 0);
            if (b + 16 * (u + DEPTH) < b1) fetch(buf[u], b + 16 * (u + DEPTH));
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][fr * 17 + 4 * fq + r] = acc[r];                // row m = fr, columns n0 + 4 fq + r
    __syncthreads();
    const int m = tid >> 4;
    const long no = n0 + (tid & 15);
    if (m >= 16 || m >= g.M || no >= g.N) return;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += red[w][m * 17 + (tid & 15)];
    if (slices > 1) {
        ws[((long)slice * g.M + m) * g.N + no] = v;
    } else {
        v += g.bias ? g.bias[no] : 0.f;
        out_st(g.C, m * g.ldc + no, g.out_dt, g.act == SGG_ACT_RELU && v < 0.f ? 0.f : v);
    }
}

// ---- (2) the middle: tiles of 128 x 128, one workgroup of eight waves per CU: two teams of four (64 x 64 each) take the blocks of 128 in turn, each through
// two LDS buffers of its own (32 KiB: one block of A and W), and add their sums in LDS at the end.  While one block is multiplied, the next one's loads are
// in flight to registers.  (Four waves and two workgroups per CU instead: 2048 x 2048 x 2048 19.9 us against 16.4, and twice the partial outputs where K is cut.)
constexpr int TILE_TEAM = 65536, TILE_SMEM = 2 * TILE_TEAM;
template <bool WIDE>
__global__ __launch_bounds__(512) void fp8_tile_kernel(const Fp8Args g, float* __restrict__ ws, int per, int slices) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = wave >> 2, tid = threadIdx.x & 255, lane = tid & 63, q = wave & 3;
    int tm, tn, slice;
    tile_and_slice((g.M + 127) / 128, (g.N + 127) / 128, tm, tn, slice);
    const long m0 = (long)tm * 128, n0 = (long)tn * 128;
    const int wm = (q >> 1) * 64, wn = (q & 1) * 64, fr = lane & 31, fh = lane >> 5;
    const int blocks = (int)(g.Kp / 128), b0 = min(slice * per, blocks), b1 = min(b0 + per, blocks);
    const long gA = ((long)g.M + 127) / 128, gW = ((long)g.N + 127) / 128;
    const unsigned *sa = reinterpret_cast<const unsigned*>(g.As) + (long)tm * 32 + fr, *sw = reinterpret_cast<const unsigned*>(g.Ws) + (long)tn * 32 + fr;
    // thread -> rows tid / 8 + 32 p, 16-byte piece tid % 8, stored at the piece permuted by half the row number (16 rows' reads of one piece then hit every bank once)
    const long RA = slab_rows(g.M), RW = slab_rows(g.N);
    const unsigned char *ap[4], *wp[4];
    int at[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int r = p * 32 + (tid >> 3), h = tid & 7;
        ap[p] = g.A + ((h >> 2) * RA + min(m0 + r, (long)g.M - 1)) * 64 + (h & 3) * 16;
        wp[p] = g.W + ((h >> 2) * RW + min(n0 + r, (long)g.N - 1)) * 64 + (h & 3) * 16;
        at[p] = r * 128 + ((h ^ (r >> 1 & 7)) << 4);
    }
    u32x4 ra[4], rw[4];
    unsigned ea_n = 0, ew_n = 0;
    auto fetch = [&](int b) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            ra[p] = *reinterpret_cast<const u32x4*>(ap[p] + b * RA * 128);
            rw[p] = *reinterpret_cast<const u32x4*>(wp[p] + b * RW * 128);
        }
        ea_n = sa[(long)b * gA * 32];
        ew_n = sw[(long)b * gW * 32];
    };
    f32x16 acc[2][2] = {};
    if (b0 + team < b1) fetch(b0 + team);
    for (int b = b0; b < b1; b += 2) {                       // (the same trips for every wave: a barrier inside)
        const bool mine = b + team < b1;
        char *sA = smem + team * TILE_TEAM + ((b - b0) >> 1 & 1) * 32768, *sW = sA + 16384;
        unsigned ea = 0, ew = 0;
        if (mine) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                *reinterpret_cast<u32x4*>(sA + at[p]) = ra[p];
                *reinterpret_cast<u32x4*>(sW + at[p]) = rw[p];
            }
            ea = ea_n >> (wm / 4), ew = ew_n >> (wn / 4);
        }
        if (b + team + 2 < b1) fetch(b + team + 2);
        // one barrier per step: this buffer's last readers (two steps ago) passed the previous step's barrier with their reads done
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (!mine) continue;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x8 a[2], w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int ra_ = wm + i * 32 + fr, rw_ = wn + i * 32 + fr, h = s * 4 + fh * 2;
                a[i] = join8(*reinterpret_cast<const u32x4*>(sA + ra_ * 128 + ((h ^ (ra_ >> 1 & 7)) << 4)), *reinterpret_cast<const u32x4*>(sA + ra_ * 128 + (((h + 1) ^ (ra_ >> 1 & 7)) << 4)));
                w[i] = join8(*reinterpret_cast<const u32x4*>(sW + rw_ * 128 + ((h ^ (rw_ >> 1 & 7)) << 4)), *reinterpret_cast<const u32x4*>(sW + rw_ * 128 + (((h + 1) ^ (rw_ >> 1 & 7)) << 4)));
            }
            if constexpr (WIDE) {
                const Wide a0 = widen(a[0], scale_f32<0>(ea)), a1 = widen(a[1], scale_f32<1>(ea)), w0 = widen(w[0], scale_f32<0>(ew)), w1 = widen(w[1], scale_f32<1>(ew));
                mma_wide(acc[0][0], w0, a0);
                mma_wide(acc[0][1], w1, a0);
                mma_wide(acc[1][0], w0, a1);
                mma_wide(acc[1][1], w1, a1);
            } else {
                acc[0][0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[0], a[0], acc[0][0], 0, 0, 0, ew, 0, ea);
                acc[0][1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[1], a[0], acc[0][1], 0, 0, 1, ew, 0, ea);
                acc[1][0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[0], a[1], acc[1][0], 0, 0, 0, ew, 1, ea);
                acc[1][1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[1], a[1], acc[1][1], 0, 0, 1, ew, 1, ea);
            }
        }
    }
    __syncthreads();                                          // (what follows lies over the operand buffers)
    float* part = slices > 1 ? ws + (long)slice * g.M * g.N : nullptr;
    // team t keeps the 32 rows mi = t of its wave's tile and hands the other 32 over; (team 0) + (team 1) either way
    f32x4* give = reinterpret_cast<f32x4*>(smem) + wave * 512 + lane;
    const f32x4* take = reinterpret_cast<const f32x4*>(smem) + (wave ^ 4) * 512 + lane;
#pragma unroll
    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const f32x16& o = team ? acc[0][ni] : acc[1][ni];
            give[(ni * 4 + c) * 64] = f32x4{o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]};
        }
    __syncthreads();
    f32x16 sum[1][2];
#pragma unroll
    for (int ni = 0; ni < 2; ++ni)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const f32x4 t = take[(ni * 4 + c) * 64];
            const f32x16& o = team ? acc[1][ni] : acc[0][ni];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[0][ni][4 * c + k] = o[4 * c + k] + t[k];
        }
    __syncthreads();
    out_wave<1, 2>(g, sum, smem + wave * EST, m0 + wm + team * 32, n0 + wn, part);
}

// ---- (3) large: tiles of 256 x 128 NI, 8 waves = two groups of four, one wave of each group per SIMD; a wave owns 128 x 32 NI.  K advances in slabs of 64
// bytes per row (half a block).  The groups run the same slabs one phase apart, one barrier per phase: while one group's waves read their fragments of a slab
// from LDS (and, for fp32 outputs, widen them), the other group's waves hold the matrix pipe:
//   slot      0        1        2        3        4   ...
//   group 0   LOAD 0   MFMA 0   LOAD 1   MFMA 1   LOAD 2
//   group 1   -        LOAD 0   MFMA 0   LOAD 1   MFMA 1
// A ring of D = 4 slabs (NI = 2: 4 x 32 KiB) is filled by loads straight to LDS, D - 1 slabs ahead, issued between the matrix instructions and counted (never
// drained before the end).  With a block's first slab travels the wave's own 256 bytes of scales: 32 dwords of its 128 rows of A, 32 of its rows of W.
// 16-byte pieces of a row are permuted by (row / 4) % 4 on the source address and on the read: fragment reads of 32 rows hit every bank once.
// Measured: 7936 x 4096 x 25088 668 us (2.44 PFLOP/s), 8192^3 402 us (2.73 PFLOP/s); fp32 outputs, on the 16-bit pipe, 1108 and 750 us (1.47 PFLOP/s).  The
// matrix pipe is busy 75 % of the cycles, but under that load the chip runs at 1.6 GHz of its 2.4: power bounds it (the same product of zeros takes a fifth
// less), so fewer bytes moved per product count for more than a fuller pipe.  256 x 256 by four waves of 128 x 128: 3 .. 10 % slower.

// one piece: uniform base + lane offset + immediate.  (The empty asm keeps the offset's widening next to the load, where it folds into the instruction's
// scalar-base form; widened outside the loop it would be a 64-bit vector add per piece.  `off` is the caller's own variable: a copy's register
// would be written again while the load is in flight, and the compiler waits for every load before that.)
template <int OFF>
__device__ __forceinline__ void lds_piece(const char* ubase, unsigned& off, char* l) {
    asm volatile("" : "+v"(off));
    __builtin_amdgcn_global_load_lds((glb_void_t*)(ubase + off), (lds_void_t*)l, 16, OFF, 0);
}

constexpr int PP_ROW = 64;
constexpr int pp_stage(int NI) { return (256 + 128 * NI) * PP_ROW; }
constexpr int PP_DEPTH = 4;                                           // slabs of the ring (a power of two; 6 measured no faster)
constexpr int pp_smem(int NI) { return PP_DEPTH * pp_stage(NI) + 4 * 8 * 256; }

template <bool WIDE, int NI>
__global__ __launch_bounds__(512) void fp8_pingpong_kernel(const Fp8Args g, float* __restrict__ ws, int per, int slices) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int D = PP_DEPTH, PP_STAGE = pp_stage(NI), PP_RING = D * PP_STAGE, PIECES = 2 + NI;
    static_assert(8 * EST <= PP_RING, "the output staging lies over the ring");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = wave >> 2, q = wave & 3, fr = lane & 31, fh = lane >> 5;
    int tm, tn, slice;
    tile_and_slice((g.M + 255) / 256, (g.N + 128 * NI - 1) / (128 * NI), tm, tn, slice);
    const long m0 = (long)tm * 256, n0 = (long)tn * 128 * NI;
    const int blocks = (int)(g.Kp / 128), b0 = min(slice * per, blocks), b1 = min(b0 + per, blocks);
    const int kb = 2 * b0, nt = 2 * b1;                       // slabs of this slice

    // ---- loads to LDS: a slab is (16 + 8 NI) pieces of 16 rows, the rows of A, then those of W; wave w loads pieces PIECES w + j.  Global address = the
    // piece's uniform base + a lane offset that never changes + the instruction's immediate, which also moves the LDS address: piece j lands j KiB
    // behind ONE LDS base (the lane offset carries -j KiB, and 3 KiB that the uniform base gives back keep it unsigned)
    const char *base_a = reinterpret_cast<const char*>(g.A + m0 * 64) - 3 * 1024, *base_w = reinterpret_cast<const char*>(g.W + n0 * 64) - 3 * 1024;
    const long step_a = slab_rows(g.M) * 64, step_w = slab_rows(g.N) * 64;              // from slab to slab
    unsigned vo[4] = {};
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int r = (PIECES * wave + j) * 16 + (lane >> 2);
        const long row = r < 256 ? min(m0 + r, (long)g.M - 1) - m0 : min(n0 + r - 256, (long)g.N - 1) - n0;        // (rows past the end: the last one again)
        vo[j] = (unsigned)(row * 64) + ((lane & 3) ^ ((r >> 2) & 3)) * 16 + 1024u * (3 - j);
    }
    unsigned vo_0 = vo[0], vo_1 = vo[1], vo_2 = vo[2], vo_3 = vo[3];
    const bool a_0 = PIECES * wave < 16, a_1 = PIECES * wave + 1 < 16, a_2 = PIECES * wave + 2 < 16, a_3 = PIECES * wave + 3 < 16;
    const int lds_rows0 = PIECES * wave * 16 * PP_ROW;
    const long gA = ((long)g.M + 127) / 128, gW = ((long)g.N + 127) / 128;
    const unsigned* sp = lane < 32 ? reinterpret_cast<const unsigned*>(g.As) + ((long)b0 * gA + min((long)tm * 2 + grp, gA - 1)) * 32 + fr
                                   : reinterpret_cast<const unsigned*>(g.Ws) + ((long)b0 * gW + min(n0 / 128 + q * NI / 4, gW - 1)) * 32 + fr;
    const long sstep = (lane < 32 ? gA : gW) * 32;
    char* const sreg = smem + PP_RING + wave * 256;
    int sblock = b0;
    // slabs are requested in order: kb .. nt - 1, then the last one D - 1 times more (into slabs of the ring that nobody reads again: the loop needs no tail)
    auto issue_scales = [&](int kt) {                         // with each even slab
        __builtin_amdgcn_global_load_lds((glb_void_t*)sp, (lds_void_t*)(sreg + ((kt >> 1) & 3) * 2048), 4, 0, 0);
        if (++sblock < b1) sp += sstep;
    };
    auto issue = [&](int kt) {
        const long k = min(kt, nt - 1);
        const char *sa = base_a + k * step_a, *sw = base_w + k * step_w;
        char* to = smem + (kt & (D - 1)) * PP_STAGE + lds_rows0;
        if (!(kt & 1)) issue_scales(kt);
        lds_piece<0>(uniform_ptr(a_0 ? sa : sw), vo_0, to);
        lds_piece<1024>(uniform_ptr(a_1 ? sa : sw), vo_1, to);
        lds_piece<2048>(uniform_ptr(a_2 ? sa : sw), vo_2, to);
        if constexpr (NI == 2) lds_piece<3 * 1024>(uniform_ptr(a_3 ? sa : sw), vo_3, to);
    };

    // LDS byte addresses of the lane's pieces fh and fh + 2 in slab 0: its first row of A and of W (the others 32 rows = 2 KiB further, same permutation)
    const unsigned lds0 = (unsigned)(unsigned long)(lds_void_t*)smem;
    const unsigned row_a = grp * 128 + fr, row_w = 256 + q * 32 * NI + fr;
    const unsigned at_a = lds0 + row_a * PP_ROW + ((fh ^ ((row_a >> 2) & 3)) << 4), at_w = lds0 + row_w * PP_ROW + ((fh ^ ((row_w >> 2) & 3)) << 4);
    const unsigned at_s = lds0 + PP_RING + wave * 256 + fr * 4;
    f32x16 acc[4][NI] = {};
    i32x8 af[4], wf[NI];
    Wide aw[4], ww[NI];
    unsigned ea = 0, ew = 0;
    // addresses of the next slab to read and of the next one to load, made while the matrix pipe is still busy with the last instructions of a phase
    unsigned ra0, ra1, rw0, rw1, rs, dst;
    const char *u0, *u1, *u2, *u3;
    auto prepare = [&](int kt) {
        const unsigned st = (kt & (D - 1)) * PP_STAGE;
        ra0 = at_a + st, ra1 = ra0 ^ 32, rw0 = at_w + st, rw1 = rw0 ^ 32;
        rs = at_s + ((kt >> 1) & 3) * 2048;
        const long k = min(kt + D - 1, nt - 1);
        const char *sa = base_a + k * step_a, *sw = base_w + k * step_w;
        u0 = uniform_ptr(a_0 ? sa : sw), u1 = uniform_ptr(a_1 ? sa : sw), u2 = uniform_ptr(a_2 ? sa : sw), u3 = uniform_ptr(a_3 ? sa : sw);
        dst = ((kt + D - 1) & (D - 1)) * PP_STAGE + lds_rows0;
    };
    auto load_frags = [&](bool even) {
        // one asm block, with its wait: the compiler waits for EVERY load to LDS in flight before an LDS read of its own
        u32x4 f[12];
        unsigned e = 0;
        // outputs 0 .. 7 the fragments of A, 8 .. the one or two of W, with a block's first slab two words of scales
#define FP8_READS_A(a0, a1)                                                                                                                    \
    "ds_read_b128 %0, " a0 "\n ds_read_b128 %1, " a1 "\n ds_read_b128 %2, " a0 " offset:2048\n ds_read_b128 %3, " a1 " offset:2048\n"         \
    "ds_read_b128 %4, " a0 " offset:4096\n ds_read_b128 %5, " a1 " offset:4096\n ds_read_b128 %6, " a0 " offset:6144\n ds_read_b128 %7, " a1 " offset:6144\n"
#define FP8_OUT_A "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3]), "=&v"(f[4]), "=&v"(f[5]), "=&v"(f[6]), "=&v"(f[7]), "=&v"(f[8]), "=&v"(f[9])
        if constexpr (NI == 2) {
            if (even)
                asm volatile("ds_read_b32 %12, %18\n ds_read_b32 %13, %18 offset:128\n"
                             "ds_read_b128 %8, %16\n ds_read_b128 %9, %17\n ds_read_b128 %10, %16 offset:2048\n ds_read_b128 %11, %17 offset:2048\n" FP8_READS_A("%14", "%15") "s_waitcnt lgkmcnt(0)"
                             : FP8_OUT_A, "=&v"(f[10]), "=&v"(f[11]), "=&v"(ea), "=&v"(e)
                             : "v"(ra0), "v"(ra1), "v"(rw0), "v"(rw1), "v"(rs)
                             : "memory");
            else
                asm volatile("ds_read_b128 %8, %14\n ds_read_b128 %9, %15\n ds_read_b128 %10, %14 offset:2048\n ds_read_b128 %11, %15 offset:2048\n" FP8_READS_A("%12", "%13") "s_waitcnt lgkmcnt(0)"
                             : FP8_OUT_A, "=&v"(f[10]), "=&v"(f[11])
                             : "v"(ra0), "v"(ra1), "v"(rw0), "v"(rw1)
                             : "memory");
        } else {
            if (even)
                asm volatile("ds_read_b32 %10, %16\n ds_read_b32 %11, %16 offset:128\n ds_read_b128 %8, %14\n ds_read_b128 %9, %15\n" FP8_READS_A("%12", "%13") "s_waitcnt lgkmcnt(0)"
                             : FP8_OUT_A, "=&v"(ea), "=&v"(e)
                             : "v"(ra0), "v"(ra1), "v"(rw0), "v"(rw1), "v"(rs)
                             : "memory");
            else
                asm volatile("ds_read_b128 %8, %12\n ds_read_b128 %9, %13\n" FP8_READS_A("%10", "%11") "s_waitcnt lgkmcnt(0)"
                             : FP8_OUT_A
                             : "v"(ra0), "v"(ra1), "v"(rw0), "v"(rw1)
                             : "memory");
        }
#undef FP8_READS_A
#undef FP8_OUT_A
        if (even) ew = e >> (q * NI * 8 & 31);                 // bytes: the wave's NI rows-of-32 inside the group of 128
        wf[0] = join8(f[8], f[9]);
        if constexpr (NI == 2) wf[NI - 1] = join8(f[10], f[11]);
#pragma unroll
        for (int i = 0; i < 4; ++i) af[i] = join8(f[2 * i], f[2 * i + 1]);
        if constexpr (WIDE) {
            ww[0] = widen(wf[0], scale_f32<0>(ew));
            if constexpr (NI == 2) ww[NI - 1] = widen(wf[NI - 1], scale_f32<1>(ew));
            aw[0] = widen(af[0], scale_f32<0>(ea)); aw[1] = widen(af[1], scale_f32<1>(ea));
            aw[2] = widen(af[2], scale_f32<2>(ea)); aw[3] = widen(af[3], scale_f32<3>(ea));
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#define FP8_MMA(mi)                                                                                                                              \
    if constexpr (WIDE) {                                                                                                                        \
        mma_wide(acc[mi][0], ww[0], aw[mi]);                                                                                                     \
        if constexpr (NI == 2) mma_wide(acc[mi][NI - 1], ww[NI - 1], aw[mi]);                                                                    \
    } else {                                                                                                                                     \
        acc[mi][0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[0], af[mi], acc[mi][0], 0, 0, 0, ew, mi, ea);                             \
        if constexpr (NI == 2) acc[mi][NI - 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[NI - 1], af[mi], acc[mi][NI - 1], 0, 0, 1, ew, mi, ea); \
    }
    auto compute_dma = [&](int kt, bool scales) {             // slab kt's matrix instructions with the loads of slab kt + D - 1 between them
        char* to = smem + dst;
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        FP8_MMA(0)
        if (scales) issue_scales(kt + D - 1);
        lds_piece<0>(u0, vo_0, to);
        __builtin_amdgcn_sched_barrier(0);
        FP8_MMA(1)
        lds_piece<1024>(u1, vo_1, to);
        __builtin_amdgcn_sched_barrier(0);
        FP8_MMA(2)
        lds_piece<2048>(u2, vo_2, to);
        __builtin_amdgcn_sched_barrier(0);
        FP8_MMA(3)
        if constexpr (NI == 2) lds_piece<3 * 1024>(u3, vo_3, to);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        prepare(kt + 1);
        __builtin_amdgcn_sched_barrier(0);
    };
#undef FP8_MMA
#define FP8_BARRIER()                     \
    {                                     \
        __builtin_amdgcn_s_barrier();     \
        asm volatile("" ::: "memory");    \
        __builtin_amdgcn_sched_barrier(0);\
    }
    // Waits.  A wave issues PIECES + 1 loads with an even slab (scales first), PIECES with an odd one, slabs in order.  Before the barrier behind which slab
    // kt + 1 is read, a wave may still have in flight what it issued after slab kt + 1: group 0 (at the end of MFMA kt, having issued kt + D - 1) the D - 2 slabs
    // behind it, group 1 (in LOAD kt, having issued kt + D - 2) D - 3 of them, the first of kt's own parity.
#pragma unroll
    for (int i = 0; i < D - 1; ++i) issue(kb + i);
    constexpr int AHEAD0 = (D - 2) * PIECES + (D - 2) / 2, AHEAD1 = (D - 3) * PIECES + (D - 4) / 2;
    wait_vmcnt<AHEAD0>();
    FP8_BARRIER()
    // slab kt + D - 1 goes where slab kt - 1 was: its last readers (group 1, LOAD kt - 1) had their reads done before the barrier that ended that phase
    prepare(kb);
    if (grp == 0) {
        for (int kt = kb; kt < nt; kt += 2) {
            load_frags(true);
            FP8_BARRIER()
            compute_dma(kt, false);
            wait_vmcnt<AHEAD0>();
            FP8_BARRIER()
            load_frags(false);
            FP8_BARRIER()
            compute_dma(kt + 1, true);
            wait_vmcnt<AHEAD0>();
            FP8_BARRIER()
        }
        FP8_BARRIER()                                         // slot 2 nt: group 1's last MFMA phase
    } else {
        FP8_BARRIER()                                         // slot 0
        for (int kt = kb; kt < nt; kt += 2) {
            load_frags(true);
            wait_vmcnt<AHEAD1 + 1>();
            FP8_BARRIER()
            compute_dma(kt, false);
            FP8_BARRIER()
            load_frags(false);
            wait_vmcnt<AHEAD1>();
            FP8_BARRIER()
            compute_dma(kt + 1, true);
            FP8_BARRIER()
        }
    }
    wait_vmcnt<0>();                                          // (every load to LDS has landed before the staging below lies over the ring)
    __syncthreads();
    out_wave<4, NI>(g, acc, smem + wave * EST, m0 + grp * 128, n0 + q * 32 * NI, slices > 1 ? ws + (long)slice * g.M * g.N : nullptr);
}

// ---- which kernel and how many K slices
enum { FP8_FEW16, FP8_FEW, FP8_TILE, FP8_HALF, FP8_FULL };
struct Fp8Plan { int kernel, tiles, slices, per; };

// Few rows: the stream kernels; W in slices only where its rows alone leave CUs idle and each of a workgroup's 16 | 4 waves keeps two | five blocks or more
// (M <= 32: 32 x 1024 x 8192 10.8 us whole, 8.8 in 3 slices; 17 x 4096 x 4096 7.0 and 8.0 in 2; M <= 16: 16 x 16 x 8000 5.8 and 6.8 in 2).
// Otherwise the cheapest of the three tilings and of its cuts along K: rounds of the 256 CUs x blocks of a slice x ns per block (STEP), and for a cut the
// join: its launch, its partial outputs written and read at 5 TB/s, half a us per slice.  Measured (us; 16-bit | fp32 outputs):
//                        128 x 128          256 x 128          256 x 256        chosen
//   1024 x 4096 x 4096   28.2 | 40.9        29.6 | 47.6 (2)    39.6 | 53.0 (3)  128 x 128
//   4096 x 2048 x 4096   55.0 | 84.0        36.0 | 64.5        50.4 | 77.1 (2)  256 x 128
//   512 x 4608 x 7936    45.1 | 61.9        33.5 | 50.3 (3)    40.1 | 54.7 (4)  256 x 128 in 3 slices
//   256 x 4096 x 25088   46.5 | 64.7 (4)    41.8 | 60.7 (8)    45.7 | 65.4 (12) 256 x 128 in 8 slices
//   256 x 1024 x 7936    18.5 | 21.5 (8)    19.3 | 24.6 (8)    24.3 | 31.2 (8)  128 x 128 in 8 slices
//   128 x 512 x 4096     13.3 | 14.4 (8)    13.2 | 15.8 (8)    16.4 | 19.0 (8)  128 x 128 in 8 slices (one slice: 24.5 | 35.0)
//   4096 x 4096 x 7936   -                  -                  101 | 186        256 x 256
// (slices in brackets)
Fp8Plan fp8_plan(int64_t M, int64_t N, int64_t Kp, bool wide) {
    const int64_t blocks = Kp / 128, one = 1;
    int64_t kernel = FP8_TILE, tiles, slices = 1;
    if (M <= 32) {
        kernel = M <= 16 ? FP8_FEW16 : FP8_FEW;
        tiles = M <= 16 ? (N + 15) / 16 : (N + 31) / 32;
        slices = max(min(256 / max(tiles, one), blocks / (M <= 16 ? 32 : 20)), one);
    } else {
        static const int64_t STEP[2][3] = {{700, 1000, 1500}, {1000, 1600, 2900}}, JOIN = 4000;
        const int64_t count[3] = {((M + 127) / 128) * ((N + 127) / 128), ((M + 255) / 256) * ((N + 127) / 128), ((M + 255) / 256) * ((N + 255) / 256)};
        tiles = count[0];
        double best = -1;
        for (int k = 0; k < 3 && blocks; ++k)
            for (int64_t s = 1; s == 1 || (s * count[k] <= 256 && s <= min(blocks / 2, (int64_t)32)); ++s) {
                const double t = (double)((count[k] * s + 255) / 256 * ((blocks + s - 1) / s) * STEP[wide][k]) + (s > 1 ? JOIN + 500 * s + (double)s * M * N / 625 : 0.);
                if (best < 0 || t < best) best = t, kernel = FP8_TILE + k, tiles = count[k], slices = s;
            }
    }
    const int64_t per = max((blocks + slices - 1) / slices, one);
    return {(int)kernel, tiles * slices > 0x7fffffff ? -1 : (int)tiles, (int)max((blocks + per - 1) / per, one), (int)per};       // (no empty slice)
}

template <auto kernel>
int fp8_launch(const Fp8Plan& p, int threads, int smem, const Fp8Args& g, float* ws, hipStream_t s) {
    static std::atomic<unsigned long> told{0};               // devices that know of this kernel's LDS, a bit each
    int dev = 0;
    if (smem > 65536 && hipGetDevice(&dev) != hipSuccess) return SGG_ERR_LAUNCH;
    if (smem > 65536 && !(told.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, smem) != hipSuccess) return SGG_ERR_LAUNCH;
        told.fetch_or(1ul << (dev & 63), std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(kernel, dim3(p.tiles * p.slices), dim3(threads), smem, s, g, ws, p.per, p.slices);
    SGG_CHECK_LAUNCH();
    return SGG_OK;
}

}  // namespace

extern "C" int64_t sgg_fp8_scale_bytes(int64_t rows, int64_t K) { return rows < 0 || K < 0 ? SGG_ERR_ARG : scale_bytes(rows, (K + 127) / 128); }

extern "C" int sgg_fp8_quantize(const void* x, int64_t ldx, int64_t M, int64_t K, void* rows, void* rows_scale, void* cols, void* cols_scale, float* colsum,
                                float* colsum_ws, int dtype, void* stream) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (M < 0 || K < 0 || M > 0x7fffff00 || K > 0x7fffff00 || ldx < K || (colsum && !colsum_ws)) return SGG_ERR_ARG;
    if (M > 0 && K > 0 && ((!rows && !cols) || !rows != !rows_scale || !cols != !cols_scale || (colsum && !cols))) return SGG_ERR_ARG;       // (empty forms have no memory)
    if ((((uintptr_t)rows | (uintptr_t)cols) & 15) || (((uintptr_t)rows_scale | (uintptr_t)cols_scale) & 3)) return SGG_ERR_ARG;
    const int64_t tilesM = (M + 127) / 128, tilesK = (K + 127) / 128;
    if (tilesM * tilesK > 0x7fffffff) return SGG_ERR_ARG;
    if (M > 0 && K > 0 && !x) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    if (M > 0 && K > 0) {
#define SGG_Q(R_, C_, S_)                                                                                                                               \
    SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL((fp8_quantize_kernel<T, R_, C_, S_>), dim3((unsigned)(tilesM * tilesK)), dim3(256), 0, s, (const T*)x, (long)ldx, \
                                            (long)M, (int)K, (unsigned char*)rows, (unsigned char*)rows_scale, (unsigned char*)cols,                       \
                                            (unsigned char*)cols_scale, colsum_ws, (int)tilesK))
        if (rows && cols) {
            if (colsum) { SGG_Q(true, true, true); } else { SGG_Q(true, true, false); }
        } else if (cols) {
            if (colsum) { SGG_Q(false, true, true); } else { SGG_Q(false, true, false); }
        } else {
            SGG_Q(true, false, false);
        }
#undef SGG_Q
        SGG_CHECK_LAUNCH();
    }
    return colsum && K > 0 ? sgg_reduce_parts(colsum_ws, (int)tilesM, (int)K, colsum, 0, s) : SGG_OK;
}

// K slices of a product whose output tiles alone do not fill the chip; ws then holds that many fp32 [M][N] partial outputs
extern "C" int sgg_gemm_fp8_splits(int64_t M, int64_t N, int64_t Kp, int out_dtype) {
    if (!sgg_is_dtype(out_dtype)) return SGG_ERR_DTYPE;
    if (M < 0 || N < 0 || Kp < 0 || Kp % 128 || M > 0x7fffff00 || N > 0x7fffff00 || Kp > 0x7fffff00) return SGG_ERR_ARG;
    return fp8_plan(M, N, Kp, out_dtype == SGG_F32).slices;
}

extern "C" int sgg_gemm_fp8(const void* A, const void* A_scale, const void* W, const void* W_scale, const float* bias, void* C, int64_t ldc, int64_t M,
                            int64_t N, int64_t Kp, int act, int out_dtype, float* ws, void* stream) {
    if (!sgg_is_dtype(out_dtype)) return SGG_ERR_DTYPE;
    if (M < 0 || N < 0 || Kp < 0 || Kp % 128 || M > 0x7fffff00 || N > 0x7fffff00 || Kp > 0x7fffff00 || ldc < N || (act != SGG_ACT_NONE && act != SGG_ACT_RELU))
        return SGG_ERR_ARG;
    if (M == 0 || N == 0) return SGG_OK;
    if (!C || (Kp > 0 && (!A || !A_scale || !W || !W_scale)) || (((uintptr_t)A | (uintptr_t)W) & 15) || (((uintptr_t)A_scale | (uintptr_t)W_scale) & 3)) return SGG_ERR_ARG;
    const Fp8Plan p = fp8_plan(M, N, Kp, out_dtype == SGG_F32);
    if (p.tiles < 0 || (p.slices > 1 && !ws)) return SGG_ERR_ARG;
    const Fp8Args g = {(const unsigned char*)A, (const unsigned char*)A_scale, (const unsigned char*)W, (const unsigned char*)W_scale, bias, (char*)C, (long)ldc, (long)Kp, (int)M, (int)N, act, out_dtype};
    hipStream_t s = (hipStream_t)stream;
    const bool wide = out_dtype == SGG_F32;
    int rc;
    switch (p.kernel) {
        case FP8_FEW16: rc = fp8_launch<fp8_few16_kernel<3>>(p, 1024, 0, g, ws, s); break;
        case FP8_FEW: rc = fp8_launch<fp8_few_rows_kernel<4>>(p, 256, 0, g, ws, s); break;
        case FP8_TILE: rc = wide ? fp8_launch<fp8_tile_kernel<true>>(p, 512, TILE_SMEM, g, ws, s) : fp8_launch<fp8_tile_kernel<false>>(p, 512, TILE_SMEM, g, ws, s); break;
        case FP8_HALF: rc = wide ? fp8_launch<fp8_pingpong_kernel<true, 1>>(p, 512, pp_smem(1), g, ws, s) : fp8_launch<fp8_pingpong_kernel<false, 1>>(p, 512, pp_smem(1), g, ws, s); break;
        default: rc = wide ? fp8_launch<fp8_pingpong_kernel<true, 2>>(p, 512, pp_smem(2), g, ws, s) : fp8_launch<fp8_pingpong_kernel<false, 2>>(p, 512, pp_smem(2), g, ws, s); break;
    }
    if (rc != SGG_OK || p.slices == 1) return rc;
    hipLaunchKernelGGL(fp8_join_kernel, dim3((unsigned)((N + 511) / 512), (unsigned)min((M + 3) / 4, (int64_t)1024)), dim3(256), 0, s, g, ws, p.slices);
    SGG_CHECK_LAUNCH();
    return SGG_OK;
}
