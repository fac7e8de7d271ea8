// Matrix products in 8-bit floating point (OCP e4m3) with a power-of-two scale for each block of 128 along the reduction.
//
// Operand form: row m of a matrix [M][K] is Kp = K rounded up to 128 bytes of e4m3 (zero past K); block b of it, columns 128 b .. 128 b + 127, has the
// scale 2^e, e the smallest exponent >= -126 with max|x| <= 448 * 2^e, and q = x 2^-e rounded to nearest even: |x - q 2^e| <= 2^-4 |x| down to e4m3's
// subnormals (2^-10 of the scale).  A power of two because the matrix instruction of this chip (v_mfma_scale_f32_*_f8f6f4) multiplies by an e8m0 scale
// per row and 32 columns itself: dividing by it rounds nothing and applying it costs nothing.  Non-finite elements become NaN and do not
// enter the maximum: the products they take part in are NaN, the rest of the block keeps its scale.
// Scales are bytes (e + 127), 128 rows to a group: byte ((b * G + m / 128) * 32 + m % 32) * 4 + (m / 32) % 4 with G = ceil(M / 128) -- one dword
// holds the rows r, r + 32, r + 64, r + 96 of a group, i.e. what a lane of the 32-row MFMA fragments needs, picked by the instruction's
// byte selector.
#include "gemm_args.h"

namespace {

constexpr int QB = 128;             // columns of a block

__host__ __device__ __forceinline__ long scale_bytes(long rows, long blocks) { return blocks * ((rows + 127) / 128) * 128; }
__device__ __forceinline__ long scale_at(long m, long blk, long groups) { return ((blk * groups + (m >> 7)) * 32 + (m & 31)) * 4 + ((m >> 5) & 3); }

// biased exponent byte of the block whose largest finite magnitude has the bits `top`:  max = 1.f * 2^E; 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_byte(unsigned top) {
    const int E = (int)(top >> 23);                                   // biased
    return max(1, E - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ float scale_inv(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }        // 2^-(byte - 127)
__device__ __forceinline__ unsigned finite_bits(float v) {
    const unsigned a = __float_as_uint(v) & 0x7fffffffu;
    return a < 0x7f800000u ? a : 0u;
}
__device__ __forceinline__ float scaled(float v, float inv) {         // what the conversion is given: NaN for every non-finite input
    return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : v * inv;
}
__device__ __forceinline__ unsigned pack_fp8x4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// One workgroup = a tile of 128 x 128 values; thread (tr, tc) holds rows 8 tr .. 8 tr + 7, columns 8 tc .. 8 tc + 7.  The row form needs the
// largest magnitude of each row of the tile (16 lanes meet), the transposed form that of each column (LDS), so both come from one reading.
template <typename T, bool ROWS, bool COLS>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const T* __restrict__ x, long ldx, long M, int K, unsigned char* __restrict__ rows,
                                                           unsigned char* __restrict__ rscale, unsigned char* __restrict__ cols,
                                                           unsigned char* __restrict__ cscale, int tilesM) {
    __shared__ __attribute__((aligned(16))) unsigned char tile[128 * 128];
    __shared__ unsigned cmax[16][128];
    const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;
    const int tk = blockIdx.x / tilesM;
    const long tm = blockIdx.x - (long)tk * tilesM;
    const long m0 = tm * 128;
    const int k0 = tk * QB;
    const long Kp = ((long)K + 127) / 128 * 128;
    float v[8][8];
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * (long)sizeof(T)) % 16 == 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long m = m0 + tr * 8 + i;
        const int k = k0 + tc * 8;
        const T* p = x + m * ldx + k;
        if (m < M && vec && k + 8 <= K) {
            load8(p, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = m < M && k + j < K ? Elem<T>::ld(p + j) : 0.f;
        }
    }
    if constexpr (ROWS) {
        const long groups = (M + 127) / 128;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, finite_bits(v[i][j]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 16));
            const long m = m0 + tr * 8 + i;
            const int byte = scale_byte(top);
            const float inv = scale_inv(byte);
            float q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = scaled(v[i][j], inv);
            if (m < M) *reinterpret_cast<u32x2*>(rows + m * Kp + k0 + tc * 8) = u32x2{pack_fp8x4(q[0], q[1], q[2], q[3]), pack_fp8x4(q[4], q[5], q[6], q[7])};
            if (tc == 0) rscale[scale_at(m, tk, groups)] = (unsigned char)byte;          // (rows past M of the last group: blocks of zeros)
        }
    }
    if constexpr (COLS) {
        const long Mp = (M + 127) / 128 * 128, groups = ((long)K + 127) / 128;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, finite_bits(v[i][j]));
            cmax[tr][tc * 8 + j] = top;
        }
        __syncthreads();
        if (tid < 128) {
            unsigned top = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = max(top, cmax[r][tid]);
            const int byte = scale_byte(top);
            cmax[0][tid] = (unsigned)byte;
            cscale[scale_at(k0 + tid, tm, groups)] = (unsigned char)byte;
        }
        __syncthreads();
        // transposed tile in LDS: column c's 128 bytes, their 8-byte pieces permuted by c / 8 so that neither side's accesses pile up on a bank
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = tc * 8 + j;
            const float inv = scale_inv((int)cmax[0][c]);
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = scaled(v[i][j], inv);
            *reinterpret_cast<u32x2*>(tile + c * 128 + ((tr ^ tc) << 3)) = u32x2{pack_fp8x4(q[0], q[1], q[2], q[3]), pack_fp8x4(q[4], q[5], q[6], q[7])};
        }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int c = p * 32 + (tid >> 3), h = tid & 7, key = c >> 3;               // 16 bytes: pieces 2h and 2h + 1
            const u32x2 a = *reinterpret_cast<const u32x2*>(tile + c * 128 + (((2 * h) ^ key) << 3));
            const u32x2 b = *reinterpret_cast<const u32x2*>(tile + c * 128 + (((2 * h + 1) ^ key) << 3));
            if (k0 + c < K) *reinterpret_cast<u32x4*>(cols + (long)(k0 + c) * Mp + m0 + h * 16) = u32x4{a.x, a.y, b.x, b.y};
        }
    }
}

// ---- product: C[m][n] = sum_k A[m][k] W[n][k] (+ bias, ReLU), operands in the form above
//
// Two matrix pipes.  The 8-bit one (v_mfma_scale_f32_32x32x64_f8f6f4, twice the 16-bit rate) adds the products of a few columns at a time after
// aligning them to the largest, and CUTS what lies 2^-13 below that one's exponent (measured; the older 8-bit instructions do the same): a sum of
// products is off by ~1.3e-4 of itself.  That is below the rounding of a 16-bit output (half a step: f16 2^-11, bf16 2^-8) and is used for those.  An
// fp32 output gets fp32 sums: e4m3 * 2^e is converted in registers to bf16 -- exactly, four significant bits and any exponent -- and multiplied on the
// bf16 pipe, whose products are whole and whose sums round at 2^-24 (2^e * e4m3 below 2^-133 or from 2^128 on leaves bf16's range: 0 / inf).

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

__device__ __forceinline__ void out_st(char* C, long at, int dt, float v) {
    if (dt == SGG_F32) reinterpret_cast<float*>(C)[at] = v;
    else if (dt == SGG_BF16) reinterpret_cast<bf16_t*>(C)[at] = f32_to_bf16(v);
    else reinterpret_cast<f16_t*>(C)[at] = (f16_t)v;
}

// the plain tile: 128 x 128 outputs, 4 waves of 64 x 64, one block of 128 per step through LDS (2 x 16 KiB), rows past the end clamped
template <bool WIDE>
__global__ __launch_bounds__(256) void fp8_gemm_kernel(const Fp8Args g) {
    __shared__ __attribute__((aligned(16))) unsigned char sA[128 * 128], sW[128 * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tilesN = (g.N + 127) / 128;
    const long tm = blockIdx.x / tilesN, tn = blockIdx.x - tm * tilesN;
    const long m0 = tm * 128, n0 = tn * 128;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64, fr = lane & 31, fh = lane >> 5;
    const long blocks = g.Kp / 128, gA = ((long)g.M + 127) / 128, gW = ((long)g.N + 127) / 128;
    f32x16 acc[2][2] = {};
    for (long b = 0; b < blocks; ++b) {
        __syncthreads();
#pragma unroll
        for (int p = 0; p < 4; ++p) {                      // 128 rows of 8 16-byte pieces; pieces permuted by the row
            const int r = p * 32 + (tid >> 3), h = tid & 7, at = r * 128 + ((h ^ (r & 7)) << 4);
            *reinterpret_cast<u32x4*>(sA + at) = *reinterpret_cast<const u32x4*>(g.A + min(m0 + r, (long)g.M - 1) * g.Kp + b * 128 + h * 16);
            *reinterpret_cast<u32x4*>(sW + at) = *reinterpret_cast<const u32x4*>(g.W + min(n0 + r, (long)g.N - 1) * g.Kp + b * 128 + h * 16);
        }
        __syncthreads();
        const unsigned ea = reinterpret_cast<const unsigned*>(g.As)[(b * gA + tm) * 32 + fr] >> (wm / 4);
        const unsigned ew = reinterpret_cast<const unsigned*>(g.Ws)[(b * gW + tn) * 32 + fr] >> (wn / 4);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x8 a[2], w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int ra = wm + i * 32 + fr, rw = wn + i * 32 + fr, h = s * 4 + fh * 2;
                const u32x4 a0 = *reinterpret_cast<const u32x4*>(sA + ra * 128 + ((h ^ (ra & 7)) << 4)), a1 = *reinterpret_cast<const u32x4*>(sA + ra * 128 + (((h + 1) ^ (ra & 7)) << 4));
                const u32x4 w0 = *reinterpret_cast<const u32x4*>(sW + rw * 128 + ((h ^ (rw & 7)) << 4)), w1 = *reinterpret_cast<const u32x4*>(sW + rw * 128 + (((h + 1) ^ (rw & 7)) << 4));
                a[i] = join8(a0, a1);
                w[i] = join8(w0, w1);
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
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long m = m0 + wm + i * 32 + fr;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const long n = n0 + wn + j * 32 + 8 * (r >> 2) + 4 * fh + (r & 3);
                if (n >= g.N) continue;
                float t = acc[i][j][r] + (g.bias ? g.bias[n] : 0.f);
                if (g.act == SGG_ACT_RELU) t = t < 0.f ? 0.f : t;                         // (keeps NaN)
                out_st(g.C, m * g.ldc + n, g.out_dt, t);
            }
    }
}

}  // namespace

extern "C" int64_t sgg_fp8_scale_bytes(int64_t rows, int64_t K) { return rows < 0 || K < 0 ? SGG_ERR_ARG : scale_bytes(rows, (K + 127) / 128); }

extern "C" int sgg_fp8_quantize(const void* x, int64_t ldx, int64_t M, int64_t K, void* rows, void* rows_scale, void* cols, void* cols_scale, int dtype,
                                void* stream) {
    if (!sgg_is_dtype(dtype)) return SGG_ERR_DTYPE;
    if (M < 0 || K < 0 || M > 0x7fffff00 || K > 0x7fffff00 || ldx < K || (!rows && !cols) || !rows != !rows_scale || !cols != !cols_scale) return SGG_ERR_ARG;
    if (((uintptr_t)rows | (uintptr_t)cols) & 15) return SGG_ERR_ARG;
    if (M == 0 || K == 0) return SGG_OK;
    if (!x) return SGG_ERR_ARG;
    const int64_t tilesM = (M + 127) / 128, tilesK = (K + 127) / 128;
    if (tilesM * tilesK > 0x7fffffff) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
#define SGG_Q(R_, C_)                                                                                                                               \
    SGG_FOR_DTYPE(dtype, hipLaunchKernelGGL((fp8_quantize_kernel<T, R_, C_>), dim3((unsigned)(tilesM * tilesK)), dim3(256), 0, s, (const T*)x, (long)ldx, \
                                            (long)M, (int)K, (unsigned char*)rows, (unsigned char*)rows_scale, (unsigned char*)cols,                 \
                                            (unsigned char*)cols_scale, (int)tilesM))
    if (rows && cols) { SGG_Q(true, true); } else if (rows) { SGG_Q(true, false); } else { SGG_Q(false, true); }
#undef SGG_Q
    SGG_CHECK_LAUNCH();
    return SGG_OK;
}

// K slices of a product whose output tiles alone do not fill the chip; ws then holds that many fp32 [M][N] partial outputs
extern "C" int sgg_gemm_fp8_splits(int64_t M, int64_t N, int64_t Kp) {
    if (M < 0 || N < 0 || Kp < 0 || Kp % 128) return SGG_ERR_ARG;
    return 1;
}

extern "C" int sgg_gemm_fp8(const void* A, const void* A_scale, const void* W, const void* W_scale, const float* bias, void* C, int64_t ldc, int64_t M,
                            int64_t N, int64_t Kp, int act, int out_dtype, float* ws, void* stream) {
    if (!sgg_is_dtype(out_dtype)) return SGG_ERR_DTYPE;
    if (M < 0 || N < 0 || Kp < 0 || Kp % 128 || M > 0x7fffff00 || N > 0x7fffff00 || ldc < N || (act != SGG_ACT_NONE && act != SGG_ACT_RELU)) return SGG_ERR_ARG;
    if (M == 0 || N == 0) return SGG_OK;
    if (!C || (Kp > 0 && (!A || !A_scale || !W || !W_scale)) || (((uintptr_t)A | (uintptr_t)W) & 15) || (((uintptr_t)A_scale | (uintptr_t)W_scale) & 3)) return SGG_ERR_ARG;
    const int splits = sgg_gemm_fp8_splits(M, N, Kp);
    if (splits > 1 && !ws) return SGG_ERR_ARG;
    const Fp8Args g = {(const unsigned char*)A, (const unsigned char*)A_scale, (const unsigned char*)W, (const unsigned char*)W_scale, bias, (char*)C, (long)ldc, (long)Kp, (int)M, (int)N, act, out_dtype};
    const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
    if (tiles > 0x7fffffff) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    if (out_dtype == SGG_F32) hipLaunchKernelGGL(fp8_gemm_kernel<true>, dim3((unsigned)tiles), dim3(256), 0, s, g);
    else hipLaunchKernelGGL(fp8_gemm_kernel<false>, dim3((unsigned)tiles), dim3(256), 0, s, g);
    SGG_CHECK_LAUNCH();
    return SGG_OK;
}
