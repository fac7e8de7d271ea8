// Global norm of many tensors and their clipping:  n = |s| sqrt(sum_t sum_i g_ti^2),  out_ti = g_ti * s * min(1, max / (n + 1e-6)).
// Squares are summed in 64 bits: fp32 gradients of any finite size neither overflow nor vanish, and the sum over 10^8 elements keeps its
// last bits.  The factor stays in 64 bits too (beside gradients of 1e38 it is an fp32 subnormal); a clipped value is rounded once.  No atomics: one partial per workgroup, added in a fixed order -- the same gradients give the same bits every time.
#include "common.h"

namespace {

constexpr int CLIP_TAB = 96;            // tensors per launch (the table travels by value in the kernel arguments)
constexpr int CLIP_CHUNK = 8192;        // elements a workgroup takes at a time
constexpr int CLIP_BLOCKS = 1024;       // partials per launch

struct ClipTab {
    const void* g[CLIP_TAB];
    void* out[CLIP_TAB];
    long n[CLIP_TAB];
    int chunk0[CLIP_TAB + 1];           // prefix sums of ceil(n / CLIP_CHUNK)
    unsigned char gdt[CLIP_TAB], odt[CLIP_TAB];
    int count;
};

__device__ __forceinline__ int clip_find(const ClipTab& t, int c) {      // the tensor whose chunks hold chunk c
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (c >= t.chunk0[mid]) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float clip_ld(const void* p, long i, int dt) {
    return dt == SGG_F32 ? ((const float*)p)[i] : dt == SGG_BF16 ? bf16_to_f32(((const bf16_t*)p)[i]) : (float)((const f16_t*)p)[i];
}
__device__ __forceinline__ void clip_st(void* p, long i, int dt, float v) {
    if (dt == SGG_F32) ((float*)p)[i] = v;
    else if (dt == SGG_BF16) ((bf16_t*)p)[i] = f32_to_bf16(v);
    else ((f16_t*)p)[i] = (f16_t)v;
}

__device__ __forceinline__ double clip_block_sum(double v, double* red) {       // 256 threads; every thread gets the sum
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void clip_norm_kernel(const ClipTab tab, double* __restrict__ part) {
    __shared__ double red[4];
    const int total = tab.chunk0[tab.count];
    double s = 0.0;
    for (int c = blockIdx.x; c < total; c += gridDim.x) {
        const int t = clip_find(tab, c);
        const long base = (long)(c - tab.chunk0[t]) * CLIP_CHUNK, end = min(tab.n[t], base + CLIP_CHUNK);
        for (long i = base + threadIdx.x; i < end; i += 256) {
            const double v = (double)clip_ld(tab.g[t], i, tab.gdt[t]);
            s = fma(v, v, s);
        }
    }
    s = clip_block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the norm and the factor from the partials: the same sum in the same order in every workgroup that asks for it
__device__ __forceinline__ double clip_factor(const double* __restrict__ part, int parts, double max_norm, double scale, double* red, float* norm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
    const double n = sqrt(clip_block_sum(s, red)) * fabs(scale);
    if (norm && threadIdx.x == 0) *norm = (float)n;
    const double c = max_norm / (n + 1e-6);
    return (c > 1.0 ? 1.0 : c) * scale;                     // (a NaN norm stays one: every gradient becomes NaN)
}

__global__ __launch_bounds__(256) void clip_scale_kernel(const ClipTab tab, const double* __restrict__ part, int parts, double max_norm, double scale,
                                                         float* __restrict__ norm, int in_place) {
    __shared__ double red[4];
    const double f = clip_factor(part, parts, max_norm, scale, red, blockIdx.x == 0 ? norm : nullptr);
    if (in_place && f == 1.0) return;
    const int total = tab.chunk0[tab.count];
    for (int c = blockIdx.x; c < total; c += gridDim.x) {
        const int t = clip_find(tab, c);
        const long base = (long)(c - tab.chunk0[t]) * CLIP_CHUNK, end = min(tab.n[t], base + CLIP_CHUNK);
        for (long i = base + threadIdx.x; i < end; i += 256) clip_st(tab.out[t], i, tab.odt[t], (float)((double)clip_ld(tab.g[t], i, tab.gdt[t]) * f));
    }
}

__global__ __launch_bounds__(256) void clip_finish_kernel(const double* __restrict__ part, int parts, double scale, float* __restrict__ norm) {
    __shared__ double red[4];
    clip_factor(part, parts, 1.0, scale, red, norm);
}

int clip_fill(ClipTab& tab, int lo, int hi, const void* const* g, void* const* out, const int64_t* n, const int* gdt, const int* odt) {
    tab.count = 0;
    tab.chunk0[0] = 0;
    for (int i = lo; i < hi; ++i) {
        if (n[i] == 0) continue;
        const int k = tab.count++;
        tab.g[k] = g[i];
        tab.out[k] = out ? out[i] : nullptr;
        tab.n[k] = (long)n[i];
        tab.gdt[k] = (unsigned char)gdt[i];
        tab.odt[k] = (unsigned char)(out ? odt[i] : gdt[i]);
        tab.chunk0[k + 1] = tab.chunk0[k] + (int)((n[i] + CLIP_CHUNK - 1) / CLIP_CHUNK);
    }
    return tab.chunk0[tab.count];
}

}  // namespace

extern "C" int sgg_clip_grads_parts(int count) { return count < 0 ? SGG_ERR_ARG : max(1, (count + CLIP_TAB - 1) / CLIP_TAB) * CLIP_BLOCKS; }

extern "C" int sgg_clip_grads(const void* const* g, void* const* out, const int64_t* n, const int* g_dtype, const int* out_dtype, int count, double max_norm,
                              double grad_scale, double* ws, float* norm, void* stream) {
    if (count < 0 || !norm || !ws || (count > 0 && (!g || !n || !g_dtype)) || (out && !out_dtype) || (out && !(max_norm >= 0.0))) return SGG_ERR_ARG;
    int in_place = out != nullptr;
    int64_t chunks_all = 0;
    for (int i = 0; i < count; ++i) {
        if (!sgg_is_dtype(g_dtype[i]) || (out && !sgg_is_dtype(out_dtype[i]))) return SGG_ERR_DTYPE;
        if (n[i] < 0 || (n[i] > 0 && (!g[i] || (out && !out[i])))) return SGG_ERR_ARG;
        if (out && n[i] > 0 && out[i] != g[i]) in_place = 0;
        chunks_all += (n[i] + CLIP_CHUNK - 1) / CLIP_CHUNK;
    }
    if (chunks_all > 0x7fffffff) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    int parts = 0;
    ClipTab tab;
    for (int lo = 0; lo < count; lo += CLIP_TAB) {
        const int chunks = clip_fill(tab, lo, min(count, lo + CLIP_TAB), g, out, n, g_dtype, out_dtype);
        if (!chunks) continue;
        const int grid = min(chunks, CLIP_BLOCKS);
        hipLaunchKernelGGL(clip_norm_kernel, dim3(grid), dim3(256), 0, s, tab, ws + parts);
        SGG_CHECK_LAUNCH();
        parts += grid;
    }
    if (!out || parts == 0) {
        hipLaunchKernelGGL(clip_finish_kernel, dim3(1), dim3(256), 0, s, ws, parts, grad_scale, norm);
        SGG_CHECK_LAUNCH();
        return SGG_OK;
    }
    bool told = false;
    for (int lo = 0; lo < count; lo += CLIP_TAB) {
        const int chunks = clip_fill(tab, lo, min(count, lo + CLIP_TAB), g, out, n, g_dtype, out_dtype);
        if (!chunks) continue;
        hipLaunchKernelGGL(clip_scale_kernel, dim3(min(chunks, CLIP_BLOCKS)), dim3(256), 0, s, tab, ws, parts, max_norm, grad_scale,
                           told ? (float*)nullptr : norm, in_place);
        SGG_CHECK_LAUNCH();
        told = true;
    }
    return SGG_OK;
}
