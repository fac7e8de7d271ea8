// Global norm of many tensors and their clipping:  n = |s| sqrt(sum_t sum_i g_ti^2),  out_ti = g_ti * s * min(1, max / (n + 1e-6)).
// Squares are summed in 64 bits: fp32 gradients of any finite size neither overflow nor vanish, and the sum over 10^8 elements keeps its
// last bits.  The factor stays in 64 bits too (beside gradients of 1e38 it is an fp32 subnormal); a clipped value is rounded to fp32, and a 16-bit one from
// there to its type (the chip has no way from 64 bits to 16): at most 2^-24 of it beside its own half step.
// No atomics: one partial per workgroup, added in a fixed order -- the same gradients give the same bits every time.
// Memory-bound, two readings and one writing (the factor is known only after the first).  Measured: 40 tensors of 248 M fp32 elements: norm 162 us (6.1 TB/s),
// scaling 382 .. 407 us (4.9 .. 5.2 TB/s, a copy's rate); 32 tensors of 17 M elements fp16 -> fp32: 12 + 30 us; 8 tensors of 17 K elements: 4 + 5 us.
#include <algorithm>
#include <memory>
#include <new>

#include "common.h"

namespace {

constexpr int CLIP_TAB = 96;            // tensors per launch (the table travels by value in the kernel arguments)
constexpr int CLIP_CHUNK = 8192;        // elements a workgroup takes at a time
constexpr int CLIP_BLOCKS = 2048;       // partials per launch: 8 workgroups per CU
// Chunks up to which one workgroup does it all in one launch (a chunk ends with its tensor: nine short tensors are nine chunks).  What a call takes, host
// and GPU: 8 chunks 10.0 us in place and 13.3 into other tensors, by two launches 13.1 either way; 4 chunks 10.1 and 13.2; 12 chunks 10.0 .. 19.9 and 13.2 ..
// 18.3.  (On the GPU alone one workgroup pays up to 4 chunks: 4.3 us in place against 4.4; 8 chunks 6.3 against 4.8.)
constexpr int CLIP_SMALL = 8;

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

typedef u32x4 u32x4_any __attribute__((aligned(2)));       // 16 bytes at the alignment of an element: this chip's loads and stores need no more
typedef f32x4 f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ float clip_ld(const void* p, long i, int dt) {
    return dt == SGG_F32 ? ((const float*)p)[i] : dt == SGG_BF16 ? bf16_to_f32(((const bf16_t*)p)[i]) : (float)((const f16_t*)p)[i];
}
__device__ __forceinline__ void clip_st(void* p, long i, int dt, float v) {
    if (dt == SGG_F32) ((float*)p)[i] = v;
    else if (dt == SGG_BF16) ((bf16_t*)p)[i] = f32_to_bf16(v);
    else ((f16_t*)p)[i] = (f16_t)v;
}
__device__ __forceinline__ void clip_st8(void* p, long i, int dt, const float (&v)[8]) {
    if (dt == SGG_F32) {
        __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4_any*>((float*)p + i));
        __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4_any*>((float*)p + i + 4));
    } else {
        __builtin_nontemporal_store(dt == SGG_BF16 ? pack8<bf16_t>(v) : pack8<f16_t>(v), reinterpret_cast<u32x4_any*>((unsigned short*)p + i));
    }
}

// Walks chunk c of tensor t with THREADS threads: f8(values, index) for whole pieces of 8, f1(value, index) for the elements of a last, partial
// one.  All of a thread's loads are issued before its first value is used.
template <int THREADS, typename F8, typename F1>
__device__ __forceinline__ void clip_walk(const ClipTab& tab, int t, int c, F8&& f8, F1&& f1) {
    const long base = (long)(c - tab.chunk0[t]) * CLIP_CHUNK;
    const int left = (int)min((long)CLIP_CHUNK, tab.n[t] - base), dt = tab.gdt[t];
    constexpr int PASS = CLIP_CHUNK / (THREADS * 8);
    const char* p = (const char*)tab.g[t] + base * (dt == SGG_F32 ? 4 : 2);
    const int at = threadIdx.x * 8;
    if (dt == SGG_F32) {
        f32x4 r[PASS][2];
#pragma unroll
        for (int q = 0; q < PASS; ++q)
            if (q * THREADS * 8 + at + 8 <= left) {
                const float* e = (const float*)p + q * THREADS * 8 + at;
                r[q][0] = *reinterpret_cast<const f32x4_any*>(e);
                r[q][1] = *reinterpret_cast<const f32x4_any*>(e + 4);
            }
#pragma unroll
        for (int q = 0; q < PASS; ++q)
            if (q * THREADS * 8 + at + 8 <= left) {
                const float v[8] = {r[q][0].x, r[q][0].y, r[q][0].z, r[q][0].w, r[q][1].x, r[q][1].y, r[q][1].z, r[q][1].w};
                f8(v, base + q * THREADS * 8 + at);
            }
    } else {
        u32x4 r[PASS];
#pragma unroll
        for (int q = 0; q < PASS; ++q)
            if (q * THREADS * 8 + at + 8 <= left) r[q] = *reinterpret_cast<const u32x4_any*>((const unsigned short*)p + q * THREADS * 8 + at);
#pragma unroll
        for (int q = 0; q < PASS; ++q)
            if (q * THREADS * 8 + at + 8 <= left) {
                float v[8];
                if (dt == SGG_BF16) unpack8<bf16_t>(r[q], v);
                else unpack8<f16_t>(r[q], v);
                f8(v, base + q * THREADS * 8 + at);
            }
    }
    if ((int)threadIdx.x < (left & 7)) f1(clip_ld(p, (left & ~7) + threadIdx.x, dt), base + (left & ~7) + threadIdx.x);
}

template <int THREADS>
__device__ __forceinline__ double clip_block_sum(double v, double* red) {       // every thread gets the sum
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) v += red[i];
    return v;
}

template <int THREADS>
__device__ __forceinline__ double clip_squares(const ClipTab& tab, int first, int step) {
    const int total = tab.chunk0[tab.count];
    double s[2] = {0.0, 0.0};
    for (int c = first; c < total; c += step)
        clip_walk<THREADS>(tab, clip_find(tab, c), c, [&](const float (&v)[8], long) {
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k & 1] = fma((double)v[k], (double)v[k], s[k & 1]);
        }, [&](float v, long) { s[0] = fma((double)v, (double)v, s[0]); });
    return s[0] + s[1];
}

template <int THREADS>
__device__ __forceinline__ void clip_scale(const ClipTab& tab, int first, int step, double f) {
    // the last chunks first: they are what the norm's walk has left in the memory-side cache
    for (int c = tab.chunk0[tab.count] - 1 - first; c >= 0; c -= step) {
        const int t = clip_find(tab, c);
        clip_walk<THREADS>(tab, t, c, [&](const float (&v)[8], long i) {
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = (float)((double)v[k] * f);
            clip_st8(tab.out[t], i, tab.odt[t], o);
        }, [&](float v, long i) { clip_st(tab.out[t], i, tab.odt[t], (float)((double)v * f)); });
    }
}

// norm and factor from the sum of squares
__device__ __forceinline__ double clip_factor(double sum, double max_norm, double scale, float* norm) {
    const double n = sqrt(sum) * fabs(scale);
    if (norm && threadIdx.x == 0) *norm = (float)n;
    const double c = max_norm / (n + 1e-6);
    return (c > 1.0 ? 1.0 : c) * scale;                     // (a NaN norm stays one: every gradient becomes NaN)
}

__global__ __launch_bounds__(256) void clip_norm_kernel(const ClipTab tab, double* __restrict__ part) {
    __shared__ double red[4];
    const double s = clip_block_sum<256>(clip_squares<256>(tab, blockIdx.x, gridDim.x), red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the partials' sum, the same in the same order in every workgroup that asks for it
__device__ __forceinline__ double clip_total(const double* __restrict__ part, int parts, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
    return clip_block_sum<256>(s, red);
}

__global__ __launch_bounds__(256) void clip_scale_kernel(const ClipTab tab, const double* __restrict__ part, int parts, double max_norm, double scale,
                                                         float* __restrict__ norm, int in_place) {
    __shared__ double red[4];
    const double f = clip_factor(clip_total(part, parts, red), max_norm, scale, blockIdx.x == 0 ? norm : nullptr);
    if (in_place && f == 1.0) return;
    clip_scale<256>(tab, blockIdx.x, gridDim.x, f);
}

__global__ __launch_bounds__(256) void clip_finish_kernel(const double* __restrict__ part, int parts, double scale, float* __restrict__ norm) {
    __shared__ double red[4];
    clip_factor(clip_total(part, parts, red), 1.0, scale, norm);
}

// Few elements: one workgroup does both in one launch (a second launch costs more than reading them again out of the cache)
__global__ __launch_bounds__(1024) void clip_small_kernel(const ClipTab tab, double max_norm, double scale, float* __restrict__ norm, int want, int in_place) {
    __shared__ double red[16];
    const double f = clip_factor(clip_block_sum<1024>(clip_squares<1024>(tab, 0, 1), red), max_norm, scale, norm);
    if (!want || (in_place && f == 1.0)) return;
    clip_scale<1024>(tab, 0, 1, f);
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

// Every tensor is written by workgroups of its own: no two of them may share memory (one given twice would be scaled twice), but an output may be
// its own gradient.
bool clip_apart(int count, const void* const* g, void* const* out, const int64_t* n, const int* gdt, const int* odt) {
    struct Range { uintptr_t lo, hi; };
    std::unique_ptr<Range[]> r(new (std::nothrow) Range[2 * (size_t)count + 1]);
    if (!r) return false;
    size_t k = 0;
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        const uintptr_t a = (uintptr_t)g[i], b = (uintptr_t)out[i];
        r[k++] = {a, a + (uintptr_t)n[i] * (gdt[i] == SGG_F32 ? 4 : 2)};
        if (a != b || gdt[i] != odt[i]) r[k++] = {b, b + (uintptr_t)n[i] * (odt[i] == SGG_F32 ? 4 : 2)};
    }
    std::sort(r.get(), r.get() + k, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    for (size_t i = 1; i < k; ++i)
        if (r[i].lo < r[i - 1].hi) return false;
    return true;
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
    if (chunks_all > 0x7fffffff || (out && !clip_apart(count, g, out, n, g_dtype, out_dtype))) return SGG_ERR_ARG;
    hipStream_t s = (hipStream_t)stream;
    int parts = 0;
    ClipTab tab;
    if (count <= CLIP_TAB && chunks_all <= CLIP_SMALL) {
        clip_fill(tab, 0, count, g, out, n, g_dtype, out_dtype);
        hipLaunchKernelGGL(clip_small_kernel, dim3(1), dim3(1024), 0, s, tab, max_norm, grad_scale, norm, out != nullptr, in_place);
        SGG_CHECK_LAUNCH();
        return SGG_OK;
    }
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
