// Clipping of many tensors by their global norm, on the device:
//   norm = sqrt(sum_i sum g_i^2), coef = min(1, max_norm / (norm + 1e-6)), dst_i = coef * src_i
// (Network.clipGradNorm, J/engine/nn/network/Network.java:379-432; vectorL2NormKernel, J/engine/gpu/GlobalNormKernel.cu:3-30, adds its
// block sums with atomicAdd, here the order is fixed).  The tensors are cut into chunks; a workgroup takes a chunk, finds its tensor in
// a table that travels with the launch's arguments, and leaves one double; one workgroup adds these and forms coef; a second pass over
// the chunks scales.  Squares and sums are doubles: no sum overflows or loses the small gradients beside the large ones.
// Bound: bytes - every element is read twice and written once.
#include <algorithm>

#include "common.h"

#define CLIP_CHUNK 16384   // elements
#define CLIP_TENSORS 96    // tensors of a launch (its table: 2.7 KiB of arguments)

struct clip_table {
    const void *src[CLIP_TENSORS];
    void *dst[CLIP_TENSORS];
    uint64_t n[CLIP_TENSORS];       // bit 63: bf16
    uint32_t first[CLIP_TENSORS];   // first chunk of the tensor within the launch
    int tensors;
    uint32_t chunks;
};
#define CLIP_BF ((uint64_t)1 << 63)

static uint64_t clip_chunks(uint64_t n) { return (n + CLIP_CHUNK - 1) / CLIP_CHUNK; }

struct clip_piece {
    const void *src;
    void *dst;
    int n;      // elements of the chunk
    bool bf;
};
__device__ __forceinline__ clip_piece clip_find(const clip_table &t, uint32_t chunk)
{
    int lo = 0, hi = t.tensors;  // the last tensor whose first chunk is not behind this one
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    clip_piece p;
    p.bf = (t.n[lo] & CLIP_BF) != 0;
    const uint64_t n = t.n[lo] & ~CLIP_BF, at = (uint64_t)(chunk - t.first[lo]) * CLIP_CHUNK;
    p.n = (int)(n - at < CLIP_CHUNK ? n - at : CLIP_CHUNK);
    p.src = (const unsigned char *)t.src[lo] + at * (p.bf ? 2 : 4);
    p.dst = (unsigned char *)t.dst[lo] + at * (p.bf ? 2 : 4);
    return p;
}

// W elements of a piece from element i on (aligned loads)
template <bool BF>
struct clip_io {
    static constexpr int W = BF ? 8 : 4;
    static __device__ __forceinline__ void ld(const void *p, int i, float (&v)[W])
    {
        if (BF) {
            const uint4 u = *(const uint4 *)((const bf16_t *)p + i);
            const uint32_t a[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = __uint_as_float(k & 1 ? a[(k >> 1) & 3] & 0xffff0000u : a[(k >> 1) & 3] << 16);
        } else {
            *(float4 *)&v[0] = *(const float4 *)((const float *)p + i);
        }
    }
    static __device__ __forceinline__ void st(void *p, int i, const float (&v)[W])
    {
        if (BF) {
            uint32_t a[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = (uint32_t)f32_to_bf16(v[(2 * k) % W]) | (uint32_t)f32_to_bf16(v[(2 * k + 1) % W]) << 16;
            *(uint4 *)((bf16_t *)p + i) = make_uint4(a[0], a[1], a[2], a[3]);
        } else {
            *(float4 *)((float *)p + i) = *(const float4 *)&v[0];
        }
    }
    static __device__ __forceinline__ float ld1(const void *p, int i) { return BF ? bf16_to_f32(((const bf16_t *)p)[i]) : ((const float *)p)[i]; }
    static __device__ __forceinline__ void st1(void *p, int i, float v)
    {
        if (BF) ((bf16_t *)p)[i] = f32_to_bf16(v);
        else ((float *)p)[i] = v;
    }
};
// elements in front of the first 16-byte boundary
template <bool BF>
__device__ __forceinline__ int clip_head(const void *p, int n)
{
    const int es = BF ? 2 : 4;
    return min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) / es);
}

template <bool BF>
__device__ __forceinline__ double clip_sumsq(const clip_piece &p)
{
    constexpr int W = clip_io<BF>::W;
    double a[2] = {0.0, 0.0};
    const int head = clip_head<BF>(p.src, p.n), nv = (p.n - head) / W, tail = head + nv * W;
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += 256) {
        float v[W];
        clip_io<BF>::ld(p.src, head + i * W, v);
#pragma unroll
        for (int k = 0; k < W; ++k) a[k & 1] = fma((double)v[k], (double)v[k], a[k & 1]);
    }
    // at most W - 1 elements in front and behind
    int i = -1;
    if ((int)threadIdx.x < head) i = threadIdx.x;
    else if ((int)threadIdx.x >= 64 && (int)threadIdx.x - 64 < p.n - tail) i = tail + threadIdx.x - 64;
    if (i >= 0) {
        const double v = clip_io<BF>::ld1(p.src, i);
        a[0] = fma(v, v, a[0]);
    }
    return a[0] + a[1];
}

__device__ __forceinline__ double block_sum(double s, double *red)  // 256 threads or fewer, whole waves; the result in every thread
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
    const int wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = s;
    __syncthreads();
    double r = red[0];
    for (int w = 1; w < nw; ++w) r += red[w];
    return r;
}

__global__ __launch_bounds__(256) void clip_sumsq_kernel(clip_table t, double *__restrict__ part)
{
    __shared__ double red[4];
    const clip_piece p = clip_find(t, blockIdx.x);
    const double s = block_sum(p.bf ? clip_sumsq<true>(p) : clip_sumsq<false>(p), red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// out[0] = norm, out[1] = coef, and the same at norm_out
__global__ __launch_bounds__(1024) void clip_coef_kernel(const double *__restrict__ part, uint64_t n, float max_norm, float *__restrict__ out, float *__restrict__ norm_out)
{
    __shared__ double red[16];
    double a = 0.0;
#pragma unroll 8
    for (uint64_t i = threadIdx.x; i < n; i += 1024) a += part[i];
    const double norm = sqrt(block_sum(a, red));
    if (threadIdx.x == 0) {
        const double c = (double)max_norm / (norm + 1e-6);
        const float coef = isinf(max_norm) || c > 1.0 ? 1.0f : (float)c;  // (a norm that is no number: neither, coef is none)
        out[0] = (float)norm;
        out[1] = coef;
        if (norm_out) {
            norm_out[0] = (float)norm;
            norm_out[1] = coef;
        }
    }
}

template <bool BF>
__device__ __forceinline__ void clip_scale(const clip_piece &p, float coef)
{
    constexpr int W = clip_io<BF>::W;
    const int head = clip_head<BF>(p.src, p.n);
    if (clip_head<BF>(p.dst, p.n) != head) {  // source and destination are aligned differently
        for (int i = threadIdx.x; i < p.n; i += 256) clip_io<BF>::st1(p.dst, i, clip_io<BF>::ld1(p.src, i) * coef);
        return;
    }
    const int nv = (p.n - head) / W, tail = head + nv * W;
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += 256) {
        float v[W];
        clip_io<BF>::ld(p.src, head + i * W, v);
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] *= coef;
        clip_io<BF>::st(p.dst, head + i * W, v);
    }
    int i = -1;
    if ((int)threadIdx.x < head) i = threadIdx.x;
    else if ((int)threadIdx.x >= 64 && (int)threadIdx.x - 64 < p.n - tail) i = tail + threadIdx.x - 64;
    if (i >= 0) clip_io<BF>::st1(p.dst, i, clip_io<BF>::ld1(p.src, i) * coef);
}

__global__ __launch_bounds__(256) void clip_scale_kernel(clip_table t, const float *__restrict__ norm)
{
    const float coef = norm[1];
    const clip_piece p = clip_find(t, gridDim.x - 1 - blockIdx.x);
    if (coef == 1.0f && p.src == p.dst) return;  // nothing to change
    if (p.bf) clip_scale<true>(p, coef);
    else clip_scale<false>(p, coef);
}

size_t clip_workspace(const omega_grad_tensor *t, int n)
{
    uint64_t chunks = 0;
    for (int i = 0; i < n; ++i) chunks += clip_chunks(t[i].n);
    return 256 + chunks * sizeof(double);  // norm and coef, then the chunks' sums
}

// Fills a launch's table from part `at` of the list on (a long tensor takes several tables); false: the list has ended
struct clip_cursor {
    int i = 0;
    uint64_t done = 0;  // chunks of tensor i that earlier tables hold
};
#define CLIP_LAUNCH_CHUNKS (1u << 20)
static bool clip_fill(const omega_grad_tensor *t, int n, clip_cursor &c, clip_table &tab)
{
    tab.tensors = 0;
    tab.chunks = 0;
    while (c.i < n && tab.tensors < CLIP_TENSORS && tab.chunks < CLIP_LAUNCH_CHUNKS) {
        const omega_grad_tensor &x = t[c.i];
        const size_t es = x.dtype == OMEGA_DTYPE_BF16 ? 2 : 4;
        const uint64_t all = clip_chunks(x.n), take = std::min<uint64_t>(all - c.done, CLIP_LAUNCH_CHUNKS - tab.chunks);
        const uint64_t at = c.done * CLIP_CHUNK, len = std::min<uint64_t>(x.n - at, take * CLIP_CHUNK);
        const int k = tab.tensors++;
        tab.src[k] = (const unsigned char *)x.src + at * es;
        tab.dst[k] = (unsigned char *)x.dst + at * es;
        tab.n[k] = len | (es == 2 ? CLIP_BF : 0);
        tab.first[k] = tab.chunks;
        tab.chunks += (uint32_t)take;
        c.done += take;
        if (c.done == all) {
            ++c.i;
            c.done = 0;
        }
    }
    return tab.tensors > 0;
}

hipError_t launch_clip(const omega_grad_tensor *t, int n, float max_norm, float *norm_out, void *ws, hipStream_t s)
{
    float *norm = (float *)ws;
    double *part = (double *)((unsigned char *)ws + 256);
    uint64_t chunks = 0;
    clip_table tab;
    for (clip_cursor c; clip_fill(t, n, c, tab);) {
        hipLaunchKernelGGL(clip_sumsq_kernel, dim3(tab.chunks), dim3(256), 0, s, tab, part + chunks);
        chunks += tab.chunks;
    }
    hipLaunchKernelGGL(clip_coef_kernel, dim3(1), dim3(1024), 0, s, part, chunks, max_norm, norm, norm_out);
    for (clip_cursor c; clip_fill(t, n, c, tab);) hipLaunchKernelGGL(clip_scale_kernel, dim3(tab.chunks), dim3(256), 0, s, tab, norm);
    return hipGetLastError();
}
