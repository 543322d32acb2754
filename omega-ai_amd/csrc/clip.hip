// Clipping of many tensors by their global norm, on the device:
//   norm = sqrt(sum_i sum g_i^2), coef = min(1, max_norm / (norm + 1e-6)), dst_i = coef * src_i
// (Network.clipGradNorm, J/engine/nn/network/Network.java:379-432; vectorL2NormKernel, J/engine/gpu/GlobalNormKernel.cu:3-30, adds its
// block sums with atomicAdd, here the order is fixed).  The tensors are cut into chunks; a workgroup takes a chunk, finds its tensor in
// a table that travels with the launch's arguments, and leaves one double; one workgroup adds these and forms coef; a second pass over
// the chunks scales.  A thread adds up to 33 squares in fp32, all else is in double: no sum overflows or loses the small gradients beside the large.
// Bound: bytes - every element is read twice and written once.
#include <algorithm>

#include "common.h"

#define CLIP_CHUNK 8192    // elements
#define CLIP_FEW 1024      // chunks
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

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// NT: past the caches (what is written there fills them and more)
template <bool NT, class V>
__device__ __forceinline__ void clip_store(V *p, V v)
{
    if (NT) __builtin_nontemporal_store(v, p);
    else *p = v;
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
    template <bool NT>
    static __device__ __forceinline__ void st(void *p, int i, const float (&v)[W])
    {
        if (BF) {
            uint32_t a[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = (uint32_t)f32_to_bf16(v[(2 * k) % W]) | (uint32_t)f32_to_bf16(v[(2 * k + 1) % W]) << 16;
            clip_store<NT>((u4 *)((bf16_t *)p + i), u4{a[0], a[1], a[2], a[3]});
        } else {
            clip_store<NT>((f4 *)((float *)p + i), f4{v[0], v[1 % W], v[2 % W], v[3 % W]});
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

// A thread's share of a chunk: the whole 16-byte pieces threadIdx.x, + 256, ..., and one of the elements in front or behind.
template <bool BF>
struct clip_share {
    int head, nv, one;  // first whole piece, pieces, the single element (-1: none)
    __device__ __forceinline__ clip_share(const clip_piece &p)
    {
        constexpr int W = clip_io<BF>::W;
        head = clip_head<BF>(p.src, p.n);
        nv = (p.n - head) / W;
        const int tail = head + nv * W;
        one = (int)threadIdx.x < head ? (int)threadIdx.x : (int)threadIdx.x >= 64 && (int)threadIdx.x - 64 < p.n - tail ? tail + (int)threadIdx.x - 64 : -1;
    }
};
// Its sum of squares: in fp32 (33 elements at most, four sums), or, where that is too large, or so small that squares were lost, again in
// double.  (All in double: 325 us for 400 million elements, 290 so.)  Elements that are all zero, as most of an embedding's gradient and an
// idle expert's are, have lost nothing: told by their bits (norm of 400 million zeros in fp32: 441 us, 292 so, as of other values).
template <bool BF>
__device__ __forceinline__ double clip_sumsq(const clip_piece &p)
{
    constexpr int W = clip_io<BF>::W, U = 8;
    const clip_share<BF> sh(p);
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t any = 0;  // the elements' bits
    for (int i0 = threadIdx.x; i0 < sh.nv; i0 += 256 * U) {
        float v[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < W; ++k) v[u][k] = 0.0f;
            if (i0 + 256 * u < sh.nv) clip_io<BF>::ld(p.src, sh.head + (i0 + 256 * u) * W, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < W; ++k) {
                a[k & 3] = fmaf(v[u][k], v[u][k], a[k & 3]);
                any |= __float_as_uint(v[u][k]);
            }
    }
    if (sh.one >= 0) {
        const float v = clip_io<BF>::ld1(p.src, sh.one);
        a[0] = fmaf(v, v, a[0]);
        any |= __float_as_uint(v);
    }
    const float s = (a[0] + a[1]) + (a[2] + a[3]);
    if (any << 1 == 0) return 0.0;  // (zeros of either sign)
    // squares below 2^-126 keep 2^-150 each: less than 2^-26 of a sum of 1e-35; no number stays none
    if (s < 1e-35f || s > 3e38f) {
        double d = 0.0;
        for (int i = threadIdx.x; i < sh.nv; i += 256)
            for (int k = 0; k < W; ++k) {
                const double v = clip_io<BF>::ld1(p.src, sh.head + i * W + k);
                d = fma(v, v, d);
            }
        if (sh.one >= 0) {
            const double v = clip_io<BF>::ld1(p.src, sh.one);
            d = fma(v, v, d);
        }
        return d;
    }
    return s;
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

// Norm and coefficient from the chunks' sums, by a workgroup (x: norm, y: coefficient, in every thread)
__device__ __forceinline__ float2 clip_coef(const double *part, uint64_t n, float max_norm)
{
    __shared__ double red[16];
    double a = 0.0;
#pragma unroll 4
    for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) a += part[i];
    const double norm = sqrt(block_sum(a, red)), c = (double)max_norm / (norm + 1e-6);
    return make_float2((float)norm, isinf(max_norm) || c > 1.0 ? 1.0f : (float)c);  // (a norm that is no number: neither, the coefficient is none)
}
__device__ __forceinline__ void clip_tell(float2 v, float *to)
{
    if (threadIdx.x == 0 && to) {
        to[0] = v.x;
        to[1] = v.y;
    }
}
__global__ __launch_bounds__(1024) void clip_coef_kernel(const double *__restrict__ part, uint64_t n, float max_norm, float *__restrict__ out, float *__restrict__ norm_out)
{
    const float2 v = clip_coef(part, n, max_norm);
    clip_tell(v, out);
    clip_tell(v, norm_out);
}

template <bool BF, bool NT>
__device__ __forceinline__ void clip_scale(const clip_piece &p, float coef)
{
    constexpr int W = clip_io<BF>::W, U = 4;
    if (clip_head<BF>(p.dst, p.n) != clip_head<BF>(p.src, p.n)) {  // source and destination are aligned differently
        for (int i = threadIdx.x; i < p.n; i += 256) clip_io<BF>::st1(p.dst, i, clip_io<BF>::ld1(p.src, i) * coef);
        return;
    }
    const clip_share<BF> sh(p);
    for (int i0 = threadIdx.x; i0 < sh.nv; i0 += 256 * U) {
        float v[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < sh.nv) clip_io<BF>::ld(p.src, sh.head + (i0 + 256 * u) * W, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < sh.nv) {
#pragma unroll
                for (int k = 0; k < W; ++k) v[u][k] *= coef;
                clip_io<BF>::template st<NT>(p.dst, sh.head + (i0 + 256 * u) * W, v[u]);
            }
    }
    if (sh.one >= 0) clip_io<BF>::st1(p.dst, sh.one, clip_io<BF>::ld1(p.src, sh.one) * coef);
}

// FEW: the sums of all chunks, CLIP_FEW at most, are added by every workgroup for itself (a launch less: 200 000 elements 14.4 -> 10 us)
template <bool FEW, bool NT>
__global__ __launch_bounds__(256) void clip_scale_kernel(clip_table t, const float *__restrict__ norm, const double *__restrict__ part, uint64_t n, float max_norm,
                                                         float *__restrict__ norm_out)
{
    float coef;
    if (FEW) {
        const float2 v = clip_coef(part, n, max_norm);
        if (blockIdx.x == 0) clip_tell(v, norm_out);
        coef = v.y;
    } else {
        coef = norm[1];
    }
    const clip_piece p = clip_find(t, gridDim.x - 1 - blockIdx.x);  // (from the end: what the first pass read last is in the caches)
    if (coef == 1.0f && p.src == p.dst) return;  // nothing to change
    if (p.bf) clip_scale<true, NT>(p, coef);
    else clip_scale<false, NT>(p, coef);
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
    uint64_t chunks = 0, bytes = 0;
    for (int i = 0; i < n; ++i) bytes += t[i].n * (t[i].dtype == OMEGA_DTYPE_BF16 ? 2 : 4);
    clip_table tab;
    for (clip_cursor c; clip_fill(t, n, c, tab);) {
        hipLaunchKernelGGL(clip_sumsq_kernel, dim3(tab.chunks), dim3(256), 0, s, tab, part + chunks);
        chunks += tab.chunks;
    }
    if (n > 0 && chunks <= CLIP_FEW) {  // (one table: a chunk or more a tensor)
        clip_cursor c;
        clip_fill(t, n, c, tab);
        if (c.i == n) {
            hipLaunchKernelGGL((clip_scale_kernel<true, false>), dim3(tab.chunks), dim3(256), 0, s, tab, norm, part, chunks, max_norm, norm_out);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL(clip_coef_kernel, dim3(1), dim3(1024), 0, s, part, chunks, max_norm, norm, norm_out);
    // (53 million bf16 elements, 105 MB: 75 us, past the caches 62)
    const bool past = bytes >= OMEGA_LLC_BYTES / 8 * 3;
    for (clip_cursor c; clip_fill(t, n, c, tab);) {
        if (past) hipLaunchKernelGGL((clip_scale_kernel<false, true>), dim3(tab.chunks), dim3(256), 0, s, tab, norm, part, chunks, max_norm, norm_out);
        else hipLaunchKernelGGL((clip_scale_kernel<false, false>), dim3(tab.chunks), dim3(256), 0, s, tab, norm, part, chunks, max_norm, norm_out);
    }
    return hipGetLastError();
}
