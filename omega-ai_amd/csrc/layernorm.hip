// Layer norm over the rows of x [T,d].
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh gamma + beta
//   backward  g = dy gamma, dx = r (g - mean(g) - xh mean(g xh)), dgamma = sum_t dy xh, dbeta = sum_t dy
//
// A row stays in the registers of the 64 or 256 lanes that share it, so that both passes over it (the mean, then the squares of
// what differs from it: no cancellation) read memory once.  W elements a lane and load, N loads a lane; rows too long for that
// (more than 32 elements a lane) are read again by the *_long kernels.  Statistics and sums are fp32.
// The parameter gradients are summed while the rows are in registers: a workgroup takes rows w, w + n, ... and keeps a sum per
// column, the workgroups' sums are added by a second launch in a fixed order.
// Bound: bytes (x in, y out; x and dy in, dx out).
#include <algorithm>

#include "common.h"

template <bool BF, int W>
__device__ __forceinline__ void ld_w(const void *p, size_t i, float (&v)[W])
{
    if (BF) {
        const bf16_t *q = (const bf16_t *)p + i;
        if (W == 8) {
            const uint4 u = *(const uint4 *)q;
            const uint32_t a[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = __uint_as_float(k & 1 ? a[(k >> 1) & 3] & 0xffff0000u : a[(k >> 1) & 3] << 16);
        } else if (W == 4) {
            const uint2 u = *(const uint2 *)q;
            const uint32_t a[2] = {u.x, u.y};
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = __uint_as_float(k & 1 ? a[(k >> 1) & 1] & 0xffff0000u : a[(k >> 1) & 1] << 16);
        } else if (W == 2) {
            const uint32_t u = *(const uint32_t *)q;
            v[0] = __uint_as_float(u << 16);
            v[W - 1] = __uint_as_float(u & 0xffff0000u);
        } else {
            v[0] = bf16_to_f32(q[0]);
        }
    } else {
        const float *q = (const float *)p + i;
        if (W >= 4) {
#pragma unroll
            for (int k = 0; k < W; k += 4) *(float4 *)&v[k] = *(const float4 *)(q + k);
        } else if (W == 2) {
            *(float2 *)&v[0] = *(const float2 *)q;
        } else {
            v[0] = q[0];
        }
    }
}
template <bool BF, int W>
__device__ __forceinline__ void st_w(void *p, size_t i, const float (&v)[W])
{
    if (BF) {
        bf16_t *q = (bf16_t *)p + i;
        uint32_t a[(W + 1) / 2];
#pragma unroll
        for (int k = 0; k < W; k += 2) a[k >> 1] = (uint32_t)f32_to_bf16(v[k]) | (W > 1 ? (uint32_t)f32_to_bf16(v[(k + 1) % W]) << 16 : 0u);
        if (W == 8) *(uint4 *)q = make_uint4(a[0], a[1 % ((W + 1) / 2)], a[2 % ((W + 1) / 2)], a[3 % ((W + 1) / 2)]);
        else if (W == 4) *(uint2 *)q = make_uint2(a[0], a[1 % ((W + 1) / 2)]);
        else if (W == 2) *(uint32_t *)q = a[0];
        else q[0] = (bf16_t)a[0];
    } else {
        float *q = (float *)p + i;
        if (W >= 4) {
#pragma unroll
            for (int k = 0; k < W; k += 4) *(float4 *)(q + k) = *(const float4 *)&v[k];
        } else if (W == 2) {
            *(float2 *)q = *(const float2 *)&v[0];
        } else {
            q[0] = v[0];
        }
    }
}

__device__ __forceinline__ float wave_sum(float s)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
    return s;
}
// sum over the L lanes that share a row (L = 64: a wave; 256: the workgroup, `red` = 4 floats of LDS per use)
template <int L>
__device__ __forceinline__ float row_sum(float s, float *red)
{
    s = wave_sum(s);
    if (L == 64) return s;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <bool BF, int W, int N, int L>
__global__ __launch_bounds__(256) void layernorm_forward_kernel(const void *__restrict__ x, int T, int d, const float *__restrict__ gamma,
                                                                const float *__restrict__ beta, float eps, void *__restrict__ out,
                                                                float *__restrict__ mean, float *__restrict__ rstd)
{
    __shared__ float red[2][4];
    const int l = threadIdx.x & (L - 1), t = blockIdx.x * (256 / L) + threadIdx.x / L;
    if (L == 64 && t >= T) return;  // (whole waves: nothing below waits for them)
    const size_t row = (size_t)t * d;
    float v[N][W];
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (n * L + l) * W;
#pragma unroll
        for (int k = 0; k < W; ++k) v[n][k] = 0.0f;
        if (c < d) ld_w<BF, W>(x, row + c, v[n]);
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int k = 0; k < W; ++k) s += v[n][k];
    const float mu = row_sum<L>(s, red[0]) / (float)d;
    float q = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int k = 0; k < W; ++k) {
            v[n][k] -= mu;
            if ((n * L + l) * W < d) q = fmaf(v[n][k], v[n][k], q);
        }
    const float r = 1.0f / sqrtf(row_sum<L>(q, red[1]) / (float)d + eps);
    if (l == 0) {
        if (mean) mean[t] = mu;
        if (rstd) rstd[t] = r;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (n * L + l) * W;
        if (c >= d) continue;
        float g[W], b[W], o[W];
        ld_w<false, W>(gamma, c, g);
        ld_w<false, W>(beta, c, b);
#pragma unroll
        for (int k = 0; k < W; ++k) o[k] = fmaf(v[n][k] * r, g[k], b[k]);
        st_w<BF, W>(out, row + c, o);
    }
}

// Rows that do not fit the registers: a workgroup per row reads it three times (the later times from the caches).
template <bool BF>
__global__ __launch_bounds__(256) void layernorm_forward_long_kernel(const void *__restrict__ x, int T, int d, const float *__restrict__ gamma,
                                                                     const float *__restrict__ beta, float eps, void *__restrict__ out,
                                                                     float *__restrict__ mean, float *__restrict__ rstd)
{
    __shared__ float red[2][4];
    const int t = blockIdx.x;
    const size_t row = (size_t)t * d;
    float v[1], s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < d; c += 256) {
        ld_w<BF, 1>(x, row + c, v);
        s += v[0];
    }
    const float mu = row_sum<256>(s, red[0]) / (float)d;
    for (int c = threadIdx.x; c < d; c += 256) {
        ld_w<BF, 1>(x, row + c, v);
        q = fmaf(v[0] - mu, v[0] - mu, q);
    }
    const float r = 1.0f / sqrtf(row_sum<256>(q, red[1]) / (float)d + eps);
    if (threadIdx.x == 0) {
        if (mean) mean[t] = mu;
        if (rstd) rstd[t] = r;
    }
    for (int c = threadIdx.x; c < d; c += 256) {
        ld_w<BF, 1>(x, row + c, v);
        v[0] = fmaf((v[0] - mu) * r, gamma[c], beta[c]);
        st_w<BF, 1>(out, row + c, v);
    }
}

// part [gridDim.x][2][d]: a workgroup's sums of dy xh and of dy
template <bool BF, int W, int N, int L>
__global__ __launch_bounds__(256) void layernorm_backward_kernel(const void *__restrict__ x, const void *__restrict__ dout, int T, int d,
                                                                 const float *__restrict__ gamma, const float *__restrict__ mean,
                                                                 const float *__restrict__ rstd, void *__restrict__ dx, float *__restrict__ part)
{
    __shared__ float red[2][2][4];
    extern __shared__ __attribute__((aligned(16))) float cols[];  // L = 64: [3][2][d rounded up to a multiple of W], the sums of waves 1 .. 3
    constexpr int R = 256 / L;
    const int l = threadIdx.x & (L - 1), sub = threadIdx.x / L;
    float g[N][W], ag[N][W], ab[N][W];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (n * L + l) * W;
#pragma unroll
        for (int k = 0; k < W; ++k) g[n][k] = ag[n][k] = ab[n][k] = 0.0f;
        if (c < d) ld_w<false, W>(gamma, c, g[n]);
    }
    int turn = 0;
    for (int t0 = blockIdx.x * R; t0 < T; t0 += gridDim.x * R) {
        const int t = t0 + sub;
        if (L == 64 && t >= T) break;  // (whole waves; they meet the others behind the loop)
        const size_t row = (size_t)t * d;
        const float mu = mean[t], r = rstd[t];
        float xv[N][W], dv[N][W];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * L + l) * W;
#pragma unroll
            for (int k = 0; k < W; ++k) xv[n][k] = mu, dv[n][k] = 0.0f;
            if (c < d) {
                ld_w<BF, W>(x, row + c, xv[n]);
                ld_w<BF, W>(dout, row + c, dv[n]);
            }
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) {
                xv[n][k] = (xv[n][k] - mu) * r;
                ag[n][k] = fmaf(dv[n][k], xv[n][k], ag[n][k]);
                ab[n][k] += dv[n][k];
                dv[n][k] *= g[n][k];
                s1 += dv[n][k];
                s2 = fmaf(dv[n][k], xv[n][k], s2);
            }
        // (two sets of LDS words in turn: the next row's sums do not meet those another wave still reads)
        if (L == 64) {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
        } else {
            s1 = wave_sum(s1);
            s2 = wave_sum(s2);
            if ((threadIdx.x & 63) == 0) {
                red[turn][0][threadIdx.x >> 6] = s1;
                red[turn][1][threadIdx.x >> 6] = s2;
            }
            __syncthreads();
            s1 = (red[turn][0][0] + red[turn][0][1]) + (red[turn][0][2] + red[turn][0][3]);
            s2 = (red[turn][1][0] + red[turn][1][1]) + (red[turn][1][2] + red[turn][1][3]);
            turn ^= 1;
        }
        const float m1 = s1 / (float)d, m2 = s2 / (float)d;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * L + l) * W;
            if (c >= d) continue;
            float o[W];
#pragma unroll
            for (int k = 0; k < W; ++k) o[k] = r * (dv[n][k] - m1 - xv[n][k] * m2);
            st_w<BF, W>(dx, row + c, o);
        }
    }
    float *pg = part + (size_t)blockIdx.x * 2 * d, *pb = pg + d;
    const int dp = ceil_div(d, W) * W;
    if (L == 64) {
        if (sub > 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (n * L + l) * W;
                if (c >= d) continue;
                float *o = cols + (size_t)(sub - 1) * 2 * dp + c;
#pragma unroll
                for (int k = 0; k < W; ++k) o[k] = ag[n][k], o[dp + k] = ab[n][k];
            }
        }
        __syncthreads();
        if (sub > 0) return;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * L + l) * W;
            if (c >= d) continue;
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    ag[n][k] += cols[(size_t)w * 2 * dp + c + k];
                    ab[n][k] += cols[(size_t)w * 2 * dp + dp + c + k];
                }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (n * L + l) * W;
        if (c >= d) continue;
#pragma unroll
        for (int k = 0; k < W; ++k) pg[c + k] = ag[n][k], pb[c + k] = ab[n][k];
    }
}

template <bool BF>
__global__ __launch_bounds__(256) void layernorm_backward_long_kernel(const void *__restrict__ x, const void *__restrict__ dout, int T, int d,
                                                                      const float *__restrict__ gamma, const float *__restrict__ mean,
                                                                      const float *__restrict__ rstd, void *__restrict__ dx)
{
    __shared__ float red[2][4];
    const int t = blockIdx.x;
    const size_t row = (size_t)t * d;
    const float mu = mean[t], r = rstd[t];
    float xv[1], dv[1], s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < d; c += 256) {
        ld_w<BF, 1>(x, row + c, xv);
        ld_w<BF, 1>(dout, row + c, dv);
        const float g = dv[0] * gamma[c];
        s1 += g;
        s2 = fmaf(g, (xv[0] - mu) * r, s2);
    }
    const float m1 = row_sum<256>(s1, red[0]) / (float)d, m2 = row_sum<256>(s2, red[1]) / (float)d;
    for (int c = threadIdx.x; c < d; c += 256) {
        ld_w<BF, 1>(x, row + c, xv);
        ld_w<BF, 1>(dout, row + c, dv);
        dv[0] = r * (dv[0] * gamma[c] - m1 - (xv[0] - mu) * r * m2);
        st_w<BF, 1>(dx, row + c, dv);
    }
}
// the parameter gradients of long rows: a thread per column, a slice of the rows per workgroup (part as above)
template <bool BF>
__global__ __launch_bounds__(256) void layernorm_columns_kernel(const void *__restrict__ x, const void *__restrict__ dout, int T, int d,
                                                                const float *__restrict__ mean, const float *__restrict__ rstd, float *__restrict__ part)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= d) return;
    float ag = 0.0f, ab = 0.0f, xv[1], dv[1];
    for (int t = blockIdx.y; t < T; t += gridDim.y) {
        ld_w<BF, 1>(x, (size_t)t * d + c, xv);
        ld_w<BF, 1>(dout, (size_t)t * d + c, dv);
        ag = fmaf(dv[0], (xv[0] - mean[t]) * rstd[t], ag);
        ab += dv[0];
    }
    part[(size_t)blockIdx.y * 2 * d + c] = ag;
    part[(size_t)blockIdx.y * 2 * d + d + c] = ab;
}

// dgamma | dbeta = sums of n rows of part [n][2d]: a workgroup takes 16 columns, 64 threads each a fixed share of the rows, joined in LDS
__global__ __launch_bounds__(1024) void layernorm_join_kernel(const float *__restrict__ part, int n, int d, float *__restrict__ dgamma, float *__restrict__ dbeta)
{
    __shared__ float red[64][17];
    const int cc = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + cc;
    float s = 0.0f;
    if (c < 2 * d)
#pragma unroll 8
        for (int i = k; i < n; i += 64) s += part[(size_t)i * 2 * d + c];
    red[k][cc] = s;
    __syncthreads();
    for (int h = 32; h > 0; h >>= 1) {
        if (k < h) red[k][cc] += red[k + h][cc];
        __syncthreads();
    }
    if (k == 0 && c < 2 * d) (c < d ? dgamma + c : dbeta + (c - d))[0] = red[0][cc];
}

// How a row is shared: elements a load, loads a lane and lanes a row (lanes = 0: too long for the registers)
struct ln_shape {
    int w, n, lanes;
};
// (addresses of the rows, and of the fp32 parameters, which are read in as many elements)
static ln_shape ln_shape_of(int dtype, int d, int T, uintptr_t rows, uintptr_t pars)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16;
    ln_shape s = {1, 0, 0};
    // the widest load that every row start is aligned to
    for (int w = bf ? 8 : 4; w > 1; w >>= 1)
        if (d % w == 0 && rows % (w * (bf ? 2 : 4)) == 0 && pars % std::min(16, 4 * w) == 0) {
            s.w = w;
            break;
        }
    // a wave per row while it needs no more than 32 elements a lane, and a workgroup for rows that are few: a lane's loads go out
    // together, so that more lanes do not shorten a full device's pass
    for (int lanes = d > 512 && T < 2048 ? 256 : 64; lanes <= 256; lanes *= 4)
        if (d <= 32 * lanes) {
            s.lanes = lanes;
            const int per = ceil_div(d, lanes);
            s.n = (per <= 8 ? 8 : per <= 16 ? 16 : 32) / s.w;
            break;
        }
    return s;
}

// (the widths a dtype can have: 8, 4, 2, 1 elements of bf16, 4, 2, 1 of fp32)
#define LN_N(B, W, L, K, ...)                                                                              \
    do {                                                                                                    \
        if (sh.n * W == 8) hipLaunchKernelGGL((K<B, W, 8 / W, L>), __VA_ARGS__);                            \
        else if (sh.n * W == 16) hipLaunchKernelGGL((K<B, W, 16 / W, L>), __VA_ARGS__);                     \
        else hipLaunchKernelGGL((K<B, W, 32 / W, L>), __VA_ARGS__);                                         \
    } while (0)
#define LN_L(B, W, K, ...)                                 \
    do {                                                    \
        if (sh.lanes == 64) LN_N(B, W, 64, K, __VA_ARGS__); \
        else LN_N(B, W, 256, K, __VA_ARGS__);               \
    } while (0)
#define LN_RUN(K, ...)                                                 \
    do {                                                                \
        if (bf) {                                                       \
            if (sh.w == 8) LN_L(true, 8, K, __VA_ARGS__);               \
            else if (sh.w == 4) LN_L(true, 4, K, __VA_ARGS__);          \
            else if (sh.w == 2) LN_L(true, 2, K, __VA_ARGS__);          \
            else LN_L(true, 1, K, __VA_ARGS__);                         \
        } else {                                                        \
            if (sh.w == 4) LN_L(false, 4, K, __VA_ARGS__);              \
            else if (sh.w == 2) LN_L(false, 2, K, __VA_ARGS__);         \
            else LN_L(false, 1, K, __VA_ARGS__);                        \
        }                                                               \
    } while (0)

hipError_t launch_layernorm_forward(const void *x, int dtype, int T, int d, const float *gamma, const float *beta, float eps, void *out, float *mean,
                                    float *rstd, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16;
    const ln_shape sh = ln_shape_of(dtype, d, T, (uintptr_t)x | (uintptr_t)out, (uintptr_t)gamma | (uintptr_t)beta);
    if (sh.lanes == 0) {
        if (bf) hipLaunchKernelGGL(layernorm_forward_long_kernel<true>, dim3(T), dim3(256), 0, s, x, T, d, gamma, beta, eps, out, mean, rstd);
        else hipLaunchKernelGGL(layernorm_forward_long_kernel<false>, dim3(T), dim3(256), 0, s, x, T, d, gamma, beta, eps, out, mean, rstd);
        return hipGetLastError();
    }
    LN_RUN(layernorm_forward_kernel, dim3(ceil_div(T, 256 / sh.lanes)), dim3(256), 0, s, x, T, d, gamma, beta, eps, out, mean, rstd);
    return hipGetLastError();
}

// workgroups of the backward launch = rows of partial sums: two per compute unit
static int ln_backward_groups(const omega_ctx *ctx, int T) { return std::max(1, std::min(2 * ctx->num_cus, T)); }

size_t layernorm_backward_workspace(const omega_ctx *ctx, int T, int d) { return (size_t)ln_backward_groups(ctx, T) * 2 * d * sizeof(float); }

hipError_t launch_layernorm_backward(const omega_ctx *ctx, const void *x, const void *dout, int dtype, int T, int d, const float *gamma, const float *mean,
                                     const float *rstd, void *dx, float *dgamma, float *dbeta, void *ws, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16;
    float *part = (float *)ws;
    int n = 0;
    if (T > 0) {
        const ln_shape sh = ln_shape_of(dtype, d, T, (uintptr_t)x | (uintptr_t)dout | (uintptr_t)dx, (uintptr_t)gamma);
        n = ln_backward_groups(ctx, T);
        if (sh.lanes == 0) {
            const dim3 grid(ceil_div(d, 256), n);
            if (bf) {
                hipLaunchKernelGGL(layernorm_backward_long_kernel<true>, dim3(T), dim3(256), 0, s, x, dout, T, d, gamma, mean, rstd, dx);
                hipLaunchKernelGGL(layernorm_columns_kernel<true>, grid, dim3(256), 0, s, x, dout, T, d, mean, rstd, part);
            } else {
                hipLaunchKernelGGL(layernorm_backward_long_kernel<false>, dim3(T), dim3(256), 0, s, x, dout, T, d, gamma, mean, rstd, dx);
                hipLaunchKernelGGL(layernorm_columns_kernel<false>, grid, dim3(256), 0, s, x, dout, T, d, mean, rstd, part);
            }
        } else {
            n = std::min(n, ceil_div(T, 256 / sh.lanes));
            const size_t lds = sh.lanes == 64 ? (size_t)3 * 2 * ceil_div(d, sh.w) * sh.w * sizeof(float) : 0;
            LN_RUN(layernorm_backward_kernel, dim3(n), dim3(256), lds, s, x, dout, T, d, gamma, mean, rstd, dx, part);
        }
    }
    hipLaunchKernelGGL(layernorm_join_kernel, dim3(ceil_div(2 * d, 16)), dim3(1024), 0, s, part, n, d, dgamma, dbeta);
    return hipGetLastError();
}
