// Layer norm over the rows of x [T,d].
//
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh gamma + beta
//   backward  g = dy gamma, dx = r (g - mean(g) - xh mean(g xh)), dgamma = sum_t dy xh, dbeta = sum_t dy
//
// A row stays in the registers of the lanes that share it, 8 elements each (a wave, or a workgroup of 4, 8 or 16), so that both passes over it (the mean, then the squares of
// what differs from it: no cancellation) read memory once.  A lane loads 16 bytes at a time, N times; rows may start at any element
// (16-byte loads need no alignment here), a row's last piece is read element by element where it is not whole.  Rows too long for
// that (more than 8192 elements) are read again by the *_long kernels.  Statistics and sums are fp32.
// The parameter gradients are summed while the rows are in registers: a workgroup takes rows w, w + n, ... and keeps a sum per
// column, the workgroups' sums are added by a second launch in a fixed order.  The next row is asked for before the current one is worked on.
// Bound: bytes (x in, y out; x and dy in, dx out).
#include <algorithm>

#include "common.h"
#include "rows.h"

#define LN_THREADS(L) ((L) < 256 ? 256 : (L))
// sum over the L lanes that share a row (L = 64: a wave; more: the workgroup, `red` = a float of LDS per wave and use)
template <int L>
__device__ __forceinline__ float row_sum(float s, float *red)
{
    s = wave_sum(s);
    if (L == 64) return s;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) s += red[w];
    return s;
}

template <bool BF, int N, int L>
__global__ __launch_bounds__(LN_THREADS(L)) void layernorm_forward_kernel(const void *__restrict__ x, int T, int d, const float *__restrict__ gamma,
                                                                          const float *__restrict__ beta, float eps, void *__restrict__ out,
                                                                          float *__restrict__ mean, float *__restrict__ rstd)
{
    constexpr int W = piece<BF>::W, R = LN_THREADS(L) / L;
    __shared__ float red[4][16];
    const int l = threadIdx.x & (L - 1), step = gridDim.x * R;
    int t = blockIdx.x * R + threadIdx.x / L, turn = 0;
    if (t >= T) return;  // (L = 64: whole waves, nothing below waits for them)
    piece<BF> nx[N];     // the next row
    auto ask = [&](int row) {
#pragma unroll
        for (int n = 0; n < N; ++n) nx[n] = ld_piece<BF>(x, (size_t)row * d + (n * L + l) * W, d - (n * L + l) * W);
    };
    ask(t);
    float g[N][W], b[N][W];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        ld_par<W>(gamma, (n * L + l) * W, d - (n * L + l) * W, g[n]);
        ld_par<W>(beta, (n * L + l) * W, d - (n * L + l) * W, b[n]);
    }
    for (; t < T; t += step) {
        float v[N][W];
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) v[n][k] = el<BF>(nx[n], k);
        if (t + step < T) ask(t + step);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) s += v[n][k];
        // (LDS words in turn: the next row's sums do not meet those another wave still reads)
        const float mu = row_sum<L>(s, red[2 * turn]) / (float)d;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) {
                v[n][k] = (n * L + l) * W + k < d ? v[n][k] - mu : 0.0f;
                q = fmaf(v[n][k], v[n][k], q);
            }
        const float r = 1.0f / sqrtf(row_sum<L>(q, red[2 * turn + 1]) / (float)d + eps);
        turn ^= 1;
        if (l == 0) {
            if (mean) mean[t] = mu;
            if (rstd) rstd[t] = r;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * L + l) * W;
            if (c >= d) continue;
            float o[W];
#pragma unroll
            for (int k = 0; k < W; ++k) o[k] = fmaf(v[n][k] * r, g[n][k], b[n][k]);
            st_piece<BF>(out, (size_t)t * d + c, d - c, o);
        }
    }
}

// Rows that do not fit the registers: a workgroup per row reads it three times (the later times from the caches).
template <bool BF>
__global__ __launch_bounds__(256) void layernorm_forward_long_kernel(const void *__restrict__ x, int T, int d, const float *__restrict__ gamma,
                                                                     const float *__restrict__ beta, float eps, void *__restrict__ out,
                                                                     float *__restrict__ mean, float *__restrict__ rstd)
{
    __shared__ float red[2][16];
    const int t = blockIdx.x;
    const size_t row = (size_t)t * d;
    float v[1], s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < d; c += 256) {
        v[0] = ld1<BF>(x, row + c);
        s += v[0];
    }
    const float mu = row_sum<256>(s, red[0]) / (float)d;
    for (int c = threadIdx.x; c < d; c += 256) {
        v[0] = ld1<BF>(x, row + c);
        q = fmaf(v[0] - mu, v[0] - mu, q);
    }
    const float r = 1.0f / sqrtf(row_sum<256>(q, red[1]) / (float)d + eps);
    if (threadIdx.x == 0) {
        if (mean) mean[t] = mu;
        if (rstd) rstd[t] = r;
    }
    for (int c = threadIdx.x; c < d; c += 256) {
        v[0] = ld1<BF>(x, row + c);
        v[0] = fmaf((v[0] - mu) * r, gamma[c], beta[c]);
        st1<BF>(out, row + c, v[0]);
    }
}

// part [gridDim.x][2][d]: a workgroup's sums of dy xh and of dy
template <bool BF, int N, int L>
__global__ __launch_bounds__(LN_THREADS(L)) void layernorm_backward_kernel(const void *__restrict__ x, const void *__restrict__ dout, int T, int d,
                                                                 const float *__restrict__ gamma, const float *__restrict__ mean,
                                                                 const float *__restrict__ rstd, void *__restrict__ dx, float *__restrict__ part)
{
    constexpr int W = piece<BF>::W, R = LN_THREADS(L) / L;
    __shared__ float red[2][2][16];
    extern __shared__ __attribute__((aligned(16))) float cols[];  // L = 64: [3][2][d rounded up to a multiple of W], the sums of waves 1 .. 3
    const int l = threadIdx.x & (L - 1), sub = threadIdx.x / L;
    float g[N][W], ag[N][W], ab[N][W];
    piece<BF> nx[N], nd[N];  // the next row
    float nmu = 0.0f, nr = 0.0f;
    auto ask = [&](int t) {
        const size_t row = (size_t)t * d;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * L + l) * W;
            nx[n] = ld_piece<BF>(x, row + c, d - c);
            nd[n] = ld_piece<BF>(dout, row + c, d - c);
        }
        nmu = mean[t];
        nr = rstd[t];
    };
    int t = blockIdx.x * R + sub;
    const int step = gridDim.x * R;
    if (t < T) ask(t);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (n * L + l) * W;
        ld_par<W>(gamma, c, d - c, g[n]);
#pragma unroll
        for (int k = 0; k < W; ++k) ag[n][k] = ab[n][k] = 0.0f;
    }
    int turn = 0;
    for (; t < T; t += step) {  // (L = 64: whole waves; they meet the others behind the loop)
        const float mu = nmu, r = nr;
        float xv[N][W], dv[N][W];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) {
                xv[n][k] = el<BF>(nx[n], k);
                dv[n][k] = el<BF>(nd[n], k);
            }
        if (t + step < T) ask(t + step);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < W; ++k) {  // (elements behind the row's end: dy is zero, so are their terms)
                xv[n][k] = (xv[n][k] - mu) * r;
                ag[n][k] = fmaf(dv[n][k], xv[n][k], ag[n][k]);
                ab[n][k] += dv[n][k];
                dv[n][k] *= g[n][k];
                s1 += dv[n][k];
                s2 = fmaf(dv[n][k], xv[n][k], s2);
            }
        s1 = wave_sum(s1);
        s2 = wave_sum(s2);
        if (L > 64) {
            // (two sets of LDS words in turn: the next row's sums do not meet those another wave still reads)
            if ((threadIdx.x & 63) == 0) {
                red[turn][0][threadIdx.x >> 6] = s1;
                red[turn][1][threadIdx.x >> 6] = s2;
            }
            __syncthreads();
            s1 = s2 = 0.0f;
#pragma unroll
            for (int w = 0; w < L / 64; ++w) {
                s1 += red[turn][0][w];
                s2 += red[turn][1][w];
            }
            turn ^= 1;
        }
        const float m1 = s1 / (float)d, m2 = s2 / (float)d;
        const size_t row = (size_t)t * d;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * L + l) * W;
            if (c >= d) continue;
            float o[W];
#pragma unroll
            for (int k = 0; k < W; ++k) o[k] = r * (dv[n][k] - m1 - xv[n][k] * m2);
            st_piece<BF>(dx, row + c, d - c, o);
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
#pragma unroll
        for (int k = 0; k < W; ++k)
            if (c + k < d) pg[c + k] = ag[n][k], pb[c + k] = ab[n][k];
    }
}

template <bool BF>
__global__ __launch_bounds__(256) void layernorm_backward_long_kernel(const void *__restrict__ x, const void *__restrict__ dout, int T, int d,
                                                                      const float *__restrict__ gamma, const float *__restrict__ mean,
                                                                      const float *__restrict__ rstd, void *__restrict__ dx)
{
    __shared__ float red[2][16];
    const int t = blockIdx.x;
    const size_t row = (size_t)t * d;
    const float mu = mean[t], r = rstd[t];
    float xv[1], dv[1], s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < d; c += 256) {
        xv[0] = ld1<BF>(x, row + c);
        dv[0] = ld1<BF>(dout, row + c);
        const float g = dv[0] * gamma[c];
        s1 += g;
        s2 = fmaf(g, (xv[0] - mu) * r, s2);
    }
    const float m1 = row_sum<256>(s1, red[0]) / (float)d, m2 = row_sum<256>(s2, red[1]) / (float)d;
    for (int c = threadIdx.x; c < d; c += 256) {
        xv[0] = ld1<BF>(x, row + c);
        dv[0] = ld1<BF>(dout, row + c);
        dv[0] = r * (dv[0] * gamma[c] - m1 - (xv[0] - mu) * r * m2);
        st1<BF>(dx, row + c, dv[0]);
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
        xv[0] = ld1<BF>(x, (size_t)t * d + c);
        dv[0] = ld1<BF>(dout, (size_t)t * d + c);
        ag = fmaf(dv[0], (xv[0] - mean[t]) * rstd[t], ag);
        ab += dv[0];
    }
    part[(size_t)blockIdx.y * 2 * d + c] = ag;
    part[(size_t)blockIdx.y * 2 * d + d + c] = ab;
}

// dgamma | dbeta = sums of n rows of part [n][2d]: a workgroup takes 64 columns, its 16 waves a sixteenth of the rows each, joined in LDS
__global__ __launch_bounds__(1024) void layernorm_join_kernel(const float *__restrict__ part, int n, int d, float *__restrict__ dgamma, float *__restrict__ dbeta)
{
    __shared__ float red[16][64];
    const int cc = threadIdx.x & 63, k = threadIdx.x >> 6, c = blockIdx.x * 64 + cc;
    float s = 0.0f;
    for (int i0 = k; i0 < n && c < 2 * d; i0 += 16 * 16) {  // sixteen rows asked for together
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = i0 + 16 * j < n ? part[(size_t)(i0 + 16 * j) * 2 * d + c] : 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) s += v[j];
    }
    red[k][cc] = s;
    __syncthreads();
    if (k > 0 || c >= 2 * d) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) s += red[w][cc];
    (c < d ? dgamma + c : dbeta + (c - d))[0] = s;
}

// Lanes that share a row of d elements, 8 each: a wave, or a workgroup of 4, 8 or 16 (0: too long for them)
static int ln_lanes(int d) { return d <= 512 ? 64 : d <= 2048 ? 256 : d <= 4096 ? 512 : d <= 8192 ? 1024 : 0; }

#define LN_L(B, K, grid, lds, s, ...)                                                                                   \
    do {                                                                                                                \
        if (lanes == 64) hipLaunchKernelGGL((K<B, 8 / (B ? 8 : 4), 64>), grid, dim3(256), lds, s, __VA_ARGS__);          \
        else if (lanes == 256) hipLaunchKernelGGL((K<B, 8 / (B ? 8 : 4), 256>), grid, dim3(256), 0, s, __VA_ARGS__);     \
        else if (lanes == 512) hipLaunchKernelGGL((K<B, 8 / (B ? 8 : 4), 512>), grid, dim3(512), 0, s, __VA_ARGS__);     \
        else hipLaunchKernelGGL((K<B, 8 / (B ? 8 : 4), 1024>), grid, dim3(1024), 0, s, __VA_ARGS__);                     \
    } while (0)
#define LN_RUN(K, ...)                         \
    do {                                        \
        if (bf) LN_L(true, K, __VA_ARGS__);     \
        else LN_L(false, K, __VA_ARGS__);       \
    } while (0)

hipError_t launch_layernorm_forward(const omega_ctx *ctx, const void *x, int dtype, int T, int d, const float *gamma, const float *beta, float eps, void *out, float *mean,
                                    float *rstd, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16;
    const int lanes = ln_lanes(d);
    if (lanes == 0) {
        if (bf) hipLaunchKernelGGL(layernorm_forward_long_kernel<true>, dim3(T), dim3(256), 0, s, x, T, d, gamma, beta, eps, out, mean, rstd);
        else hipLaunchKernelGGL(layernorm_forward_long_kernel<false>, dim3(T), dim3(256), 0, s, x, T, d, gamma, beta, eps, out, mean, rstd);
        return hipGetLastError();
    }
    // workgroups: what the device holds at once, 2048 lanes a compute unit, so that gamma and beta are fetched once for several rows
    const int all = lanes == 64 ? ceil_div(T, 4) : T, held = ctx->num_cus * (2048 / std::max(lanes, 256));
    LN_RUN(layernorm_forward_kernel, dim3(std::min(all, held)), 0, s, x, T, d, gamma, beta, eps, out, mean, rstd);
    return hipGetLastError();
}

// Workgroups of the backward launch = rows of partial sums, which are written and read besides: two a compute unit of 256 lanes (16384 rows
// x 2048 bf16: one 64 us, two 50, three 52, four 57), one of 512 or 1024 (4096 x 8192: one 62 us, two 87), and two rows of x or more each.
static int ln_backward_groups(const omega_ctx *ctx, int T, int d)
{
    const int lanes = ln_lanes(d), per = lanes == 64 ? 3 : lanes == 256 ? 2 : 1, rows = lanes == 64 ? 4 : 1;
    return std::max(1, std::min(per * ctx->num_cus, ceil_div(T, 2 * rows)));
}

size_t layernorm_backward_workspace(const omega_ctx *ctx, int T, int d) { return (size_t)ln_backward_groups(ctx, T, d) * 2 * d * sizeof(float); }

hipError_t launch_layernorm_backward(const omega_ctx *ctx, const void *x, const void *dout, int dtype, int T, int d, const float *gamma, const float *mean,
                                     const float *rstd, void *dx, float *dgamma, float *dbeta, void *ws, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16;
    float *part = (float *)ws;
    int n = 0;
    if (T > 0) {
        const int lanes = ln_lanes(d);
        n = ln_backward_groups(ctx, T, d);
        if (lanes == 0) {
            const dim3 grid(ceil_div(d, 256), n);
            if (bf) {
                hipLaunchKernelGGL(layernorm_backward_long_kernel<true>, dim3(T), dim3(256), 0, s, x, dout, T, d, gamma, mean, rstd, dx);
                hipLaunchKernelGGL(layernorm_columns_kernel<true>, grid, dim3(256), 0, s, x, dout, T, d, mean, rstd, part);
            } else {
                hipLaunchKernelGGL(layernorm_backward_long_kernel<false>, dim3(T), dim3(256), 0, s, x, dout, T, d, gamma, mean, rstd, dx);
                hipLaunchKernelGGL(layernorm_columns_kernel<false>, grid, dim3(256), 0, s, x, dout, T, d, mean, rstd, part);
            }
        } else {
            const size_t lds = lanes == 64 ? (size_t)3 * 2 * ((d + 7) & ~7) * sizeof(float) : 0;
            LN_RUN(layernorm_backward_kernel, dim3(n), lds, s, x, dout, T, d, gamma, mean, rstd, dx, part);
        }
    }
    hipLaunchKernelGGL(layernorm_join_kernel, dim3(ceil_div(2 * d, 64)), dim3(1024), 0, s, part, n, d, dgamma, dbeta);
    return hipGetLastError();
}
