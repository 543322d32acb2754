// RMS norm over the rows of x [T,d], with the addition of a residual in front of it and copies of 8 bits behind it.
//
//   forward   h = x + residual (rounded to the rows' type: what the next block adds to), q = 1 / sqrt(mean(h^2) + eps), y = h q gamma
//   backward  g = dy gamma, xh = h q, dh = q (g - xh mean(g xh)) + dsum, dgamma = sum_t dy xh   (dsum: gradient that reaches h past the norm)
//
// y in the rows' type, or in 8 bits with scales (eight.h, the form that matrix cores read); h may be kept in 8 bits for the backward pass,
// which then reads those.  A row stays in the registers of the lanes that share it, eight elements a lane and piece, so that memory is passed
// over once; rows may start at any element.  Rows too long for that are read again by the *_long kernels.
// The sum of squares is taken in double, which costs two of some ten operations an element that the memory leaves time for: q is then right to a
// rounding, and a y next to a border of its 8 bits can be formed again in double, by the lane that finds it there.
// The next row is asked for before the current one is worked on.  Gamma's gradient as in layernorm.hip: a sum per column and workgroup, joined by a
// second launch in a fixed order.  Bound: bytes (16384 x 2048 bf16 with a residual: forward 48.7 us, backward 48.7, 5.5 TB/s each; the same that keeps its input
// in 8 bits 55 and 48.8; 16384 x 4096 with 8-bit output 97 to 100 us, 4.7 TB/s and more; 16384 x 4096 fp32 with a residual: forward 197, backward 194, 5.5 TB/s
// each, with 8-bit output 160).
#include <algorithm>

#include "eight.h"

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ double lane_add(double s)
{
    const int2 u = *(const int2 *)&s;
    int2 v;
    v.x = __builtin_amdgcn_update_dpp(0, u.x, CTRL, 0xf, 0xf, true);
    v.y = __builtin_amdgcn_update_dpp(0, u.y, CTRL, 0xf, 0xf, true);
    return s + *(const double *)&v;
}
// sum over a wave, the same in every lane: around the rows of 16 lanes, then between them
__device__ __forceinline__ double wave_sum(double s)
{
    s = lane_add<0x128>(s);  // row_ror 8, 4, 2, 1
    s = lane_add<0x124>(s);
    s = lane_add<0x122>(s);
    s = lane_add<0x121>(s);
#define ACROSS(swap)                                                              \
    do {                                                                          \
        const u32x2 u = *(const u32x2 *)&s;                                       \
        const u32x2 lo = swap(u[0], u[0], false, false), hi = swap(u[1], u[1], false, false); \
        const u32x2 a = {lo[0], hi[0]}, b = {lo[1], hi[1]};                       \
        s = *(const double *)&a + *(const double *)&b;                            \
    } while (0)
    ACROSS(__builtin_amdgcn_permlane16_swap);
    ACROSS(__builtin_amdgcn_permlane32_swap);
#undef ACROSS
    return s;
}
// over the L lanes that share a row (more than a wave: the workgroup, `red` = a word of LDS per wave and use)
template <int L, class F>
__device__ __forceinline__ F row_total(F s, F *red)
{
    s = wave_sum(s);
    if (L == 64) return s;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) s += red[w];
    return s;
}
// 1 / sqrt(a) to a rounding or two of double: two steps of Newton's from the instruction's 2^-26 (which is the answer for 0 and infinity)
__device__ __forceinline__ double rsqrt64(double a)
{
    const double q = __builtin_amdgcn_rsq(a), h = 0.5 * a;
    double r = q * fma(-h * q, q, 1.5);
    r = r * fma(-h * r, r, 1.5);
    return r == r ? r : q;
}

// Codes of y = v r gamma (r: q in fp32) and their group's scale, those of v q gamma in double: y in fp32 is within three roundings of it, and what lies
// nearer to a border (of the codes, odd multiples of half a step; of the scale, 448 2^k) is formed again.
// A v r below the least normal number is off by up to 2^-149, y by that times gamma; less than 2^-30 of the scale unless the group's largest y is below 2^-110
// of its largest gamma: such groups, and rows whose r is below the least normal number, have their y from double.  (A group of zeros is one, or has codes of
// zero, up to a gamma of 2^12.  y itself may be subnormal: it is rounded to multiples of 2^-149, which the borders are too.)
struct norm_small {
    uint32_t least, span;  // groups whose largest y, as a whole number, is in least .. least + span
    __device__ __forceinline__ explicit norm_small(const float (&gamma)[8])
    {
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(gamma[k]));
        const float g = __uint_as_float(max_over_4(__float_as_uint(m)));
        least = g < 0x1p12f ? 1u : 0u;
        span = max(__float_as_uint(g * 0x1p-110f), 1u) - least;
    }
    __device__ __forceinline__ norm_small() {}
};
__device__ __forceinline__ u32x2_by norm_to_mx(const float (&v)[8], double q, float r, const float (&gamma)[8], norm_small small, float (&y)[8], uint32_t *scale)
{
    uint32_t most = max_over_4(magnitude(y));
    if (__builtin_expect(r < 0x1p-126f || most - small.least <= small.span, 0)) {  // (the same in the group's four lanes)
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = (float)((double)v[k] * q * (double)gamma[k]);
        most = max_over_4(magnitude(y));
    }
    uint32_t b = mx_scale(most);
    if ((most & 0x7fffffu) - 0x5ffffcu <= 8u && most < 0x7f800000u) {  // (as above)
        double m = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmax(m, fabs((double)v[k] * q * (double)gamma[k]));
        // above 448 2^k or not: a float on the same side of it
        const float at = __uint_as_float((most & 0x7f800000u) | 0x600000u);
        b = mx_scale(max_over_4(m > (double)at ? __float_as_uint(at) + 1u : __float_as_uint(at)));
    }
    *scale = b;
    const float inv = b == 255u ? 0.0f : mx_inverse(b);
    float u[8];
    bool near = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        u[k] = b == 255u ? 0.0f : y[k] * inv;
        const float a = fabsf(u[k]);
        // 20 bits below the code's: half of their range is a border (below 2^-6 all codes are multiples of 2^-9, as between 2^-6 and 2^-5)
        const uint32_t w = __float_as_uint(a < 0x1p-6f ? a + 0x1p-6f : a);
        near |= (w & 0xfffffu) - 0x7fffbu <= 10u;
    }
    if (near) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double z = (double)v[k] * q * (double)gamma[k] * (double)inv;
            const int e = max(__builtin_amdgcn_frexp_exp(z) - 1, -6) - 3;
            u[k] = (float)ldexp(rint(ldexp(z, -e)), e);
        }
    }
    return mx_codes(u);
}

struct rms_forward_args {
    const void *x, *res;
    int T, d;
    double inv_d, eps;
    const float *gamma;
    void *sum, *out;
    uint8_t *out8, *scale8, *keep8;
    float *keep_scale, *rstd;
};

#define RMS_THREADS(L) ((L) < 256 ? 256 : (L))
// Where the second half of a lane's eight elements lies: in fp32 a piece of the row further, so that the lanes' 16 bytes follow each other, but for codes,
// whose groups are neighbours' (4001 x 1023: forward 9.1 us, 9.8 with eight together; backward 12.0 and 13.4)
#define RMS_HALF(BF, CODES, L) ((BF) || (CODES) ? 4 : 4 * (L))

// h of eight elements (v), and to where it goes on
template <bool BF, int H>
__device__ __forceinline__ void add_residual(const rms_forward_args &a, const oct<BF> &x, const oct<BF> &r, size_t at, int n, float (&v)[8])
{
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = el8<BF>(x, k);
    if (a.res == nullptr) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += el8<BF>(r, k);
    const oct<BF> h = to_oct<BF>(v);
    if (BF) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = el8<BF>(h, k);
    }
    if (a.sum != nullptr && n > 0) st_oct<BF, H>(a.sum, at, n, h);
}
// what is written of eight elements of h once q is known
template <bool BF, bool EIGHT, int H>
__device__ __forceinline__ void write_normed(const rms_forward_args &a, const float (&v)[8], double q, const float (&gamma)[8], norm_small small, int t, int c)
{
    const int n = a.d - c;
    const size_t at = (size_t)t * a.d + c;
    const float r = (float)q;
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = v[k] * r * gamma[k];
    if (a.out != nullptr && n > 0) st_oct<BF, H>(a.out, at, n, to_oct<BF>(y));
    if (!EIGHT) return;
    if (a.out8 != nullptr) {  // (lanes behind the row's end take part in their group: zeros)
        uint32_t b;
        const u32x2_by codes = norm_to_mx(v, q, r, gamma, small, y, &b);
        if (n > 0) st_codes(a.out8, at, n, codes);
        if (n > 0 && c % KEEP8_MX_GROUP == 0) a.scale8[(size_t)t * ceil_div(a.d, KEEP8_MX_GROUP) + c / KEEP8_MX_GROUP] = (uint8_t)b;
    }
    if (a.keep8 != nullptr) {
        float s;
        const u32x2_by codes = to_int8(v, &s);
        if (n > 0) st_codes(a.keep8, at, n, codes);
        if (n > 0 && c % KEEP8_INT8_GROUP == 0) a.keep_scale[(size_t)t * ceil_div(a.d, KEEP8_INT8_GROUP) + c / KEEP8_INT8_GROUP] = s;
    }
}

template <bool BF, int N, int L, bool EIGHT>
__global__ __launch_bounds__(RMS_THREADS(L)) void rmsnorm_forward_kernel(const rms_forward_args a)
{
    constexpr int R = RMS_THREADS(L) / L, H = RMS_HALF(BF, EIGHT, L), W = H == 4 ? 8 : 4;
    __shared__ double red[2][16];
    const int l = threadIdx.x & (L - 1), step = gridDim.x * R, d = a.d;
    int t = blockIdx.x * R + threadIdx.x / L, turn = 0;
    if (t >= a.T) return;  // (L = 64: whole waves, nothing below waits for them)
    oct<BF> nx[N], nr[N];  // the next row
    auto ask = [&](int row) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = n * L * 8 + l * W;
            nx[n] = ld_oct<BF, H>(a.x, (size_t)row * d + c, d - c);
            if (a.res != nullptr) nr[n] = ld_oct<BF, H>(a.res, (size_t)row * d + c, d - c);
        }
    };
    ask(t);
    float g[N][8];
    norm_small small[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        ld_par8<H>(a.gamma, n * L * 8 + l * W, d - (n * L * 8 + l * W), g[n]);
        if (EIGHT) small[n] = norm_small(g[n]);
    }
    for (; t < a.T; t += step) {
        float v[N][8];
        double s = 0.0;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = n * L * 8 + l * W;
            add_residual<BF, H>(a, nx[n], nr[n], (size_t)t * d + c, d - c, v[n]);
        }
        if (t + step < a.T) ask(t + step);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < 8; ++k) s = fma((double)v[n][k], (double)v[n][k], s);
        // (LDS words in turn: the next row's sums do not meet those another wave still reads)
        const double q = rsqrt64(fma(row_total<L>(s, red[turn]), a.inv_d, a.eps));
        turn ^= 1;
        if (l == 0 && a.rstd != nullptr) a.rstd[t] = (float)q;
#pragma unroll
        for (int n = 0; n < N; ++n) write_normed<BF, EIGHT, H>(a, v[n], q, g[n], small[n], t, n * L * 8 + l * W);
    }
}

// Rows that do not fit the registers: a workgroup per row reads it twice (the second time from the caches; h from where it has been written).  4096 x 16384 bf16
// with a residual: forward 125 us, backward 126 and 60 for gamma's gradient, 4.3 TB/s of what has to be moved in the first two.
template <bool BF, bool EIGHT>
__global__ __launch_bounds__(256) void rmsnorm_forward_long_kernel(const rms_forward_args a)
{
    __shared__ double red[16];
    const int t = blockIdx.x, d = a.d, whole = ceil_div(d, 2048) * 2048;  // (all lanes to the end: groups are whole)
    const size_t row = (size_t)t * d;
    double s = 0.0;
    for (int c = threadIdx.x * 8; c < whole; c += 2048) {
        float v[8];
        const oct<BF> x = ld_oct<BF>(a.x, row + c, d - c), r = a.res != nullptr ? ld_oct<BF>(a.res, row + c, d - c) : x;
        add_residual<BF, 4>(a, x, r, row + c, d - c, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fma((double)v[k], (double)v[k], s);
    }
    const double q = rsqrt64(fma(row_total<256>(s, red), a.inv_d, a.eps));
    if (threadIdx.x == 0 && a.rstd != nullptr) a.rstd[t] = (float)q;
    rms_forward_args b = a;
    if (a.res != nullptr && a.sum != nullptr) b.x = a.sum, b.res = nullptr;  // (each lane reads what it has written)
    b.sum = nullptr;
    for (int c = threadIdx.x * 8; c < whole; c += 2048) {
        float v[8], g[8];
        const oct<BF> x = ld_oct<BF>(b.x, row + c, d - c), r = b.res != nullptr ? ld_oct<BF>(b.res, row + c, d - c) : x;
        add_residual<BF, 4>(b, x, r, row + c, d - c, v);
        ld_par<8>(a.gamma, c, d - c, g);
        write_normed<BF, EIGHT, 4>(b, v, q, g, EIGHT ? norm_small(g) : norm_small(), t, c);
    }
}

struct rms_backward_args {
    const void *h;          // rows, or ...
    const uint8_t *keep8;   // ... their 8-bit copy
    const float *keep_scale;
    const void *dout, *dsum;
    int T, d;
    const float *gamma, *rstd;
    void *dx;
    float *part;            // [workgroups][d]: their sums of dy xh
};
// eight elements of what is read of a row
template <bool BF, bool KEPT, int H>
struct rms_back_row {
    oct<BF> h, dy, ds;
    u32x2_by codes;
    float scale;
    __device__ __forceinline__ void ask(const rms_backward_args &a, int t, int c)
    {
        const size_t at = (size_t)t * a.d + c;
        const int n = a.d - c;
        if (KEPT) {
            codes = ld_codes(a.keep8, at, n);
            scale = n > 0 ? a.keep_scale[(size_t)t * ceil_div(a.d, KEEP8_INT8_GROUP) + c / KEEP8_INT8_GROUP] : 0.0f;
        } else h = ld_oct<BF, H>(a.h, at, n);
        dy = ld_oct<BF, H>(a.dout, at, n);
        if (a.dsum != nullptr) ds = ld_oct<BF, H>(a.dsum, at, n);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const
    {
        if (KEPT) from_int8(codes, scale, v);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = el8<BF>(h, k);
        }
    }
};

template <bool BF, int N, int L, bool KEPT>
__global__ __launch_bounds__(RMS_THREADS(L)) void rmsnorm_backward_kernel(const rms_backward_args a)
{
    constexpr int R = RMS_THREADS(L) / L, H = RMS_HALF(BF, KEPT, L), W = H == 4 ? 8 : 4;
    __shared__ float red[2][16];
    extern __shared__ __attribute__((aligned(16))) float cols[];  // L = 64: [3][N][64][8], the sums of waves 1 .. 3
    const int l = threadIdx.x & (L - 1), sub = threadIdx.x / L, d = a.d;
    float g[N][8], ag[N][8];
    rms_back_row<BF, KEPT, H> nx[N];  // the next row
    float nr = 0.0f;
    auto ask = [&](int t) {
#pragma unroll
        for (int n = 0; n < N; ++n) nx[n].ask(a, t, n * L * 8 + l * W);
        nr = a.rstd[t];
    };
    int t = blockIdx.x * R + sub, turn = 0;
    const int step = gridDim.x * R;
    if (t < a.T) ask(t);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        ld_par8<H>(a.gamma, n * L * 8 + l * W, d - (n * L * 8 + l * W), g[n]);
#pragma unroll
        for (int k = 0; k < 8; ++k) ag[n][k] = 0.0f;
    }
    for (; t < a.T; t += step) {  // (L = 64: whole waves; they meet the others behind the loop)
        const float r = nr;
        float xv[N][8], dv[N][8];
        oct<BF> ds[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            nx[n].values(xv[n]);
            ds[n] = nx[n].ds;
#pragma unroll
            for (int k = 0; k < 8; ++k) dv[n][k] = el8<BF>(nx[n].dy, k);
        }
        if (t + step < a.T) ask(t + step);
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int k = 0; k < 8; ++k) {  // (elements behind the row's end: all zero)
                xv[n][k] *= r;
                ag[n][k] = fmaf(dv[n][k], xv[n][k], ag[n][k]);
                dv[n][k] *= g[n][k];
                s = fmaf(dv[n][k], xv[n][k], s);
            }
        // (two sets of LDS words in turn: the next row's sums do not meet those another wave still reads)
        const float m = row_total<L>(s, red[turn]) / (float)d;
        turn ^= 1;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = n * L * 8 + l * W;
            if (c >= d) continue;
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = r * fmaf(-xv[n][k], m, dv[n][k]);
            if (a.dsum != nullptr) {
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] += el8<BF>(ds[n], k);
            }
            st_oct<BF, H>(a.dx, (size_t)t * d + c, d - c, to_oct<BF>(o));
        }
    }
    if (L == 64) {
        if (sub > 0) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < 8; ++k) cols[(((sub - 1) * N + n) * L + l) * 8 + k] = ag[n][k];
        }
        __syncthreads();
        if (sub > 0) return;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
                for (int k = 0; k < 8; ++k) ag[n][k] += cols[((w * N + n) * L + l) * 8 + k];
    }
    float *pg = a.part + (size_t)blockIdx.x * d;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = n * L * 8 + l * W;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int at = c + k + (k < 4 ? 0 : H - 4);
            if (at < d) pg[at] = ag[n][k];
        }
    }
}

template <bool BF, bool KEPT>
__global__ __launch_bounds__(256) void rmsnorm_backward_long_kernel(const rms_backward_args a)
{
    __shared__ float red[16];
    const int t = blockIdx.x, d = a.d;
    const float r = a.rstd[t];
    float s = 0.0f;
    auto terms = [&](int c, float (&xh)[8], float (&dv)[8], oct<BF> *ds) {
        rms_back_row<BF, KEPT, 4> o;
        float g[8];
        o.ask(a, t, c);
        o.values(xh);
        *ds = o.ds;
        ld_par<8>(a.gamma, c, d - c, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) xh[k] *= r, dv[k] = el8<BF>(o.dy, k) * g[k];
    };
    for (int c = threadIdx.x * 8; c < d; c += 2048) {
        float xh[8], dv[8];
        oct<BF> ds;
        terms(c, xh, dv, &ds);
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fmaf(dv[k], xh[k], s);
    }
    const float m = row_total<256>(s, red) / (float)d;
    for (int c = threadIdx.x * 8; c < d; c += 2048) {
        float xh[8], dv[8];
        oct<BF> ds;
        terms(c, xh, dv, &ds);
#pragma unroll
        for (int k = 0; k < 8; ++k) dv[k] = r * fmaf(-xh[k], m, dv[k]) + (a.dsum != nullptr ? el8<BF>(ds, k) : 0.0f);
        st_oct<BF>(a.dx, (size_t)t * d + c, d - c, to_oct<BF>(dv));
    }
}
// gamma's gradient of long rows: a thread per eight columns, a slice of the rows per workgroup (part as above).  In front of the kernel that writes
// dx, which may be where dsum is.
template <bool BF, bool KEPT>
__global__ __launch_bounds__(64) void rmsnorm_columns_kernel(rms_backward_args a)
{
    const int c = (blockIdx.x * 64 + threadIdx.x) * 8, d = a.d;
    if (c >= d) return;
    float ag[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    a.dsum = nullptr;
    for (int t = blockIdx.y; t < a.T; t += gridDim.y) {
        rms_back_row<BF, KEPT, 4> o;
        float v[8];
        o.ask(a, t, c);
        o.values(v);
        const float r = a.rstd[t];
#pragma unroll
        for (int k = 0; k < 8; ++k) ag[k] = fmaf(el8<BF>(o.dy, k), v[k] * r, ag[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (c + k < d) a.part[(size_t)blockIdx.y * d + c + k] = ag[k];
}

// dgamma = sums of n rows of part [n][d]: a workgroup takes 16 columns, 64 slices of the rows, joined across lanes and in LDS
__global__ __launch_bounds__(1024) void rmsnorm_join_kernel(const float *__restrict__ part, int n, int d, float *__restrict__ dgamma)
{
    __shared__ float red[16][16];
    const int cc = threadIdx.x & 15, k = threadIdx.x >> 4, c = blockIdx.x * 16 + cc;
    float s = 0.0f;
    for (int i0 = k; i0 < n && c < d; i0 += 64 * 8) {  // eight rows asked for together
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i0 + 64 * j < n ? part[(size_t)(i0 + 64 * j) * d + c] : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 48) == 0) red[threadIdx.x >> 6][cc] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || c >= d) return;
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += red[w][cc];
    dgamma[c] = s;
}

// Lanes that share a row of d elements, 8 each: a wave (16 each above 512: 4001 x 1023 in fp32, forward 9.0 us and backward 12.8, where four waves a row
// took 9.5 and 13.4), or a workgroup of 4, 8 or 16 waves (0: too long for them).  More elements a lane and fewer waves wait longer: 8192 x 4096 bf16 backward 47.8 us,
// with 16 each 51.5, 64 such rows forward 3.6 and 4.2; 2000 x 6000 fp32 backward 34.7 and 47.7.
static int rms_lanes(int d) { return d <= 1024 ? 64 : d <= 2048 ? 256 : d <= 4096 ? 512 : d <= 8192 ? 1024 : 0; }

#define RMS_L(B, K, X, grid, lds, s, ...)                                                                       \
    do {                                                                                                        \
        if (lanes == 64 && a.d <= 512) hipLaunchKernelGGL((K<B, 1, 64, X>), grid, dim3(256), lds, s, __VA_ARGS__); \
        else if (lanes == 64) hipLaunchKernelGGL((K<B, 2, 64, X>), grid, dim3(256), lds, s, __VA_ARGS__);       \
        else if (lanes == 256) hipLaunchKernelGGL((K<B, 1, 256, X>), grid, dim3(256), 0, s, __VA_ARGS__);       \
        else if (lanes == 512) hipLaunchKernelGGL((K<B, 1, 512, X>), grid, dim3(512), 0, s, __VA_ARGS__);       \
        else hipLaunchKernelGGL((K<B, 1, 1024, X>), grid, dim3(1024), 0, s, __VA_ARGS__);                       \
    } while (0)
#define RMS_RUN(K, x, ...)                          \
    do {                                            \
        if (bf && (x)) RMS_L(true, K, true, __VA_ARGS__);       \
        else if (bf) RMS_L(true, K, false, __VA_ARGS__);        \
        else if (x) RMS_L(false, K, true, __VA_ARGS__);         \
        else RMS_L(false, K, false, __VA_ARGS__);               \
    } while (0)
#define RMS_LONG(K, x, grid, threads, ...)                                                                         \
    do {                                                                                                  \
        if (bf && (x)) hipLaunchKernelGGL((K<true, true>), grid, dim3(threads), 0, s, __VA_ARGS__);           \
        else if (bf) hipLaunchKernelGGL((K<true, false>), grid, dim3(threads), 0, s, __VA_ARGS__);            \
        else if (x) hipLaunchKernelGGL((K<false, true>), grid, dim3(threads), 0, s, __VA_ARGS__);             \
        else hipLaunchKernelGGL((K<false, false>), grid, dim3(threads), 0, s, __VA_ARGS__);                   \
    } while (0)

hipError_t launch_rmsnorm_forward(const omega_ctx *ctx, const rmsnorm_forward &p, hipStream_t s)
{
    const bool bf = p.dtype == OMEGA_DTYPE_BF16, eight = p.out8 != nullptr || p.keep8 != nullptr;
    const int lanes = rms_lanes(p.d);
    const rms_forward_args a = {p.x, p.residual, p.T, p.d, 1.0 / p.d, (double)p.eps, p.gamma, p.sum, p.out, p.out8, p.scale8, p.keep8, p.keep_scale, p.rstd};
    if (lanes == 0) {
        RMS_LONG(rmsnorm_forward_long_kernel, eight, dim3(p.T), 256, a);
        return hipGetLastError();
    }
    // workgroups: what the device holds at once, 2048 lanes a compute unit, so that gamma is fetched once for several rows and the
    // next row is on its way (16384 x 2048 bf16: 48.8 us, a workgroup for every row 55.1; 16384 x 512: 13.6 and 16.2)
    const int all = lanes == 64 ? ceil_div(p.T, 4) : p.T, held = ctx->num_cus * (2048 / std::max(lanes, 256));
    RMS_RUN(rmsnorm_forward_kernel, eight, dim3(std::min(all, held)), 0, s, a);
    return hipGetLastError();
}

// Workgroups of the backward launch = rows of partial sums, which are written and read besides: as few as keep the memory busy.  A compute unit
// holds 3 of d <= 1024 (16384 x 1024 in bf16: 24.2 us, 2 of them 24.6, 4 of them 28.7), 2 of d <= 2048 (4096 x 2048: 15.2 us, 4 of them 17.5), 1 of
// longer rows (4096 x 4096: 25.6 us, 2 of them 27.2).  Small batches: two rows at least for each row of sums (2048 x 768: 7.5 us and 2.8 for the
// sums, with half as many 6.8 and 3.3).  Up to sixteen rows of a wave each, four of others: one workgroup, whose sums are dgamma (360 elements: 16 rows 5.0 us a call,
// as two launches 6.0; 32 rows 7.4 and 6.0; 4096 elements: 4 rows 6.0 and 7.0, 8 rows 8.6 and 7.0).
static int rms_backward_groups(const omega_ctx *ctx, int T, int d)
{
    const int lanes = rms_lanes(d), per = lanes == 64 ? 3 : lanes == 256 ? 2 : 1, rows = lanes == 64 ? 4 : 1;
    return T <= 4 * rows ? 1 : std::min(per * ctx->num_cus, ceil_div(T, 2 * rows));
}

size_t rmsnorm_backward_workspace(const omega_ctx *ctx, int T, int d) { return (size_t)rms_backward_groups(ctx, T, d) * d * sizeof(float); }

hipError_t launch_rmsnorm_backward(const omega_ctx *ctx, const rmsnorm_backward &p, void *ws, hipStream_t s)
{
    const bool bf = p.dtype == OMEGA_DTYPE_BF16, kept = p.keep8 != nullptr;
    int n = 0;
    if (p.T > 0) {
        const int lanes = rms_lanes(p.d);
        n = rms_backward_groups(ctx, p.T, p.d);
        const rms_backward_args a = {p.h, p.keep8, p.keep_scale, p.dout, p.dsum, p.T, p.d, p.gamma, p.rstd, p.dx, n == 1 ? p.dgamma : (float *)ws};
        if (lanes == 0) {
            RMS_LONG(rmsnorm_columns_kernel, kept, dim3(ceil_div(p.d, 512), n), 64, a);
            RMS_LONG(rmsnorm_backward_long_kernel, kept, dim3(p.T), 256, a);
        } else {
            const size_t lds = lanes == 64 ? (size_t)3 * (p.d <= 512 ? 512 : 1024) * sizeof(float) : 0;
            RMS_RUN(rmsnorm_backward_kernel, kept, dim3(n), lds, s, a);
        }
        if (n == 1) return hipGetLastError();
    }
    hipLaunchKernelGGL(rmsnorm_join_kernel, dim3(ceil_div(p.d, 16)), dim3(1024), 0, s, (const float *)ws, n, p.d, p.dgamma);
    return hipGetLastError();
}
