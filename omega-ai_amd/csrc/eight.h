// Eight consecutive elements of a row in a lane, and the two forms in which rows are held in 8 bits.
//
//   OMEGA_KEEP8_INT8  groups of 128 elements of a row: scale s = max(amax r, 2^-126) in fp32, r = 1 / 127 rounded to fp32, code = x / s to
//                     the nearest whole number, halves to even; value = code s
//   OMEGA_KEEP8_MX    groups of 32: s = 2^k, the smallest with amax <= 448 s (k >= -127), in a byte k + 127; code = x / s in e4m3 (four
//                     significant bits), to nearest even; value = code s
// A row's last group may be shorter.  A group that holds an infinity or no number has a scale that is no number (the byte 255) and comes back as
// such.  Sixteen lanes hold a group of 128, four a group of 32: its largest element is found in the lanes' own pipeline.
// Codes are those of the exact quotient: what fp32 arithmetic leaves in doubt next to a half is looked at again, which few elements need.
#pragma once
#include "rows.h"

#define KEEP8_INT8_GROUP 128
#define KEEP8_MX_GROUP 32

typedef uint32_t u32x2_by __attribute__((ext_vector_type(2), aligned(1)));

// eight elements as they lie in memory; in fp32 the second four may lie H elements behind the first
template <bool BF>
struct oct {
    uint32_t u[BF ? 4 : 8];
};
// from element i of p on, n elements to the row's end (behind it: zero; n <= 0: nothing is read)
template <bool BF, int H = 4>
__device__ __forceinline__ oct<BF> ld_oct(const void *p, size_t i, int n)
{
    oct<BF> r;
    const piece<BF> a = ld_piece<BF>(p, i, n);
#pragma unroll
    for (int k = 0; k < 4; ++k) r.u[k] = a.u[k];
    if (!BF) {
        const piece<BF> b = ld_piece<BF>(p, i + H, n - H);
#pragma unroll
        for (int k = 0; k < 4; ++k) r.u[(BF ? 0 : 4) + k] = b.u[k];
    }
    return r;
}
// as many fp32 parameters
template <int H>
__device__ __forceinline__ void ld_par8(const float *p, int i, int n, float (&v)[8])
{
    float a[4], b[4];
    ld_par<4>(p, i, n, a);
    ld_par<4>(p, i + H, n - H, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = a[k], v[4 + k] = b[k];
}
template <bool BF>
__device__ __forceinline__ float el8(const oct<BF> &r, int k)
{
    return __uint_as_float(!BF ? r.u[BF ? 0 : k] : k & 1 ? r.u[k >> 1] & 0xffff0000u : r.u[k >> 1] << 16);
}
template <bool BF>
__device__ __forceinline__ oct<BF> to_oct(const float (&v)[8])
{
    oct<BF> r;
#pragma unroll
    for (int k = 0; k < (BF ? 4 : 8); ++k) r.u[k] = BF ? pack_bf16(v[2 * k & 7], v[(2 * k + 1) & 7]) : __float_as_uint(v[k]);
    return r;
}
template <bool BF, int H = 4>
__device__ __forceinline__ void st_oct(void *p, size_t i, int n, const oct<BF> &r)
{
#pragma unroll
    for (int h = 0; h < (BF ? 1 : 2); ++h, i += H, n -= H) {
        constexpr int W = BF ? 8 : 4;
        if (n >= W) {
            u32x4_bf a;
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = r.u[BF ? k : 4 * h + k];
            if (BF) *(u32x4_bf *)((bf16_t *)p + i) = a;
            else *(u32x4_bf *)((float *)p + i) = a;
        } else {
#pragma unroll
            for (int k = 0; k < W; ++k)
                if (k < n) {
                    if (BF) ((bf16_t *)p)[i + k] = (bf16_t)(r.u[(k >> 1) & 3] >> (16 * (k & 1)));
                    else ((uint32_t *)p)[i + k] = r.u[BF ? 0 : 4 * h + (k & 3)];
                }
        }
    }
}
// eight codes, or the first four
template <int W = 8>
__device__ __forceinline__ u32x2_by ld_codes(const uint8_t *p, size_t i, int n)
{
    typedef uint32_t u32_by __attribute__((aligned(1)));
    u32x2_by r = {0u, 0u};
    if (n >= W) {
        if (W == 8) return *(const u32x2_by *)(p + i);
        r[0] = *(const u32_by *)(p + i);
        return r;
    }
#pragma unroll
    for (int k = 0; k < W; ++k)
        if (k < n) r[k >> 2] |= (uint32_t)p[i + k] << (8 * (k & 3));
    return r;
}
__device__ __forceinline__ void st_codes(uint8_t *p, size_t i, int n, u32x2_by r)
{
    if (n >= 8) {
        *(u32x2_by *)(p + i) = r;
        return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k < n) p[i + k] = (uint8_t)(r[k >> 2] >> (8 * (k & 3)));
}

template <int CTRL>
__device__ __forceinline__ uint32_t lane_max(uint32_t v)
{
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true));
}
// the largest over a group's 4 or 16 lanes, in all of them
__device__ __forceinline__ uint32_t max_over_4(uint32_t v) { return lane_max<0x4E>(lane_max<0xB1>(v)); }  // quad_perm [1,0,3,2], [2,3,0,1]
__device__ __forceinline__ uint32_t max_over_16(uint32_t v) { return lane_max<0x140>(lane_max<0x141>(max_over_4(v))); }  // row_half_mirror, row_mirror
// magnitudes as whole numbers: their order is that of the values, and no number is above infinity
__device__ __forceinline__ uint32_t magnitude(const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
    return m;
}

// Codes of eight elements of a group of 128 and the group's scale (the same in its 16 lanes).
// m = x (1/s) + 1.5 2^23, rounded once, holds the whole number in its low bits; r = x - q s is exact (a multiple of the lower of x's and s's last
// places, below s).  q is the nearest unless |r| reaches s / 2, which a quotient next to a half may do by the error of 1/s: then it moves on by one,
// on a half where it is odd.  (2 |r| against s: half of a scale below 2^-125 need not be a number of fp32.)
__device__ __forceinline__ u32x2_by to_int8(const float (&v)[8], float *scale)
{
    const uint32_t most = max_over_16(magnitude(v));
    const float s = fmaxf(__uint_as_float(most) * 0x1.020408p-7f, 0x1p-126f), inv = __builtin_amdgcn_rcpf(s);
    uint32_t m[8];
    float r[8], worst = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float t = fmaf(v[k], inv, 0x1.8p23f);
        m[k] = __float_as_uint(t);
        r[k] = fmaf(-(t - 0x1.8p23f), s, v[k]);
        worst = fmaxf(worst, fabsf(r[k]));
    }
    if (worst + worst >= s) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float a = fabsf(r[k]) + fabsf(r[k]);
            if (a > s || (a == s && (m[k] & 1))) m[k] += r[k] < 0.0f ? -1 : 1;
        }
    }
    const bool none = most >= 0x7f800000u;
    *scale = none ? __builtin_nanf("") : s;
    u32x2_by c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(m[4 * h + 1], m[4 * h], 0x0c0c0400u), hi = __builtin_amdgcn_perm(m[4 * h + 3], m[4 * h + 2], 0x0c0c0400u);
        c[h] = none ? 0u : lo | hi << 16;
    }
    return c;
}
__device__ __forceinline__ void from_int8(u32x2_by c, float s, float (&v)[8])
{
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (float)(int8_t)(c[k >> 2] >> (8 * (k & 3))) * s;
}

// Byte of the scale of a group of 32 whose largest magnitude is `most`
__device__ __forceinline__ uint32_t mx_scale(uint32_t most)
{
    if (most >= 0x7f800000u) return 255u;
    return (uint32_t)max(0, (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1 : 0));  // 448 = 1.75 2^8
}
__device__ __forceinline__ float mx_inverse(uint32_t b) { return __uint_as_float((254u - min(b, 253u)) << 23); }  // 2^-k
__device__ __forceinline__ float mx_value(uint32_t b) { return __uint_as_float(b == 255u ? 0x7fc00000u : b ? b << 23 : 0x400000u); }
__device__ __forceinline__ u32x2_by mx_codes(const float (&u)[8])
{
    u32x2_by c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(u[4 * h], u[4 * h + 1], 0, false);
        c[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(u[4 * h + 2], u[4 * h + 3], w, true);
    }
    return c;
}
// Codes of eight elements of a group of 32 and the group's scale (the same in its 4 lanes).  A power of two leaves x / s exact.
__device__ __forceinline__ u32x2_by to_mx(const float (&v)[8], uint32_t *scale)
{
    const uint32_t b = mx_scale(max_over_4(magnitude(v)));
    const float inv = mx_inverse(b);
    float u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = b == 255u ? 0.0f : v[k] * inv;
    *scale = b;
    return mx_codes(u);
}
__device__ __forceinline__ void from_mx(u32x2_by c, uint32_t b, float (&v)[8])
{
    const float s = mx_value(b);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
        v[4 * h] = lo[0] * s, v[4 * h + 1] = lo[1] * s, v[4 * h + 2] = hi[0] * s, v[4 * h + 3] = hi[1] * s;
    }
}
