// Rows of fp32 or bf16 elements in pieces of 16 bytes, at any alignment of the element, and sums over a wave: shared by the norms and by
// the 8-bit copies.
#pragma once
#include "common.h"

// 16 bytes at the alignment of an element
typedef uint32_t u32x4_bf __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_el __attribute__((ext_vector_type(4), aligned(4)));

// W elements (8 of bf16, 4 of fp32) as they lie in memory
template <bool BF>
struct piece {
    static constexpr int W = BF ? 8 : 4;
    uint32_t u[4];
};
// piece from element i of p on, `n` elements of it (the rest: zero; n <= 0: nothing is read)
template <bool BF>
__device__ __forceinline__ piece<BF> ld_piece(const void *p, size_t i, int n)
{
    piece<BF> r;
    r.u[0] = r.u[1] = r.u[2] = r.u[3] = 0u;
    if (n >= piece<BF>::W) {
        const u32x4_bf v = BF ? *(const u32x4_bf *)((const bf16_t *)p + i) : *(const u32x4_bf *)((const float *)p + i);
        r.u[0] = v[0], r.u[1] = v[1], r.u[2] = v[2], r.u[3] = v[3];
    } else {
#pragma unroll
        for (int k = 0; k < piece<BF>::W; ++k)
            if (k < n) {
                if (BF) r.u[(k >> 1) & 3] |= (uint32_t)((const bf16_t *)p)[i + k] << (16 * (k & 1));
                else r.u[k & 3] = ((const uint32_t *)p)[i + k];
            }
    }
    return r;
}
template <bool BF>
__device__ __forceinline__ float el(const piece<BF> &r, int k)
{
    return __uint_as_float(!BF ? r.u[k & 3] : k & 1 ? r.u[(k >> 1) & 3] & 0xffff0000u : r.u[(k >> 1) & 3] << 16);
}
// two floats -> two bf16 (round to nearest even) in one instruction
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const b2 r = __builtin_convertvector(f2{lo, hi}, b2);
    return *(const uint32_t *)&r;
}
template <bool BF>
__device__ __forceinline__ void st_piece(void *p, size_t i, int n, const float (&v)[piece<BF>::W])
{
    constexpr int W = piece<BF>::W;
    u32x4_bf u;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        u[k] = BF ? pack_bf16(v[(2 * k) % W], v[(2 * k + 1) % W]) : __float_as_uint(v[k]);
    if (n >= W) {
        if (BF) *(u32x4_bf *)((bf16_t *)p + i) = u;
        else *(u32x4_bf *)((float *)p + i) = u;
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k)
            if (k < n) {
                if (BF) ((bf16_t *)p)[i + k] = f32_to_bf16(v[k]);
                else ((float *)p)[i + k] = v[k];
            }
    }
}
// W fp32 parameters from element i on (n of them)
template <int W>
__device__ __forceinline__ void ld_par(const float *p, int i, int n, float (&v)[W])
{
    if (n >= W) {
#pragma unroll
        for (int k = 0; k < W; k += 4) {
            const f32x4_el u = *(const f32x4_el *)(p + i + k);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k + j] = u[j];
        }
    } else {
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = k < n ? p[i + k] : 0.0f;
    }
}
template <bool BF>
__device__ __forceinline__ float ld1(const void *p, size_t i)
{
    return BF ? bf16_to_f32(((const bf16_t *)p)[i]) : ((const float *)p)[i];
}
template <bool BF>
__device__ __forceinline__ void st1(void *p, size_t i, float v)
{
    if (BF) ((bf16_t *)p)[i] = f32_to_bf16(v);
    else ((float *)p)[i] = v;
}

// sum over a wave, in every lane: within rows of 16 lanes, then across them, without a trip through LDS
__device__ __forceinline__ float wave_sum(float s)
{
#define ROW_DPP(ctrl, rows) s += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(s), ctrl, rows, 0xf, false))
    ROW_DPP(0x111, 0xf);  // from the lane 1, 2, 4, 8 to the left
    ROW_DPP(0x112, 0xf);
    ROW_DPP(0x114, 0xf);
    ROW_DPP(0x118, 0xf);
    ROW_DPP(0x142, 0xa);  // the last lane of rows 0 and 2 into rows 1 and 3
    ROW_DPP(0x143, 0xc);  // lane 31 into rows 2 and 3
#undef ROW_DPP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), 63));
}
