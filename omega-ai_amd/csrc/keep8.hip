// Rows kept in 8 bits (eight.h describes the two forms) and brought back: activations between a forward pass and its backward pass.
// A lane takes eight elements, with no loop: the groups' largest elements are found among neighbours, and loads of many waves are in flight.  Bound: bytes (x in,
// codes and scales out, and the other way round): 16384 x 4096 bf16, whole numbers: saved in 43.4 us (4.7 TB/s), brought back in 30.7 (6.6 TB/s); 2999 x 1333 fp32 in
// e4m3: 5.8 and 5.7 us; 16384 x 4096 fp32, either form: 57 and 65 us (5.9 and 5.2 TB/s).
#include "eight.h"

// Row of a lane and eight times its place there, `per` lanes a row (a launch holds at most 2^30 lanes: the workgroup's division is of 32 bits)
__device__ __forceinline__ int keep8_lane(int per, int *c)
{
    const uint32_t i = blockIdx.x * 256u, t = i / (uint32_t)per;  // (the same in a workgroup)
    uint32_t r = i - t * (uint32_t)per + threadIdx.x, q = 0;
    if (per < 256) q = r / (uint32_t)per;
    else if (r >= (uint32_t)per) q = 1;
    *c = (int)(r - q * (uint32_t)per) * 8;
    return (int)(t + q);
}

template <bool BF, bool MX>
__global__ __launch_bounds__(256) void keep8_save_kernel(const void *__restrict__ x, int T, int d, uint8_t *__restrict__ codes, void *__restrict__ scales)
{
    const int per = ceil_div(d, KEEP8_INT8_GROUP) * 16;  // lanes of a row: whole groups of 128
    int c;
    const int row = keep8_lane(per, &c);
    if (row >= T) return;  // (whole groups of 16 lanes)
    const size_t t = row;
    const oct<BF> o = ld_oct<BF>(x, t * d + c, d - c);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = el8<BF>(o, k);
    if (MX) {
        uint32_t b;
        const u32x2_by q = to_mx(v, &b);
        st_codes(codes, t * d + c, d - c, q);
        if (c % KEEP8_MX_GROUP == 0 && c < d) ((uint8_t *)scales)[t * ceil_div(d, KEEP8_MX_GROUP) + c / KEEP8_MX_GROUP] = (uint8_t)b;
    } else {
        float s;
        const u32x2_by q = to_int8(v, &s);
        st_codes(codes, t * d + c, d - c, q);
        if (c % KEEP8_INT8_GROUP == 0) ((float *)scales)[t * (per / 16) + c / KEEP8_INT8_GROUP] = s;
    }
}

// (of fp32 rows a lane takes four elements: 16 bytes again, which the lanes write one behind the other; eight took 7.2 us in place of 5.7 for
// 2999 x 1333)
template <bool BF, bool MX>
__global__ __launch_bounds__(256) void keep8_load_kernel(const uint8_t *__restrict__ codes, const void *__restrict__ scales, int T, int d, void *__restrict__ out)
{
    constexpr int W = piece<BF>::W;
    int c;
    const int row = keep8_lane(ceil_div(d, W), &c);
    if (row >= T) return;
    c = c / 8 * W;
    const size_t t = row;
    const u32x2_by q = ld_codes<W>(codes, t * d + c, d - c);
    float v[8], o[W];
    if (MX) from_mx(q, ((const uint8_t *)scales)[t * ceil_div(d, KEEP8_MX_GROUP) + c / KEEP8_MX_GROUP], v);
    else from_int8(q, ((const float *)scales)[t * ceil_div(d, KEEP8_INT8_GROUP) + c / KEEP8_INT8_GROUP], v);
#pragma unroll
    for (int k = 0; k < W; ++k) o[k] = v[k];
    st_piece<BF>(out, t * d + c, d - c, o);
}

// Rows of a launch of at most 2^30 lanes: the others in further ones
static constexpr int keep8_rows(int per) { return (1 << 30) / per; }
static_assert(keep8_rows(1) > 0 && keep8_rows(1 << 18) > 0 && (long long)keep8_rows(1) + 255 < 1LL << 31, "the narrowest and the widest rows, the last workgroup's lanes");
#define KEEP8_RUN(K, grid, ...)                                                                          \
    do {                                                                                                 \
        if (bf && mx) hipLaunchKernelGGL((K<true, true>), grid, dim3(256), 0, s, __VA_ARGS__);            \
        else if (bf) hipLaunchKernelGGL((K<true, false>), grid, dim3(256), 0, s, __VA_ARGS__);            \
        else if (mx) hipLaunchKernelGGL((K<false, true>), grid, dim3(256), 0, s, __VA_ARGS__);            \
        else hipLaunchKernelGGL((K<false, false>), grid, dim3(256), 0, s, __VA_ARGS__);                   \
    } while (0)

hipError_t launch_keep8_save(const void *x, int dtype, int T, int d, int form, uint8_t *codes, void *scales, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16, mx = form == OMEGA_KEEP8_MX;
    const int per = ceil_div(d, KEEP8_INT8_GROUP) * 16, rows = keep8_rows(per);
    const size_t es = bf ? 2 : 4, groups = mx ? ceil_div(d, KEEP8_MX_GROUP) : (size_t)ceil_div(d, KEEP8_INT8_GROUP) * 4;
    for (int t = 0; t < T; t += rows) {
        const int n = T - t < rows ? T - t : rows;
        KEEP8_RUN(keep8_save_kernel, dim3((uint32_t)(((size_t)n * per + 255) / 256)), (const char *)x + (size_t)t * d * es, n, d, codes + (size_t)t * d,
                  (void *)((char *)scales + (size_t)t * groups));
    }
    return hipGetLastError();
}

hipError_t launch_keep8_load(const uint8_t *codes, const void *scales, int form, int T, int d, void *out, int dtype, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16, mx = form == OMEGA_KEEP8_MX;
    const int per = ceil_div(d, bf ? 8 : 4), rows = keep8_rows(per);
    const size_t es = bf ? 2 : 4, groups = mx ? ceil_div(d, KEEP8_MX_GROUP) : (size_t)ceil_div(d, KEEP8_INT8_GROUP) * 4;
    for (int t = 0; t < T; t += rows) {
        const int n = T - t < rows ? T - t : rows;
        KEEP8_RUN(keep8_load_kernel, dim3((uint32_t)(((size_t)n * per + 255) / 256)), codes + (size_t)t * d, (const void *)((const char *)scales + (size_t)t * groups), n, d,
                  (void *)((char *)out + (size_t)t * d * es));
    }
    return hipGetLastError();
}
