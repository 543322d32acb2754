// Token embedding and its gradient.
//
//   forward   out[t,:] = scale * table[ids[t],:]
//   backward  dtable[v,:] = scale * sum_{t : ids[t] = v} dout[t,:]  in ascending t
//
// The gradient sums the tokens of a row in a fixed order instead of adding rows with atomics: the tokens are sorted by id
// (a stable counting sort, index_kernel), then every row of the table is written once, from the run of tokens that belongs to
// it (rows_kernel).  Runs of hot ids are cut into aligned blocks of 32 sorted places whose sums other workgroups form first
// (block_kernel), and blocks of 32 such blocks once more, so that no workgroup adds more than about 64 rows by itself.
// Bound: bytes - dout is read once, dtable written once (every row: most of a large vocabulary has no token in a batch).
#include <algorithm>

#include "common.h"

#define IDX_IDS 512      // ids of a workgroup of the index kernel
#define IDX_WAVES 16
#define EMB_BLOCK 32     // sorted places of a partial sum

typedef __attribute__((ext_vector_type(4))) float f32x4;

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
template <bool BF>
__device__ __forceinline__ f32x4 ld4(const void *p, size_t i)
{
    if (BF) {
        const uint2 u = *(const uint2 *)((const bf16_t *)p + i);
        return f32x4{__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u)};
    }
    return *(const f32x4 *)((const float *)p + i);
}
template <bool BF>
__device__ __forceinline__ void st4(void *p, size_t i, f32x4 v)
{
    if (BF) {
        uint2 u;
        u.x = (uint32_t)f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16;
        u.y = (uint32_t)f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16;
        *(uint2 *)((bf16_t *)p + i) = u;
    } else {
        *(f32x4 *)((float *)p + i) = v;
    }
}

// ---- forward: a workgroup per 4 rows x 1024 columns (VEC: 4 columns a thread and step) ----
template <bool BF, bool VEC>
__global__ __launch_bounds__(256) void embedding_forward_kernel(const void *__restrict__ table, int V, int d, const int32_t *__restrict__ ids, int T,
                                                                float scale, void *__restrict__ out)
{
    constexpr int W = VEC ? 4 : 1;
    const int t0 = blockIdx.x * 4;
    for (int c = (blockIdx.y * 256 + threadIdx.x) * W; c < d; c += gridDim.y * 256 * W) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = t0 + r;
            if (t >= T) break;
            const int id = ids[t];
            const bool held = id >= 0 && id < V;
            if (VEC) {
                f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                if (held) v = ld4<BF>(table, (size_t)id * d + c) * scale;
                st4<BF>(out, (size_t)t * d + c, v);
            } else {
                st1<BF>(out, (size_t)t * d + c, held ? ld1<BF>(table, (size_t)id * d + c) * scale : 0.0f);
            }
        }
    }
}

hipError_t launch_embedding_forward(const void *table, int dtype, int V, int d, const int32_t *ids, int T, float scale, void *out, hipStream_t s)
{
    const bool bf = dtype == OMEGA_DTYPE_BF16;
    const bool vec = d % 4 == 0 && (((uintptr_t)table | (uintptr_t)out) % (bf ? 8 : 16)) == 0;
    const dim3 grid(ceil_div(T, 4), std::min(ceil_div(d, vec ? 1024 : 256), 64));
#define EMB_FWD(B, VV) hipLaunchKernelGGL((embedding_forward_kernel<B, VV>), grid, dim3(256), 0, s, table, V, d, ids, T, scale, out)
    if (bf) { if (vec) EMB_FWD(true, true); else EMB_FWD(true, false); }
    else { if (vec) EMB_FWD(false, true); else EMB_FWD(false, false); }
#undef EMB_FWD
    return hipGetLastError();
}

// ---- backward ----
// Stable counting sort by id.  A workgroup owns IDX_IDS ids; its sixteen waves each walk a sixteenth of the tokens, in order, twice: the
// first time they count the tokens of each of its ids (a counter per wave and id in LDS) and those of smaller ids (where its run of the
// sorted list begins), the second time they place their tokens.  Places depend on nothing but the ids: no communication between
// workgroups, one launch.  off[v] = first place of id v (V+1 entries, off[V] = tokens with an id), perm[place] = token,
// sid[place] = its id.  Tokens of a 64-token step with one id are ranked by a ballot.
__global__ __launch_bounds__(IDX_WAVES * 64) void embedding_index_kernel(const int32_t *__restrict__ ids, int T, int V, int32_t *__restrict__ off,
                                                                         int32_t *__restrict__ perm, int32_t *__restrict__ sid)
{
    __shared__ int32_t cnt[IDX_IDS][IDX_WAVES + 1];  // (a column of padding: a thread's row starts in a bank of its own)
    __shared__ int32_t below[IDX_WAVES], sums[IDX_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lo = blockIdx.x * IDX_IDS, n_ids = min(IDX_IDS, V - lo);
    for (int i = tid; i < IDX_IDS * (IDX_WAVES + 1); i += IDX_WAVES * 64) (&cnt[0][0])[i] = 0;
    __syncthreads();
    const int seg = ceil_div(ceil_div(T, 64), IDX_WAVES) * 64;
    const int first = min(wave * seg, T), last = min(first + seg, T);
    int nb = 0;
    for (int t = first; t < last; t += 256) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) id[u] = t + 64 * u + lane < last ? ids[t + 64 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (id[u] >= 0 && id[u] < lo) ++nb;
            const int k = id[u] - lo;
            if (id[u] >= lo && k < n_ids) atomicAdd(&cnt[k][wave], 1);  // (whole numbers: the order does not matter)
        }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) nb += __shfl_xor(nb, m, 64);
    if (lane == 0) below[wave] = nb;
    __syncthreads();
    // counts -> first places: a thread sums its id's sixteen counters, then a scan over the ids
    int mine = 0, incl = 0;
    if (tid < IDX_IDS) {
        for (int w = 0; w < IDX_WAVES; ++w) mine += cnt[tid][w];
        incl = mine;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(incl, m, 64);
            if (lane >= m) incl += o;
        }
        if (lane == 63) sums[wave] = incl;
    }
    __syncthreads();
    if (tid < IDX_IDS) {
        int at = incl - mine;
        for (int w = 0; w < IDX_WAVES; ++w) at += below[w];
        for (int w = 0; w < wave; ++w) at += sums[w];
        if (tid < n_ids) off[lo + tid] = at;
        if (tid == n_ids - 1 && lo + n_ids == V) off[V] = at + mine;
        for (int w = 0; w < IDX_WAVES; ++w) {
            const int n = cnt[tid][w];
            cnt[tid][w] = at;
            at += n;
        }
    }
    __syncthreads();
    const unsigned long long before = ((unsigned long long)1 << lane) - 1;
    for (int t = first; t < last; t += 256) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) id[u] = t + 64 * u + lane < last ? ids[t + 64 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = id[u] - lo;
            const bool in = id[u] >= lo && k < n_ids;
            unsigned long long left = __ballot(in);
            while (left) {
                const int leader = __ffsll((long long)left) - 1;
                const int kk = __shfl(k, leader, 64);
                const unsigned long long same = __ballot(in && k == kk);
                volatile int32_t *place = &cnt[kk][wave];  // (a counter belongs to its wave; lanes of a wave read it in turn)
                const int at = *place;
                if (in && k == kk) {
                    const int p = at + __popcll(same & before);
                    perm[p] = t + 64 * u + lane;
                    sid[p] = id[u];
                }
                __builtin_amdgcn_wave_barrier();
                if (lane == leader) *place = at + __popcll(same);
                __builtin_amdgcn_wave_barrier();
                left &= ~same;
            }
        }
    }
}

// Sums of EMB_BLOCK sorted places that belong to one id, unscaled fp32: part[block,:].  LEVEL 1: rows of dout through perm; LEVEL 2: sums of
// EMB_BLOCK blocks of level 1.  Blocks with more than one id are left alone (nobody reads them).
template <bool BF, bool VEC, int LEVEL>
__global__ __launch_bounds__(64) void embedding_block_kernel(const void *__restrict__ src, int d, int V, const int32_t *__restrict__ off,
                                                             const int32_t *__restrict__ perm, const int32_t *__restrict__ sid, float *__restrict__ part)
{
    constexpr int SPAN = LEVEL == 1 ? EMB_BLOCK : EMB_BLOCK * EMB_BLOCK;
    constexpr int W = VEC ? 4 : 1;
    const int b = blockIdx.x, p0 = b * SPAN;
    if (p0 + SPAN > off[V] || sid[p0] != sid[p0 + SPAN - 1]) return;
    const int c = (blockIdx.y * 64 + threadIdx.x) * W;
    if (c >= d) return;
    f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 16
    for (int i = 0; i < EMB_BLOCK; ++i) {
        const size_t row = LEVEL == 1 ? (size_t)perm[p0 + i] : (size_t)(b * EMB_BLOCK + i);
        if (LEVEL == 1) {
            if (VEC) a += ld4<BF>(src, row * d + c);
            else a[0] += ld1<BF>(src, row * d + c);
        } else {
            if (VEC) a += ld4<false>(src, row * d + c);
            else a[0] += ld1<false>(src, row * d + c);
        }
    }
    if (VEC) st4<false>(part, (size_t)b * d + c, a);
    else part[(size_t)b * d + c] = a[0];
}

// One row of the table after the other: the sum of its run of sorted places.
#define EMB_ROWS 16
template <bool BF, bool VEC, bool GBF>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const void *__restrict__ dout, int V, int d, float scale, int accumulate,
                                                             const int32_t *__restrict__ off, const int32_t *__restrict__ perm,
                                                             const float *__restrict__ part1, const float *__restrict__ part2, void *__restrict__ dtable)
{
    constexpr int W = VEC ? 4 : 1;
    const int v0 = blockIdx.x * EMB_ROWS, c = (blockIdx.y * 256 + threadIdx.x) * W;
    if (c >= d) return;
    int p1 = off[v0];
    for (int v = v0; v < min(v0 + EMB_ROWS, V); ++v) {
        const int p0 = p1;
        p1 = off[v + 1];
        if (accumulate && p0 == p1) continue;
        f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p = p0; p < p1;) {
            if (part2 != nullptr && p % (EMB_BLOCK * EMB_BLOCK) == 0 && p + EMB_BLOCK * EMB_BLOCK <= p1) {
                const size_t i = (size_t)(p / (EMB_BLOCK * EMB_BLOCK)) * d + c;
                if (VEC) a += ld4<false>(part2, i);
                else a[0] += part2[i];
                p += EMB_BLOCK * EMB_BLOCK;
            } else if (part1 != nullptr && p % EMB_BLOCK == 0 && p + EMB_BLOCK <= p1) {
                const size_t i = (size_t)(p / EMB_BLOCK) * d + c;
                if (VEC) a += ld4<false>(part1, i);
                else a[0] += part1[i];
                p += EMB_BLOCK;
            } else {
                const size_t i = (size_t)perm[p] * d + c;
                if (VEC) a += ld4<BF>(dout, i);
                else a[0] += ld1<BF>(dout, i);
                ++p;
            }
        }
        a *= scale;
        const size_t o = (size_t)v * d + c;
        if (VEC) {
            if (accumulate) a += ld4<GBF>(dtable, o);
            st4<GBF>(dtable, o, a);
        } else {
            if (accumulate) a[0] += ld1<GBF>(dtable, o);
            st1<GBF>(dtable, o, a[0]);
        }
    }
}

// off [V+1] | perm [T] | sid [T] | part1 [T/32, d] | part2 [T/1024, d]
struct emb_layout {
    size_t perm, sid, part1, part2, bytes;
    int n1, n2;
};
static emb_layout emb_layout_of(int V, int d, int T)
{
    emb_layout l;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    l.n1 = T / EMB_BLOCK;
    l.n2 = T / (EMB_BLOCK * EMB_BLOCK);
    l.perm = up(((size_t)V + 1) * 4);
    l.sid = l.perm + up((size_t)T * 4);
    l.part1 = l.sid + up((size_t)T * 4);
    l.part2 = l.part1 + up((size_t)l.n1 * d * 4);
    l.bytes = l.part2 + up((size_t)l.n2 * d * 4);
    return l;
}

size_t embedding_backward_workspace(int V, int d, int T) { return emb_layout_of(V, d, T).bytes; }

template <bool BF, bool VEC>
static void emb_blocks(const emb_layout &l, const void *dout, int d, int V, const int32_t *off, const int32_t *perm, const int32_t *sid, float *part1,
                       float *part2, hipStream_t s)
{
    const int gy = ceil_div(d, VEC ? 256 : 64);
    if (l.n1 > 0) hipLaunchKernelGGL((embedding_block_kernel<BF, VEC, 1>), dim3(l.n1, gy), dim3(64), 0, s, dout, d, V, off, perm, sid, part1);
    if (l.n2 > 0) hipLaunchKernelGGL((embedding_block_kernel<BF, VEC, 2>), dim3(l.n2, gy), dim3(64), 0, s, (const void *)part1, d, V, off, perm, sid, part2);
}

hipError_t launch_embedding_backward(const int32_t *ids, int T, const void *dout, int dtype, int V, int d, float scale, bool accumulate, void *dtable,
                                     int grad_dtype, void *ws, hipStream_t s)
{
    const emb_layout l = emb_layout_of(V, d, T);
    unsigned char *base = (unsigned char *)ws;
    int32_t *off = (int32_t *)base, *perm = (int32_t *)(base + l.perm), *sid = (int32_t *)(base + l.sid);
    float *part1 = l.n1 > 0 ? (float *)(base + l.part1) : nullptr, *part2 = l.n2 > 0 ? (float *)(base + l.part2) : nullptr;
    const bool bf = dtype == OMEGA_DTYPE_BF16, gbf = grad_dtype == OMEGA_DTYPE_BF16;
    const bool vec = d % 4 == 0 && (uintptr_t)dout % (bf ? 8 : 16) == 0 && (uintptr_t)dtable % (gbf ? 8 : 16) == 0;
    hipLaunchKernelGGL(embedding_index_kernel, dim3(ceil_div(V, IDX_IDS)), dim3(IDX_WAVES * 64), 0, s, ids, T, V, off, perm, sid);
    if (bf) { if (vec) emb_blocks<true, true>(l, dout, d, V, off, perm, sid, part1, part2, s); else emb_blocks<true, false>(l, dout, d, V, off, perm, sid, part1, part2, s); }
    else { if (vec) emb_blocks<false, true>(l, dout, d, V, off, perm, sid, part1, part2, s); else emb_blocks<false, false>(l, dout, d, V, off, perm, sid, part1, part2, s); }
    const dim3 grid(ceil_div(V, EMB_ROWS), ceil_div(d, vec ? 1024 : 256));
#define EMB_ROWS_K(B, VV, G) \
    hipLaunchKernelGGL((embedding_rows_kernel<B, VV, G>), grid, dim3(256), 0, s, dout, V, d, scale, accumulate ? 1 : 0, off, perm, part1, part2, dtable)
#define EMB_ROWS_V(B, G) do { if (vec) EMB_ROWS_K(B, true, G); else EMB_ROWS_K(B, false, G); } while (0)
    if (bf) { if (gbf) EMB_ROWS_V(true, true); else EMB_ROWS_V(true, false); }
    else { if (gbf) EMB_ROWS_V(false, true); else EMB_ROWS_V(false, false); }
#undef EMB_ROWS_V
#undef EMB_ROWS_K
    return hipGetLastError();
}
