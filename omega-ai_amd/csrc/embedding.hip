// Token embedding and its gradient.
//
//   forward   out[t,:] = scale * table[ids[t],:]
//   backward  dtable[v,:] = scale * sum_{t : ids[t] = v} dout[t,:]  in ascending t
//
// The gradient sums the tokens of a row in a fixed order instead of adding rows with atomics: the tokens are sorted by id
// (a stable counting sort, index_kernel), then every row of the table is written once, from the run of tokens that belongs to
// it (rows_kernel).  Runs of hot ids are cut into aligned blocks of 64 sorted places whose sums other workgroups form first
// (block_kernel), in large batches blocks of 64 such blocks once more.
// Bound: bytes - dout is read once, dtable written once (every row: most of a large vocabulary has no token in a batch).
#include <algorithm>

#include "common.h"

#define IDX_BITS 9
#define IDX_IDS (1 << IDX_BITS)  // ids of a workgroup of the index kernel
#define IDX_WAVES 16
#define IDX_NOTES 1024    // tokens a wave of the index kernel can note
#define EMB_BLOCK 64     // sorted places of a partial sum
#define EMB_LAUNCH_ROWS (1 << 22)  // rows of a launch (whose lanes in x are counted in 32 bits), a multiple of EMB_ROWS

typedef __attribute__((ext_vector_type(4))) float f32x4;
// four elements at the alignment of one
typedef uint32_t u32x2_el __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_el __attribute__((ext_vector_type(4), aligned(4)));

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
// Four columns of a row of d elements at p: `w` .. w + 3, all there.  TINY (rows of less than four): columns 0 .. d - 1, the rest zero.
template <bool BF, bool TINY>
__device__ __forceinline__ f32x4 ld4(const void *p, size_t row, int d, int w)
{
    if (TINY) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < d) v[k] = ld1<BF>(p, row * d + k);
        return v;
    }
    const size_t i = row * d + w;
    if (BF) {
        const u32x2_el u = *(const u32x2_el *)((const bf16_t *)p + i);
        return f32x4{__uint_as_float(u[0] << 16), __uint_as_float(u[0] & 0xffff0000u), __uint_as_float(u[1] << 16), __uint_as_float(u[1] & 0xffff0000u)};
    }
    const f32x4_el v = *(const f32x4_el *)((const float *)p + i);
    return f32x4{v[0], v[1], v[2], v[3]};
}
// The thread's columns c .. c + 3 of a row.  A row's last columns, fewer than four, are read as the four that end the row (w), so that every
// lane's loads are whole and none waits for another's; of those only the thread's own are stored.
struct emb_cols {
    int c, w;
    __device__ __forceinline__ emb_cols(int c0, int d) : c(c0), w(min(c0, max(d - 4, 0))) {}
};
template <bool BF, bool NT = false>
__device__ __forceinline__ void st4(void *p, size_t row, int d, const emb_cols &x, f32x4 v)
{
    const size_t i = row * d + x.c;
    if (x.c + 4 <= d) {
        const u32x2_el h = {(uint32_t)f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16, (uint32_t)f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16};
        const f32x4_el f = {v[0], v[1], v[2], v[3]};
        if (BF && NT) __builtin_nontemporal_store(h, (u32x2_el *)((bf16_t *)p + i));
        else if (BF) *(u32x2_el *)((bf16_t *)p + i) = h;
        else if (NT) __builtin_nontemporal_store(f, (f32x4_el *)((float *)p + i));
        else *(f32x4_el *)((float *)p + i) = f;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (x.w + k >= x.c && x.w + k < d) st1<BF>(p, row * d + x.w + k, v[k]);
}

// ---- forward: a workgroup per 4 rows x 1024 columns, 4 columns a thread (any alignment of an element serves), rows `first` .. T - 1 ----
template <bool BF, bool TINY>
__global__ __launch_bounds__(256) void embedding_forward_kernel(const void *__restrict__ table, int V, int d, const int32_t *__restrict__ ids, int first, int T,
                                                                float scale, void *__restrict__ out)
{
    const int t0 = first + blockIdx.x * 4;
    int id[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) id[r] = t0 + r < T ? ids[t0 + r] : -1;
    for (int c = (blockIdx.y * 256 + threadIdx.x) * 4; c < d; c += gridDim.y * 1024) {
        const emb_cols x(c, d);
        f32x4 v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            v[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (id[r] >= 0 && id[r] < V) v[r] = ld4<BF, TINY>(table, id[r], d, x.w) * scale;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (t0 + r < T) st4<BF>(out, t0 + r, d, x, v[r]);
    }
}

hipError_t launch_embedding_forward(const void *table, int dtype, int V, int d, const int32_t *ids, int T, float scale, void *out, hipStream_t s)
{
    for (int first = 0; first < T; first += EMB_LAUNCH_ROWS) {
        const int end = std::min(T, first + EMB_LAUNCH_ROWS);
        const dim3 grid(ceil_div(end - first, 4), std::min(ceil_div(d, 1024), 64));
#define EMB_FWD(B, TY) hipLaunchKernelGGL((embedding_forward_kernel<B, TY>), grid, dim3(256), 0, s, table, V, d, ids, first, end, scale, out)
        if (dtype == OMEGA_DTYPE_BF16) { if (d < 4) EMB_FWD(true, true); else EMB_FWD(true, false); }
        else { if (d < 4) EMB_FWD(false, true); else EMB_FWD(false, false); }
#undef EMB_FWD
    }
    return hipGetLastError();
}

// ---- backward ----
// Stable counting sort by id.  A workgroup owns IDX_IDS ids; its sixteen waves each walk a sixteenth of the tokens, in order, twice: the
// first time they count the tokens of each of its ids (a counter per wave and id in LDS) and those of smaller ids (where its run of the
// sorted list begins) and note the former, the second time they place them (from the notes; by looking again where those are too many).  Places depend on nothing but the ids: no communication between
// workgroups, one launch.  off[v] = first place of id v (V+1 entries, off[V] = tokens with an id), perm[place] = token,
// sid[place] = its id.  Tokens of a 64-token step with one id are ranked by ballots.
__global__ __launch_bounds__(IDX_WAVES * 64) void embedding_index_kernel(const int32_t *__restrict__ ids, int T, int V, int32_t *__restrict__ off,
                                                                         int32_t *__restrict__ perm, int32_t *__restrict__ sid)
{
    __shared__ int32_t cnt[IDX_IDS][IDX_WAVES + 1];  // (a column of padding: a thread's row starts in a bank of its own)
    __shared__ int32_t below[IDX_WAVES], sums[IDX_WAVES];
    __shared__ uint32_t notes[IDX_WAVES][IDX_NOTES];  // id - lo, and the token counted from the wave's first
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lo = blockIdx.x * IDX_IDS, n_ids = min(IDX_IDS, V - lo);
    for (int i = tid; i < IDX_IDS * (IDX_WAVES + 1); i += IDX_WAVES * 64) (&cnt[0][0])[i] = 0;
    __syncthreads();
    const int seg = ceil_div(ceil_div(T, 64), IDX_WAVES) * 64;
    const int first = min(wave * seg, T), last = min(first + seg, T);
    const unsigned long long before = ((unsigned long long)1 << lane) - 1;
    const bool short_seg = seg <= 1 << 23;  // (a note holds 23 bits of a token)
    int nb = 0, noted = 0;
    for (int t = first; t < last; t += 256) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) id[u] = t + 64 * u + lane < last ? ids[t + 64 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (id[u] >= 0 && id[u] < lo) ++nb;
            const int k = id[u] - lo;
            const bool in = id[u] >= lo && k < n_ids;
            if (in) atomicAdd(&cnt[k][wave], 1);  // (whole numbers: the order does not matter)
            const unsigned long long all = __ballot(in);
            const int at = noted + __popcll(all & before);
            if (in && at < IDX_NOTES) notes[wave][at] = (uint32_t)k << 23 | (uint32_t)((t + 64 * u + lane - first) & 0x7fffff);
            noted += __popcll(all);
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
    // tokens `token` of ids lo + k (lanes where `in`) to their places: lanes with one id find each other by the bits of its number
    auto place = [&](bool in, int k, int token) {
        unsigned long long same = __ballot(in);
        if (same == 0) return;
#pragma unroll
        for (int b = 0; b < IDX_BITS; ++b) {
            const unsigned long long ones = __ballot(in && (k >> b & 1));
            same &= k >> b & 1 ? ones : ~ones;
        }
        // (a counter belongs to its wave: its lanes read it, then the first of those with one id moves it on)
        volatile int32_t *next = &cnt[in ? k : 0][wave];
        const int at = *next;
        __builtin_amdgcn_wave_barrier();
        if (in) {
            const int rank = __popcll(same & before), p = at + rank;
            perm[p] = token;
            sid[p] = lo + k;
            if (rank == 0) *next = at + __popcll(same);
        }
        __builtin_amdgcn_wave_barrier();
    };
    if (noted <= IDX_NOTES && short_seg) {
        for (int i = 0; i < noted; i += 64) {
            const bool in = i + lane < noted;
            const uint32_t n = in ? notes[wave][i + lane] : 0u;
            place(in, (int)(n >> 23), first + (int)(n & 0x7fffff));
        }
        return;
    }
    for (int t = first; t < last; t += 256) {
        int id[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) id[u] = t + 64 * u + lane < last ? ids[t + 64 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 4; ++u) place(id[u] >= lo && id[u] - lo < n_ids, id[u] - lo, t + 64 * u + lane);
    }
}

// Sums of EMB_BLOCK sorted places that belong to one id, unscaled fp32: part[block,:].  LEVEL 1: rows of dout through perm; LEVEL 2: sums of
// EMB_BLOCK blocks of level 1.  Blocks with more than one id are left alone (nobody reads them).
template <bool BF, bool TINY, int LEVEL>
__global__ __launch_bounds__(64) void embedding_block_kernel(const void *__restrict__ src, int d, int V, const int32_t *__restrict__ off,
                                                             const int32_t *__restrict__ perm, const int32_t *__restrict__ sid, float *__restrict__ part)
{
    constexpr int SPAN = LEVEL == 1 ? EMB_BLOCK : EMB_BLOCK * EMB_BLOCK;
    const int b = blockIdx.x, p0 = b * SPAN;
    if (p0 + SPAN > off[V] || sid[p0] != sid[p0 + SPAN - 1]) return;
    const emb_cols x((blockIdx.y * 64 + threadIdx.x) * 4, d);
    const int mine = LEVEL == 1 ? perm[p0 + threadIdx.x] : b * EMB_BLOCK + threadIdx.x;  // (a lane per row)
    f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 16
    for (int i = 0; i < EMB_BLOCK; ++i) a += ld4<LEVEL == 1 ? BF : false, TINY>(src, (size_t)__builtin_amdgcn_readlane(mine, i), d, x.w);
    if (x.c < d) st4<false>(part, b, d, x, a);
}

// Rows `first` .. V - 1 of the table, EMB_ROWS a workgroup: first those without a token (most of them: zeros go out without waiting for anything),
// then the others, each the sum of its run of sorted places.  The places of all rows are walked as one list, 64 to an aligned block and
// eight rows of dout asked for together, so that short runs do not wait one after the other; blocks that a long run fills are
// taken from their sums.  NT: a gradient larger than the caches goes past them (16384 tokens x 2048, vocabulary 128000, 1.05 GB: 266 -> 224 us).
#define EMB_ROWS 16
template <bool BF, bool GBF, bool TINY, bool NT>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const void *__restrict__ dout, int first, int V, int d, float scale, int accumulate,
                                                             const int32_t *__restrict__ off, const int32_t *__restrict__ perm, const int32_t *__restrict__ sid,
                                                             const float *__restrict__ part1, const float *__restrict__ part2, void *__restrict__ dtable)
{
    constexpr int B1 = EMB_BLOCK, B2 = EMB_BLOCK * EMB_BLOCK;
    const int v0 = first + blockIdx.x * EMB_ROWS, lane = threadIdx.x & 63, rows = min(EMB_ROWS, V - v0);
    const emb_cols x((blockIdx.y * 256 + threadIdx.x) * 4, d);
    const int mine = off[v0 + min(lane, rows)];  // lane r: where row r's run begins
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!accumulate && x.c < d) {
#pragma unroll 4
        for (int r = 0; r < rows; ++r)
            if (__builtin_amdgcn_readlane(mine, r) == __builtin_amdgcn_readlane(mine, r + 1)) st4<GBF, NT>(dtable, v0 + r, d, x, zero);
    }
    const int end = __builtin_amdgcn_readlane(mine, rows);
    int row = -1;  // the row that `a` belongs to
    f32x4 a = zero;
    auto write = [&]() {
        if (row < 0 || x.c >= d) return;
        a *= scale;
        if (accumulate) a += ld4<GBF, TINY>(dtable, row, d, x.w);  // (of the four that end a row, another thread's may have its sum by now: only the thread's own are kept)
        st4<GBF, NT>(dtable, row, d, x, a);
    };
    for (int p = __builtin_amdgcn_readlane(mine, 0); p < end;) {
        const int n = min(end - p, B1 - p % B1), tok = perm[p + min(lane, n - 1)], id = sid[p + min(lane, n - 1)];
        const int id0 = __builtin_amdgcn_readlane(id, 0);
        if (part1 != nullptr && n == B1 && id0 == __builtin_amdgcn_readlane(id, B1 - 1)) {
            // a block of one id, and what follows it of the same (a batch of fewer than two blocks has no sums: its rows are added one by one)
            if (id0 != row) {
                write();
                row = id0;
                a = zero;
            }
            const int stop = __builtin_amdgcn_readlane(mine, id0 - v0 + 1);
            while (p + B1 <= stop) {
                if (part2 != nullptr && p % B2 == 0 && p + B2 <= stop) {
                    a += ld4<false, TINY>(part2, p / B2, d, x.w);
                    p += B2;
                    continue;
                }
                int m = (stop - p) / B1;
                if (part2 != nullptr) m = min(m, (B2 - p % B2) / B1);
#pragma unroll 8
                for (int i = 0; i < m; ++i) a += ld4<false, TINY>(part1, p / B1 + i, d, x.w);
                p += m * B1;
            }
            continue;
        }
        for (int i = 0; i < n; i += 8) {
            f32x4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k < n) v[k] = ld4<BF, TINY>(dout, (size_t)__builtin_amdgcn_readlane(tok, i + k), d, x.w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (i + k >= n) break;
                const int next = __builtin_amdgcn_readlane(id, i + k);
                if (next != row) {
                    write();
                    row = next;
                    a = zero;
                }
                a += v[k];
            }
        }
        p += n;
    }
    write();
}

// off [V+1] | perm [T] | sid [T] | part1 [T/64, d] | part2 [T/4096, d]
struct emb_layout {
    size_t perm, sid, part1, part2, bytes;
    int n1, n2;
};
static emb_layout emb_layout_of(int V, int d, int T)
{
    emb_layout l;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    l.n1 = T >= 2 * EMB_BLOCK ? T / EMB_BLOCK : 0;
    // blocks of blocks: where one id could have so many blocks that adding them outweighs a launch (64 blocks are 4 us or so of one workgroup)
    l.n2 = T >= 8 * EMB_BLOCK * EMB_BLOCK ? T / (EMB_BLOCK * EMB_BLOCK) : 0;
    l.perm = up(((size_t)V + 1) * 4);
    l.sid = l.perm + up((size_t)T * 4);
    l.part1 = l.sid + up((size_t)T * 4);
    l.part2 = l.part1 + up((size_t)l.n1 * d * 4);
    l.bytes = l.part2 + up((size_t)l.n2 * d * 4);
    return l;
}

size_t embedding_backward_workspace(int V, int d, int T) { return emb_layout_of(V, d, T).bytes; }

hipError_t launch_embedding_backward(const int32_t *ids, int T, const void *dout, int dtype, int V, int d, float scale, bool accumulate, void *dtable,
                                     int grad_dtype, void *ws, hipStream_t s)
{
    const emb_layout l = emb_layout_of(V, d, T);
    unsigned char *base = (unsigned char *)ws;
    int32_t *off = (int32_t *)base, *perm = (int32_t *)(base + l.perm), *sid = (int32_t *)(base + l.sid);
    float *part1 = l.n1 > 0 ? (float *)(base + l.part1) : nullptr, *part2 = l.n2 > 0 ? (float *)(base + l.part2) : nullptr;
    const bool bf = dtype == OMEGA_DTYPE_BF16, gbf = grad_dtype == OMEGA_DTYPE_BF16;
    hipLaunchKernelGGL(embedding_index_kernel, dim3(ceil_div(V, IDX_IDS)), dim3(IDX_WAVES * 64), 0, s, ids, T, V, off, perm, sid);
    const int gy = ceil_div(d, 256);
#define EMB_BLOCKS(B, TY)                                                                                                                                        \
    do {                                                                                                                                                     \
        if (l.n1 > 0) hipLaunchKernelGGL((embedding_block_kernel<B, TY, 1>), dim3(l.n1, gy), dim3(64), 0, s, dout, d, V, off, perm, sid, part1);             \
        if (l.n2 > 0) hipLaunchKernelGGL((embedding_block_kernel<B, TY, 2>), dim3(l.n2, gy), dim3(64), 0, s, (const void *)part1, d, V, off, perm, sid, part2); \
    } while (0)
#define EMB_ROWS_N(B, G, TY, NT) \
    hipLaunchKernelGGL((embedding_rows_kernel<B, G, TY, NT>), grid, dim3(256), 0, s, dout, first, end, d, scale, accumulate ? 1 : 0, off, perm, sid, part1, part2, dtable)
#define EMB_ROWS_K(B, G, TY) do { if (past) EMB_ROWS_N(B, G, TY, true); else EMB_ROWS_N(B, G, TY, false); } while (0)
#define EMB_RUN(TY)                                                                       \
    do {                                                                                  \
        if (bf) { if (gbf) EMB_ROWS_K(true, true, TY); else EMB_ROWS_K(true, false, TY); } \
        else { if (gbf) EMB_ROWS_K(false, true, TY); else EMB_ROWS_K(false, false, TY); }  \
    } while (0)
    if (bf) { if (d < 4) EMB_BLOCKS(true, true); else EMB_BLOCKS(true, false); }
    else { if (d < 4) EMB_BLOCKS(false, true); else EMB_BLOCKS(false, false); }
    // (67 MB stay in the caches: 33 us, 35 past them; 131 MB: 91 and 70)
    const bool past = !accumulate && (size_t)V * d * (gbf ? 2 : 4) >= OMEGA_LLC_BYTES / 8 * 3;
    for (int first = 0; first < V; first += EMB_LAUNCH_ROWS) {
        const int end = std::min(V, first + EMB_LAUNCH_ROWS);
        const dim3 grid(ceil_div(end - first, EMB_ROWS), ceil_div(d, 1024));
        if (d < 4) EMB_RUN(true);
        else EMB_RUN(false);
    }
#undef EMB_RUN
#undef EMB_ROWS_K
#undef EMB_ROWS_N
#undef EMB_BLOCKS
    return hipGetLastError();
}
