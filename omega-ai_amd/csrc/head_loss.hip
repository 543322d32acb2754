// The head of a language model with its loss: softmax cross entropy of logits = x W^T (x [T,d], W [V,d]) against targets, and its
// gradients, in pieces of the vocabulary.  Large [T,V] logits are never in memory: the forward product's epilogue keeps, for every
// token and 128 columns, the maximum and the sum of exp(logit - maximum); a second launch joins these; the backward pass computes the
// logits of a piece of the vocabulary again and turns them, in registers, into their gradient P, of which one piece at a time exists:
//   loss_t = m_t + log s_t - l[t,y_t],   P[t,v] = exp(l[t,v] - m_t) / s_t - [v = y_t],   dx = g P W,   dW = g P^T x,   g = dloss / n
// (m_t, s_t: a row's maximum and sum.  The pair is kept instead of m + log s, whose rounding would stand in every exp.  g multiplies the
// products' fp32 sums: within P, whose elements are rounded to bf16, the rounding of a row's -g would be the same for all rows.)
//
// All products are one kernel (head_product_kernel): C[m,n] = sum_k A[m,k] B[n,k], bf16 on v_mfma_f32_16x16x32_bf16 with fp32 sums.  A
// tile is 256 x 256, four waves of 128 x 128, one per SIMD; operands stream from memory to LDS in a ring of five or more steps of 32 k;
// persistent, the ring runs on from tile to tile.  Operands are tile images (pack.h) that head_tokens_kernel, head_images_kernel or the
// product before writes, zero where k goes beyond the matrix; W itself is read in place where its rows are whole and aligned.  Where the
// product sums over an operand's rows (W for dx, P and x for dW), the LDS reads transpose.  Tokens without a target are in no image: the
// products' rows are the others, whose number is read on the device.
// fp32 operands are split into three bf16 parts, each the rounding of what those before it leave (24 bits: exact from 2^-110 on; a smaller
// number loses up to 2^-134), an image each, and the product runs over six pairs of parts (hh, hm, mh, mm, hl, lh, the small ones first);
// what is left out, ml, lm and ll, is at most 2^-24 of a term, of either sign (|m| <= 2^-8, |l| <= 2^-17 of the number).
// Forward passes of up to 64 tokens (fp32: 128) stream W through a wave's LDS or registers (head_stream_kernel, head_few_kernel).
// A small vocabulary's logits make too few tiles: they are formed in k slices, whose sums stay in memory until they are joined.
// Bound: the matrix cores (2 T V d for the loss, 8 T V d with gradients, logits formed twice); few tokens: the bytes of W.
#include <algorithm>

#include "common.h"
#include "pack.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

#define HP_BK 32
#define HP_TILE 256
#define HP_SMEM (160 * 1024)                    // all of a compute unit's LDS
// A tile of 32 NU rows: bytes of its A operand's step and of a stage of the ring, stages (lower tiles are through with a step
// sooner and need more of them to cover the same latency: fp32 1611 x 1760, vocabulary 1689, 64-row tiles, five stages 114 us, seven 93),
// direct loads of a wave and step
#define HP_A_BYTES(NU) ((NU) * 2048)
#define HP_STAGE_BYTES(NU) (HP_A_BYTES(NU) + HP_TILE * HP_BK * 2)
#define HP_STAGES(NU) ((NU) == 2 ? 7 : (NU) == 4 ? 6 : 5)
#define HP_LOADS(NU) ((NU) / 2 + 4)
// Tokens up to which the streaming kernels take a forward pass: W once for up to 64; fp32 twice for up to 128, whose other way is three
// images of W
#define HEAD_FEW(dtype) ((dtype) == OMEGA_DTYPE_BF16 ? 64 : 128)

// What a product does with its tile:
//   LSE  rows = tokens, columns = vocabulary: (max, sum) of every token and 128 columns, the target's logit
//   P    the same product: gradient of the logits as tile images (1 or 3 parts)
//   LOG  the same product's fp32 sums, where its tiles are too few: a slab for each k slice
//   ACC  fp32 sums, ADD: added to what is there (dx over the pieces; a k slice has a slab of its own)
//   OUT  the caller's rows (dW)
enum { HEAD_LSE = 0, HEAD_P, HEAD_LOG, HEAD_ACC, HEAD_ADD, HEAD_OUT };

struct head_prod {
    const unsigned char *A, *B;      // tile images, or B: rows of b_ld bytes
    size_t planeA, planeB;           // bytes from one part to the next (fp32)
    size_t b_ld;                     // 0: image
    int kt;                          // k steps (even, 8 or more)
    int ktA, ktB;                    // k steps of a row group of the images (an operand read across its rows: its columns / 32)
    int rowsA;                       // A's rows as far as the product needs them
    int rowsB;                       // B read across its rows in place: the rows there are
    int M, N, mt, nt, slices;        // mt row tiles of 32 NU rows, nt column tiles of 256
    const int32_t *held;             // tokens with a target (M; of dW kt), tile heights (head_rows) of LSE / P / LOG and of ACC / ADD
    // epilogues
    const int32_t *targets;          // of the tokens that have one, as their statistics
    const float *row_stats, *mean, *dloss;
    int T, v0;                       // all tokens, first column of the piece
    float2 *part;                    // LSE
    float *tlogit;
    unsigned char *P;                // P
    size_t planeP;
    float *C;                        // ACC: slabs [slices][rows][ld]
    size_t slab;
    int ld;                          // (a multiple of 256)
    void *out;                       // OUT: row-major, ld = N
    int out_bf, out_vec;
};

// Operands that are read across their rows (the rows are k): W for dx, both for dW.  Their steps are 32 rows x 256 columns, in LDS the same
// blocks of 16 rows x 32 columns as those of an image, two for each 32 columns; ds_read_b64_tr_b16 hands each lane 4 rows of its column.
// The reads are twice as many, each half as long, without bank conflicts.  Against images of the transposes, made by kernels of their own:
// gradients of 4096 tokens, vocabulary 128000, d 4096: 9.62 -> 9.09 ms (the products 740 to 790 us each per 32000 rows of W either way);
// 512 x 4096, 32000: 587 -> 446 us; 131 x 2072, 51750: 417 -> 361.
#define HP_TR_A(EPI) ((EPI) == HEAD_OUT)
#define HP_TR_B(EPI) ((EPI) >= HEAD_ACC)

template <int LDS_OFF>
__device__ __forceinline__ void hp_dma16(const void *sbase, uint32_t voff, uint32_t lds_base)
{
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" ::"s"(sbase), "v"(voff), "s"(lds_base), "n"(LDS_OFF)
                 : "memory", "scc");
}

// past the caches: what is read once
template <int LDS_OFF>
__device__ __forceinline__ void hp_dma16_nt(const void *sbase, uint32_t voff, uint32_t lds_base)
{
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0 nt" ::"s"(sbase), "v"(voff), "s"(lds_base), "n"(LDS_OFF)
                 : "memory", "scc");
}

__device__ __forceinline__ const unsigned char *hp_uniform(const unsigned char *p)
{
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const unsigned char *)(((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ uint32_t hp_pack2(float lo, float hi)
{
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const b2 r = __builtin_convertvector(f2{lo, hi}, b2);
    return *(const uint32_t *)&r;
}

// Three bf16 parts of two fp32 numbers (w[0] the leading ones, a's in the low halves).  ANY: also numbers that would round to infinity, whose
// leading part is cut instead; without, |a| and |b| are 1 at most.  What is no number, or infinite, has parts that are none.
template <bool ANY>
__device__ __forceinline__ void hp_split2(float a, float b, uint32_t (&w)[3])
{
    w[0] = hp_pack2(a, b);
    if (ANY && fmaxf(fabsf(a), fabsf(b)) >= 0x1.ffp127f) w[0] = __float_as_uint(a) >> 16 | (__float_as_uint(b) & 0xffff0000u);
    const float ra = a - __uint_as_float(w[0] << 16), rb = b - __uint_as_float(w[0] & 0xffff0000u);
    w[1] = hp_pack2(ra, rb);
    w[2] = hp_pack2(ra - __uint_as_float(w[1] << 16), rb - __uint_as_float(w[1] & 0xffff0000u));
}

// One tile of a product, or a k slice of one
struct hp_item {
    const unsigned char *A, *B;   // first step of the tile's rows and columns
    int row0, n0, slice;          // first row and column
    int kt;                       // steps (of a part)
    int phase, rows;              // of an operand read across its rows: first step's place in its row group, rows from there on
};

template <int NU, int EPI>
__device__ __forceinline__ hp_item hp_make_item(const head_prod &p, int idx)
{
    hp_item it;
    const int per = p.mt * p.nt;
    // column tiles outside, up to 8 row tiles inside: the 32 neighbours that an XCD works on share operand tiles in its L2
    const int sl = idx / per, rem = idx - sl * per, g = rem / (8 * p.nt), gm = min(8, p.mt - 8 * g), r2 = rem - g * 8 * p.nt, n = r2 / gm;
    it.row0 = __builtin_amdgcn_readfirstlane((8 * g + (r2 - n * gm)) * 32 * NU);
    it.n0 = __builtin_amdgcn_readfirstlane(n * HP_TILE);
    it.slice = __builtin_amdgcn_readfirstlane(sl);
    const int first = ((it.slice * p.kt) / p.slices) & ~1;
    it.kt = __builtin_amdgcn_readfirstlane((it.slice + 1 == p.slices ? p.kt : (((it.slice + 1) * p.kt) / p.slices) & ~1) - first);
    it.phase = __builtin_amdgcn_readfirstlane(first & 3);
    it.rows = __builtin_amdgcn_readfirstlane(p.b_ld == 0 ? 0x7fffffff : p.rowsB - 32 * first);
    const size_t rgA = (size_t)p.ktA * 8192, rgB = (size_t)p.ktB * 8192;  // bytes of a row group of an image
    const size_t across = (size_t)(first >> 2), in = (size_t)(first & 3) * 2048;
    if (HP_TR_A(EPI)) it.A = hp_uniform(p.A + across * rgA + in + (size_t)(it.row0 >> 5) * 8192);
    else it.A = hp_uniform(p.A + (size_t)(it.row0 >> 7) * rgA + (size_t)first * 8192);
    if (HP_TR_B(EPI))
        it.B = hp_uniform(p.b_ld == 0 ? p.B + across * rgB + in + (size_t)(it.n0 >> 5) * 8192 : p.B + (size_t)first * 32 * p.b_ld + (size_t)it.n0 * 2);
    else
        it.B = hp_uniform(p.b_ld == 0 ? p.B + (size_t)(it.n0 >> 7) * rgB + (size_t)first * 8192 : p.B + (size_t)it.n0 * p.b_ld + (size_t)first * 64);
    return it;
}
// The lane number, counted anew wherever it is needed, as a value that the compiler cannot carry over: nor can it what follows from it.
// (Kept from item to item these are spilled, and the wait for a reload in the middle of a k loop drains the ring: 49 % of the matrix rate
// instead of 80.)
__device__ __forceinline__ int hp_lane()
{
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
    return lane;
}
// what the lane adds for the wave's loads, blocks wave + 4 n of the step: of 16 rows each; of an operand read across its rows, 16 rows and
// 32 columns, the upper and the lower 16 rows in turn
template <int NU, int EPI>
__device__ __forceinline__ void hp_lane_offsets(const head_prod &p, const hp_item &it, int wave, int lane, uint32_t (&va)[4], uint32_t (&vb)[4])
{
    const uint32_t rgA = (uint32_t)p.ktA * 8192u, rgB = (uint32_t)p.ktB * 8192u;
    const int blk0 = (it.row0 & 127) >> 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int q = wave + 4 * k;
        if (HP_TR_A(EPI)) {
            const bool valid = q < 2 * NU && it.row0 + 32 * (q >> 1) < 32 * p.ktA;
            va[k] = valid ? (uint32_t)(q >> 1) * 8192u + (uint32_t)(q & 1) * 1024u + (uint32_t)lane * 16u : 0u;
        } else {
            const bool valid = q < 2 * NU && it.row0 + 16 * q < p.rowsA;  // (a block without rows: every lane reads the first 16 bytes of the item's first block)
            const int b = blk0 + (valid ? q : 0);
            va[k] = (uint32_t)(b >> 3) * rgA + (uint32_t)(b & 7) * 1024u + (valid ? (uint32_t)lane * 16u : 0u);
        }
        if (HP_TR_B(EPI) && p.b_ld == 0) {
            vb[k] = it.n0 + 32 * (q >> 1) < 32 * p.ktB ? (uint32_t)(q >> 1) * 8192u + (uint32_t)(q & 1) * 1024u + (uint32_t)lane * 16u : 0u;
        } else if (HP_TR_B(EPI)) {
            const int r = 16 * (q & 1) + (lane >> 2), c = 32 * (q >> 1) + 8 * ((lane & 3) ^ pk_swz(r));
            vb[k] = (uint32_t)min(r, it.rows - 1) * (uint32_t)p.b_ld + (uint32_t)min(c, p.N - 8 - it.n0) * 2u;
        } else {
            // (both forms and a choice: a branch here costs registers that the product has not got)
            const int r = 16 * q + (lane >> 2);
            const uint32_t image = (uint32_t)(q >> 3) * rgB + (uint32_t)(q & 7) * 1024u + (uint32_t)lane * 16u;
            uint32_t rows = (uint32_t)min(r, p.N - 1 - it.n0) * (uint32_t)p.b_ld + (uint32_t)(((lane & 3) ^ pk_swz(r)) << 4);
            asm volatile("" : "+v"(rows));
            vb[k] = p.b_ld == 0 ? image : rows;
        }
    }
}

// where the loads have got to
struct hp_at {
    const unsigned char *A, *B;
    int phase, rows;
};
// ... and a step on.  Rows of W in place: where the last ones are fewer than 32, the lanes behind them read the last one, and a step that
// has none reads the step before once more (P is zero there).
template <int EPI>
__device__ __forceinline__ void hp_advance(const head_prod &p, hp_at &at, uint32_t (&vb)[4], int wave)
{
    if (!HP_TR_B(EPI)) {
        at.A += 8192;
        at.B += p.b_ld == 0 ? 8192 : 64;
        return;
    }
    at.phase = (at.phase + 1) & 3;
    const bool next = at.phase == 0;  // the next row group
    if (HP_TR_A(EPI)) at.A += next ? (size_t)p.ktA * 8192 - 6144 : 2048;
    else at.A += 8192;
    if (HP_TR_A(EPI) || p.b_ld == 0) {
        at.B += next ? (size_t)p.ktB * 8192 - 6144 : 2048;
    } else {
        at.rows -= 32;
        at.B += at.rows > 0 ? (size_t)32 * p.b_ld : 0;
        if (at.rows > 0 && at.rows < 32) {
            const int behind = max(16 * (wave & 1) + (hp_lane() >> 2) - (at.rows - 1), 0);
#pragma unroll
            for (int k = 0; k < 4; ++k) vb[k] -= (uint32_t)behind * (uint32_t)p.b_ld;
        }
    }
}

// Where a lane's fragments lie in a stage.  a0, b0 / b1 (even / odd fragments of 16 columns): the 16-byte chunk lane / 16 of its row.  Read
// across rows: rows 8 kc .. + 3 (4 more: the other address + 256) of a fragment's columns, kc = (0, 2, 1, 3)[lane / 16], which keeps the
// lanes of a half wave in different banks; the other operand takes its chunks in the same order.
struct hp_frag {
    uint32_t a0, a1, b0, b1;
};
template <int NU, int EPI>
__device__ __forceinline__ hp_frag hp_frag_of(int wm, int wn, int lane)
{
    const int l16 = lane & 15, lq = lane >> 4;
    const int kc = HP_TR_B(EPI) ? ((lq & 1) << 1) | (lq >> 1) : lq;
    const uint32_t across = (uint32_t)((lq & 1) * 1024 + (8 * (lq >> 1) + (l16 >> 2)) * 64 + ((((l16 >> 1) ^ (l16 >> 3) ^ (lq >> 1)) & 1) << 4) + 8 * (l16 & 1));
    hp_frag f;
    if (HP_TR_A(EPI)) {
        f.a0 = across + 32u * (uint32_t)(wm ^ (lq & 1));
        f.a1 = f.a0 ^ 32u;
    } else {
        f.a0 = (uint32_t)(wm * 16 + l16) * 64 + ((uint32_t)(kc ^ pk_swz(l16 | (wm << 4))) << 4);
        f.a1 = 0;
    }
    if (HP_TR_B(EPI)) {
        f.b0 = HP_A_BYTES(NU) + wn * 8192u + across + 32u * (uint32_t)(lq & 1);
        f.b1 = f.b0 ^ 32u;
    } else {
        f.b0 = HP_A_BYTES(NU) + (uint32_t)(wn * 128 + l16) * 64 + ((uint32_t)(kc ^ pk_swz(l16)) << 4);
        f.b1 = HP_A_BYTES(NU) + (uint32_t)(wn * 128 + 16 + l16) * 64 + ((uint32_t)(kc ^ pk_swz(l16 | 16)) << 4);
    }
    return f;
}
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(8))) short s16x8_t;
__device__ __forceinline__ bf16x8_t hp_across(const unsigned char *lo, const unsigned char *hi)
{
    typedef __attribute__((address_space(3))) s16x4_t lds_t;
    const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)lo), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)hi);
    const s16x8_t v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return *(const bf16x8_t *)&v;
}

// pairs of parts in the order they are added: (A, B) = mm, lh, hl, mh, hm, hh
#define HP_SEG_A 0x001021  // nibble s = part of segment s, from the right: 1, 2, 0, 1, 0, 0
#define HP_SEG_B 0x010201  // 1, 0, 2, 0, 1, 0

struct hp_state {
    int cur;                             // ring position
    bf16x8_t fa0[8], fb0[8], fa1[8], fb1[8];
    hp_at at;
    uint32_t va[4], vb[4];
};

// Loads and fragments of the ring, the MFMAs of a step.  The first 8 groups of 4 MFMAs carry the fragment reads of the next step (two
// MFMAs apart: next to each other those across rows cost 4 % of a product), every other group one of the direct loads of the step that
// the ring is ahead.
#define HP_READ(FA, FB, r)                                                                                                     \
    do {                                                                                                                       \
        if ((r) < 8) {                                                                                                         \
            const unsigned char *b0 = ((r) & 1 ? rb1 : rb0) + (((r) & 7) >> 1) * 2048u;                                        \
            if (HP_TR_B(EPI)) FB[(r) & 7] = hp_across(b0, ((r) & 1 ? rb0 : rb1) + (((r) & 7) >> 1) * 2048u + 256u);            \
            else FB[(r) & 7] = *(const bf16x8_t *)b0;                                                                          \
        } else if ((r) - 8 < NU) {                                                                                             \
            if (HP_TR_A(EPI)) FA[((r) - 8) & 7] = hp_across(ra + (((r) - 8) & 7) * 2048u, ra1 + (((r) - 8) & 7) * 2048u + 256u); \
            else FA[((r) - 8) & 7] = *(const bf16x8_t *)(ra + (((r) - 8) & 7) * 2048u);                                        \
        }                                                                                                                      \
    } while (0)
#define HP_LOAD(l, sb)                                                                                                         \
    do {                                                                                                                       \
        if ((l) < NU / 2) hp_dma16<((l) & 3) * 4096>(at.A, st.va[(l) & 3], sb);                                                \
        else if ((l) < HP_LOADS(NU)) hp_dma16<HP_A_BYTES(NU) + (((l) - NU / 2) & 3) * 4096>(at.B, st.vb[((l) - NU / 2) & 3], sb); \
    } while (0)
// fragments of the stage behind `cur`
#define HP_STAGE_ADDR()                                                                                 \
    do {                                                                                                \
        const unsigned char *sn = smem + (cur + 1 == ST ? 0 : cur + 1) * HP_STAGE_BYTES(NU);            \
        ra = sn + fr.a0;                                                                                \
        ra1 = sn + fr.a1;                                                                               \
        rb0 = sn + fr.b0;                                                                               \
        rb1 = sn + fr.b1;                                                                               \
    } while (0)
#define HP_MFMA(PA, PB, iu, c)                                                                                                    \
    do {                                                                                                                             \
        if ((iu) < NU)                                                                                                               \
            acc[(iu) % NU][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(PB[c], PA[iu], acc[(iu) % NU][c], 0, 0, 0);    \
    } while (0)
#define HP_GROUP(PA, PB, QA, QB, g)                     \
    do {                                                   \
        HP_MFMA(PA, PB, (g) >> 1, 4 * ((g) & 1));       \
        if ((g) < 8) HP_READ(QA, QB, 2 * (g));             \
        __builtin_amdgcn_sched_barrier(0);                 \
        HP_MFMA(PA, PB, (g) >> 1, 4 * ((g) & 1) + 1);   \
        if ((g) & 1) HP_LOAD((g) >> 1, sb);                \
        __builtin_amdgcn_sched_barrier(0);                 \
        HP_MFMA(PA, PB, (g) >> 1, 4 * ((g) & 1) + 2);   \
        if ((g) < 8) HP_READ(QA, QB, 2 * (g) + 1);         \
        __builtin_amdgcn_sched_barrier(0);                 \
        HP_MFMA(PA, PB, (g) >> 1, 4 * ((g) & 1) + 3);   \
        __builtin_amdgcn_sched_barrier(0);                 \
    } while (0)
#define HP_STEP(PA, PB, QA, QB)                                                                          \
    do {                                                                                                    \
        HP_GROUP(PA, PB, QA, QB, 0); HP_GROUP(PA, PB, QA, QB, 1); HP_GROUP(PA, PB, QA, QB, 2);     \
        HP_GROUP(PA, PB, QA, QB, 3); HP_GROUP(PA, PB, QA, QB, 4); HP_GROUP(PA, PB, QA, QB, 5);     \
        HP_GROUP(PA, PB, QA, QB, 6); HP_GROUP(PA, PB, QA, QB, 7); HP_GROUP(PA, PB, QA, QB, 8);     \
        HP_GROUP(PA, PB, QA, QB, 9); HP_GROUP(PA, PB, QA, QB, 10); HP_GROUP(PA, PB, QA, QB, 11);   \
        HP_GROUP(PA, PB, QA, QB, 12); HP_GROUP(PA, PB, QA, QB, 13); HP_GROUP(PA, PB, QA, QB, 14);  \
        HP_MFMA(PA, PB, 7, 4);                                                                           \
        __builtin_amdgcn_sched_barrier(0);                                                                  \
        HP_MFMA(PA, PB, 7, 5);                                                                           \
        HP_LOAD(7, sb);                                                                                     \
        __builtin_amdgcn_sched_barrier(0);                                                                  \
        HP_MFMA(PA, PB, 7, 6);                                                                           \
        cur = cur + 1 == ST ? 0 : cur + 1;                                                                \
        sb = lds_wave + cur * HP_STAGE_BYTES(NU);                                                           \
        hp_advance<EPI>(p, at, st.vb, wave);                                                                \
        __builtin_amdgcn_sched_barrier(0);                                                                  \
        HP_MFMA(PA, PB, 7, 7);                                                                           \
        HP_STAGE_ADDR();                                                                                    \
        __builtin_amdgcn_sched_barrier(0);                                                                  \
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((ST - 2) * HP_LOADS(NU)) : "memory");           \
        __syncthreads();                                                                                    \
    } while (0)

// exp of a difference to the row's maximum.  bf16: v_exp_f32 of v log2(e), whose rounding weighs a few 2^-24 for the differences that
// count; fp32: what the rounding of the product leaves is put back, exp2(t + e) = exp2(t) (1 + e ln 2).
// (differences below -200 are 0 either way; a comparison, not a maximum, so that no number stays none)
template <int NSEG>
__device__ __forceinline__ float hp_exp(float v)
{
    if (NSEG == 1) return __expf(v);
    v = v < -200.0f ? -200.0f : v;
    const float t = v * 1.44269504088896341f;
    const float e = fmaf(v, 1.92596299e-8f, fmaf(v, 1.44269504088896341f, -t));
    const float r = __builtin_amdgcn_exp2f(t);
    return fmaf(r, e * 0.693147181f, r);
}

// Stores into the caller's rows that fall away where `ok` is false, without a branch: a buffer store beyond its range does nothing.
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
#define HP_OUTSIDE 0xffffffffu

// Quarters of the wave (16 lanes) 1 and 3 of a change places with quarters 0 and 2 of b: [0] = a0 b0 a2 b2, [1] = a1 b1 a3 b3
__device__ __forceinline__ u32x2_t hp_swap16(uint32_t a, uint32_t b)
{
    return __builtin_amdgcn_permlane16_swap(a, b, false, false);
}

// what the gradients are multiplied by: dloss / tokens with a target
__device__ __forceinline__ float head_scale(const float *mean, const float *dloss) { return (dloss ? dloss[0] : 1.0f) / fmaxf(mean[1], 1.0f); }

// Writers of the two products with the vocabulary.  WHOLE: every column of the wave is there.
template <int NU, int NSEG, bool WHOLE>
__device__ __forceinline__ void hp_write_lse(const head_prod &p, const hp_item &it, const f32x4_t (&acc)[NU][8], int wm, int wn, int l16, int lq)
{
    const int col0 = it.n0 + wn * 128 + 4 * lq;
    // maximum and sum of a lane's 32 columns first, unit by unit; the four lanes of a row are joined for all units together, so that
    // the latencies of the targets' loads and of the lane exchanges are paid once
    float m[NU], s[NU];
    int y[NU];
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) y[iu] = p.targets[min(it.row0 + 16 * (2 * iu + wm) + l16, p.M - 1)];
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) {
        __builtin_amdgcn_sched_barrier(0);  // (a unit at a time: the registers are full)
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = WHOLE || col0 + 16 * (k >> 2) + (k & 3) < p.N ? acc[iu][k >> 2][k & 3] : -INFINITY;  // (exp(-inf) is zero)
        m[iu] = v[0];
#pragma unroll
        for (int k = 1; k < 32; ++k) m[iu] = fmaxf(m[iu], v[k]);
        const float m0 = m[iu] == -INFINITY ? 0.0f : m[iu];  // (no column, or every logit -inf: the sum is 0)
        s[iu] = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s[iu] += hp_exp<NSEG>(v[k] - m0);
        // the target's logit, where it is among the lane's columns
        const int t = it.row0 + 16 * (2 * iu + wm) + l16, at = y[iu] - p.v0 - col0;
        const bool mine = t < p.M && at >= 0 && at < 128 && (at & 12) == 0 && col0 + at < p.N;
        if (__ballot(mine)) {
            float l = 0.0f;
#pragma unroll
            for (int k = 0; k < 32; ++k) l = at == 16 * (k >> 2) + (k & 3) ? v[k] : l;
            if (mine) p.tlogit[t] = l;
        }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) {
        float all = fmaxf(m[iu], __shfl_xor(m[iu], 16, 64));
        all = fmaxf(all, __shfl_xor(all, 32, 64));
        s[iu] *= hp_exp<NSEG>(m[iu] - (all == -INFINITY ? 0.0f : all));
        m[iu] = all;
    }
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) s[iu] += __shfl_xor(s[iu], 16, 64);
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) s[iu] += __shfl_xor(s[iu], 32, 64);
    float2 *part = p.part + (size_t)((p.v0 + it.n0) / 128 + wn) * p.T;
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) {
        const int t = it.row0 + 16 * (2 * iu + wm) + l16;
        if (lq == 0 && t < p.M) part[t] = make_float2(m[iu], s[iu]);
    }
}
// P of a bf16 head is rounded to bf16, an element by 2^-8 of itself at most, as x and W were when they became bf16, and each for itself: dx
// and dw, which have 0.0017 (2-norm, against 64 bits) from their own rounding, have 0.0019 with it (4096 tokens x 4096, vocabulary 128000;
// rows of dw without a target 0.0022).  A second part of P would take away the 0.0009 between these (in squares), for two more
// products of 3 ms each on top of 12, and another piece of P.  fp32 heads carry all of P in three parts.
template <int NU, int NSEG, bool WHOLE>
__device__ __forceinline__ void hp_write_p(const head_prod &p, const hp_item &it, const f32x4_t (&acc)[NU][8], int wm, int wn, int l16, int lq)
{
    const int col0 = it.n0 + wn * 128 + 4 * lq;
    // (rows behind the last token, whose image rows are zeros, are written as zeros: they are k places of dW)
    const int KTp = p.nt * (HP_TILE / HP_BK);
    constexpr int NP = NSEG > 1 ? 3 : 1;
    // (to the image's end: rows of the tile behind it fall away)
    const int rgs = min(((p.rowsA + 127) >> 7) - (it.row0 >> 7), 3), kb = (it.n0 >> 5) + 4 * wn;
    __amdgpu_buffer_rsrc_t rs[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q)
        rs[q] = __builtin_amdgcn_make_buffer_rsrc((void *)hp_uniform(p.P + q * p.planeP + (size_t)(it.row0 >> 7) * KTp * 8192 + (size_t)kb * 8192), 0,
                                                  (rgs * KTp - kb) * 8192, 0x00020000);
    int y[NU];
    float m[NU], f[NU];
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) {
        const int t = min(it.row0 + 16 * (2 * iu + wm) + l16, p.M - 1);
        y[iu] = p.targets[t];
        m[iu] = p.row_stats[t];
        f[iu] = p.row_stats[p.T + t];
    }
#pragma unroll
    for (int iu = 0; iu < NU; ++iu) {
        __builtin_amdgcn_sched_barrier(0);  // (a unit at a time: the registers are full)
        const int row = it.row0 + 16 * (2 * iu + wm) + l16;
        const bool held = row < p.M;
        const float fu = held ? 1.0f / f[iu] : 0.0f, mu = held ? m[iu] : 0.0f;
        const int k = y[iu] - p.v0 - col0;
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            v[e] = hp_exp<NSEG>(acc[iu][e >> 2][e & 3] - mu) * fu;
            if (!WHOLE) v[e] = col0 + 16 * (e >> 2) + (e & 3) < p.N ? v[e] : 0.0f;
        }
        if (__ballot(held && k >= 0 && k < 128 && (k & 12) == 0)) {
            const float g1 = held ? 1.0f : 0.0f;
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] -= k == 16 * (e >> 2) + (e & 3) ? g1 : 0.0f;
        }
        // two fragments of 16 columns are a k step of the image: lanes of neighbouring quarters exchange halves, so that a lane has the 8
        // columns of a 16-byte chunk and the wave stores a whole block of 16 rows x 32 columns at once
        const uint32_t at = (uint32_t)((row >> 7) - (it.row0 >> 7)) * (uint32_t)KTp * 8192u +
                            (uint32_t)(((row & 127) >> 4) * 1024 + (row & 15) * 64 + (((2 * (lq & 1) + (lq >> 1)) ^ pk_swz(row)) << 4));
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
            uint32_t h[NP][4];  // parts of fragment c (two words) and of fragment c + 1
            if (NSEG == 1) {
#pragma unroll
                for (int w = 0; w < 4; ++w) h[0][w] = hp_pack2(v[4 * c + 2 * w], v[4 * c + 2 * w + 1]);
            } else {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t two[3];
                    hp_split2<false>(v[4 * c + 2 * w], v[4 * c + 2 * w + 1], two);
#pragma unroll
                    for (int q = 0; q < NP; ++q) h[q][w] = two[q];
                }
            }
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const u32x2_t a = hp_swap16(h[q][0], h[q][2]), b = hp_swap16(h[q][1], h[q][3]);
                __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{a[0], b[0], a[1], b[1]}, rs[q], at + (c >> 1) * 8192, 0, 0);
            }
            if (NSEG > 1) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// A tile of 32 NU rows by 256 columns.  acc[iu][c][r]: row 16 (2 iu + wm) + lane % 16, column 128 wn + 16 c + 4 (lane / 16) + r.
template <int NU, int EPI, int NSEG>
__device__ __forceinline__ void hp_run_item(unsigned char *smem, hp_state &st, const head_prod &p, const hp_item &it, hp_item &nxt, int next_idx, int wave)
{
    constexpr int ST = HP_STAGES(NU);
    const int wm = wave >> 1, wn = wave & 1;
    int lane = hp_lane(), l16 = lane & 15, lq = lane >> 4;
    const int kt = __builtin_amdgcn_readfirstlane(it.kt);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
    const uint32_t lds_wave = lds0 + wave * 1024;
    const hp_frag fr = hp_frag_of<NU, EPI>(wm, wn, lane);
    int cur = __builtin_amdgcn_readfirstlane(st.cur);
    hp_at at = {hp_uniform(st.at.A), hp_uniform(st.at.B), __builtin_amdgcn_readfirstlane(st.at.phase), __builtin_amdgcn_readfirstlane(st.at.rows)};
    nxt = hp_make_item<NU, EPI>(p, next_idx);
    uint32_t sb = lds_wave + cur * HP_STAGE_BYTES(NU);
    const unsigned char *ra, *ra1, *rb0, *rb1;
    HP_STAGE_ADDR();
    f32x4_t acc[NU][8];
    const f32x4_t zero4 = {0.0f, 0.0f, 0.0f, 0.0f};
    // The steps of a pair of parts two at a time (their number is even, at least 8).  The loads of the last ST are the next pair's or the
    // next item's first (behind the last item: this one's once more, which nobody reads).
    // (zeros in the registers: a first step that starts from zero operands instead costs as many moves of registers)
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[i][c] = zero4;
    // (the sums stay in accumulation registers: with other uses in sight, the compiler keeps some elsewhere and moves them in the loop)
#define HP_PIN()                          \
    _Pragma("unroll") for (int i = 0; i < NU; ++i) \
        _Pragma("unroll") for (int c = 0; c < 8; ++c) asm volatile("" : "+a"(acc[i][c]))
    HP_PIN();
#pragma unroll 1
    for (int seg = 0; seg < NSEG; ++seg) {
        int k = kt - ST - (ST & 1);
        if (NU > 2 || k > 0) {  // (eight steps, seven stages: nothing yet)
            do {
                HP_STEP(st.fa0, st.fb0, st.fa1, st.fb1);
                HP_STEP(st.fa1, st.fb1, st.fa0, st.fb0);
            } while ((k -= 2) > 0);
        }
        if (ST & 1) HP_STEP(st.fa0, st.fb0, st.fa1, st.fb1);
        {
            const int ns = seg + 1 < NSEG ? seg + 1 : 0;
            const hp_item &li = ns == 0 ? nxt : it;  // the item of the loads from here on
            const size_t a0 = NSEG > 1 ? (size_t)((HP_SEG_A >> (4 * ns)) & 3) * p.planeA : 0, b0 = NSEG > 1 ? (size_t)((HP_SEG_B >> (4 * ns)) & 3) * p.planeB : 0;
            at = {hp_uniform(li.A + a0), hp_uniform(li.B + b0), li.phase, li.rows};
            hp_lane_offsets<NU, EPI>(p, li, wave, hp_lane(), st.va, st.vb);
        }
        if (ST & 1) HP_STEP(st.fa1, st.fb1, st.fa0, st.fb0);
        for (k = 0; k < ST / 2; ++k) {
            HP_STEP(st.fa0, st.fb0, st.fa1, st.fb1);
            HP_STEP(st.fa1, st.fb1, st.fa0, st.fb0);
        }
    }
    HP_PIN();
    st.cur = cur;
    st.at = at;

    lane = hp_lane();
    l16 = lane & 15;
    lq = lane >> 4;
    const int col0 = it.n0 + wn * 128 + 4 * lq;  // column of acc[.][0][0]
    const bool whole = it.n0 + wn * 128 + 128 <= p.N;  // (the wave's columns are all there)
    if (EPI == HEAD_LSE) {
        if (whole) hp_write_lse<NU, NSEG, true>(p, it, acc, wm, wn, l16, lq);
        else hp_write_lse<NU, NSEG, false>(p, it, acc, wm, wn, l16, lq);
    } else if (EPI == HEAD_P) {
        if (whole) hp_write_p<NU, NSEG, true>(p, it, acc, wm, wn, l16, lq);
        else hp_write_p<NU, NSEG, false>(p, it, acc, wm, wn, l16, lq);
    } else if (EPI == HEAD_LOG || EPI == HEAD_ACC || EPI == HEAD_ADD) {
        // (a slab has room for whole tiles)
        float *tile = p.C + (size_t)it.slice * p.slab + (size_t)it.row0 * p.ld + it.n0 + wn * 128;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)hp_uniform((const unsigned char *)tile), 0, 256 * p.ld * 4, 0x00020000);
        uint32_t off = (uint32_t)(16 * wm + l16) * (uint32_t)p.ld * 4u + (uint32_t)lq * 16u;
#pragma unroll
        for (int iu = 0; iu < NU; ++iu) {
            __builtin_amdgcn_sched_barrier(0);
            if (EPI == HEAD_ADD) {
                f32x4_t old[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const u32x4_t u = __builtin_amdgcn_raw_buffer_load_b128(rs, off + 64 * c, 0, 0);
                    old[c] = *(const f32x4_t *)&u;
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) acc[iu][c] += old[c];
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4_t *)&acc[iu][c], rs, off + 64 * c, 0, 0);
            off += 32u * (uint32_t)p.ld * 4u;
        }
    } else {
        const int es = p.out_bf ? 2 : 4;
        const float g = head_scale(p.mean, p.dloss);
        // from the tile's first row on: at most 256 rows of N values
        const uint64_t tile = (uint64_t)p.out + (uint64_t)it.row0 * p.N * es;
        const int rows = min(32 * NU, p.M - it.row0);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)hp_uniform((const unsigned char *)tile), 0, rows * p.N * es, 0x00020000);
        const int step = 32 * p.N * es, row1 = 16 * wm + l16;
        int off = (row1 * p.N + col0) * es;
        const int cols = p.N - col0;  // columns from there on
#pragma unroll
        for (int iu = 0; iu < NU; ++iu) {
            __builtin_amdgcn_sched_barrier(0);
            if (p.out_vec && p.out_bf) {  // (rows of whole 16 bytes; halves exchanged as in the image of P)
#pragma unroll
                for (int c = 0; c < 8; c += 2) {
                    const f32x4_t v = acc[iu][c] * g, w = acc[iu][c + 1] * g;
                    const u32x2_t a = hp_swap16(hp_pack2(v[0], v[1]), hp_pack2(w[0], w[1])), b = hp_swap16(hp_pack2(v[2], v[3]), hp_pack2(w[2], w[3]));
                    const int cc = 16 * (c + (lq & 1)) + 8 * (lq >> 1) - 4 * lq;  // from col0
                    __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{a[0], b[0], a[1], b[1]}, rs, cc < cols ? (uint32_t)(off + cc * 2) : HP_OUTSIDE, 0, 0);
                }
            } else if (p.out_vec) {  // (fp32, a multiple of 4 columns)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const f32x4_t v = acc[iu][c] * g;
                    __builtin_amdgcn_raw_buffer_store_b128(*(const u32x4_t *)&v, rs, 16 * c < cols ? (uint32_t)(off + 64 * c) : HP_OUTSIDE, 0, 0);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = acc[iu][c][r] * g;
                        const uint32_t at = 16 * c + r < cols ? (uint32_t)(off + (16 * c + r) * es) : HP_OUTSIDE;
                        if (p.out_bf) __builtin_amdgcn_raw_buffer_store_b16((unsigned short)hp_pack2(v, 0.0f), rs, at, 0, 0);
                        else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), rs, at, 0, 0);
                    }
            }
            off += step;
        }
    }
}

// Persistent: workgroup w takes items w, w + n, ... in rounds of n = gridDim.x; within a round XCD x (w % 8) takes neighbouring items.
template <int NU, int EPI, int NSEG>
__device__ __forceinline__ void hp_run(unsigned char *smem, const head_prod &p, int wave)
{
    // (fewer items than workgroups: as many of each XCD.  Were the first XCDs filled first, or neighbours dealt out over all of them, the
    // operands would come through fewer L2s, or through each of them: fp32 400 x 1024, vocabulary 9000: 157 us instead of 88)
    const int total = p.mt * p.nt * p.slices;
    const int n_wg = gridDim.x % 8 == 0 ? min((int)gridDim.x, (total + 7) & ~7) : (int)gridDim.x;
    int idx = blockIdx.x;
    if (gridDim.x % 8 == 0) {
        if ((int)(blockIdx.x >> 3) >= n_wg >> 3) return;
        idx = (blockIdx.x & 7) * (n_wg >> 3) + (blockIdx.x >> 3);
    }
    if (idx >= total) return;
    hp_item it = hp_make_item<NU, EPI>(p, idx);
    hp_state st;
    hp_at at = {hp_uniform(it.A + (NSEG > 1 ? (size_t)(HP_SEG_A & 3) * p.planeA : 0)), hp_uniform(it.B + (NSEG > 1 ? (size_t)(HP_SEG_B & 3) * p.planeB : 0)),
                it.phase, it.rows};
    hp_lane_offsets<NU, EPI>(p, it, wave, hp_lane(), st.va, st.vb);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
    constexpr int ST = HP_STAGES(NU);
    for (int i = 0; i < ST; ++i) {  // the first item's first steps (of 8 or more of its first part)
        const uint32_t sb = lds0 + wave * 1024 + i * HP_STAGE_BYTES(NU);
        HP_LOAD(0, sb); HP_LOAD(1, sb); HP_LOAD(2, sb); HP_LOAD(3, sb);
        HP_LOAD(4, sb); HP_LOAD(5, sb); HP_LOAD(6, sb); HP_LOAD(7, sb);
        hp_advance<EPI>(p, at, st.vb, wave);
    }
    st.at = at;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * HP_LOADS(NU)) : "memory");
    __syncthreads();
    {
        const hp_frag fr = hp_frag_of<NU, EPI>(wave >> 1, wave & 1, hp_lane());
        const int cur = ST - 1;  // (stage 0 is the one behind it)
        const unsigned char *ra, *ra1, *rb0, *rb1;
        HP_STAGE_ADDR();
        HP_READ(st.fa0, st.fb0, 0); HP_READ(st.fa0, st.fb0, 1); HP_READ(st.fa0, st.fb0, 2); HP_READ(st.fa0, st.fb0, 3);
        HP_READ(st.fa0, st.fb0, 4); HP_READ(st.fa0, st.fb0, 5); HP_READ(st.fa0, st.fb0, 6); HP_READ(st.fa0, st.fb0, 7);
        HP_READ(st.fa0, st.fb0, 8); HP_READ(st.fa0, st.fb0, 9); HP_READ(st.fa0, st.fb0, 10); HP_READ(st.fa0, st.fb0, 11);
        HP_READ(st.fa0, st.fb0, 12); HP_READ(st.fa0, st.fb0, 13); HP_READ(st.fa0, st.fb0, 14); HP_READ(st.fa0, st.fb0, 15);
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((ST - 2) * HP_LOADS(NU)) : "memory");  // step 1 has landed; every wave has taken step 0 out of its stage
    __syncthreads();
    st.cur = 0;
    for (;;) {
        const bool more = idx + n_wg < total;
        if (more) idx += n_wg;
        hp_item nxt;  // (behind the last item: this one's loads once more, which nobody reads)
        hp_run_item<NU, EPI, NSEG>(smem, st, p, it, nxt, idx, wave);
        if (!more) break;
        it = nxt;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the loads behind the last item land in LDS that nobody reads)
}

// Height of a row tile, 64 times the result: the one that takes the least time by rounds of one tile per compute unit.  A step of a tile of
// k x 64 rows takes k + 7/4 parts, of fp32's products k + 3/4 (its columns' loads count most where they are W's rows in place): measured
// with all compute units at work, 512 x 4096, vocabulary 32000, bf16 0.39, 0.52, 0.62 and 0.82 us for k = 1 to 4, fp32 1500 x 1024, 32000
// 0.27, 0.43, 0.61 and 0.73.
__host__ __device__ static inline int head_rows(int M, int nt, int slices, int cus, int planes)
{
    uint32_t n = 0, best = 0;
    for (uint32_t k = 4; k >= 1; --k) {
        const uint32_t cost = (((uint32_t)M + 64 * k - 1) / (64 * k) * (uint32_t)(nt * slices) + (uint32_t)cus - 1) / (uint32_t)cus * (4 * k + (planes == 1 ? 7 : 3));
        if (n == 0 || cost < best) n = k, best = cost;
    }
    return (int)n;
}

// Fixed: the height is the host's (dW, whose rows are the vocabulary).  Otherwise the rows are the tokens with a target, whose number is known
// on the device alone, and the height is what head_tokens_kernel found for them: as against the height for all T, fp32 274 x 1120,
// vocabulary 59721, 10 % masked: 1505 -> 1235 us; nothing masked, 700 x 1024, 9000: 1 us a product more.
template <int NU, int EPI, int NSEG>
__global__ __launch_bounds__(256) void head_product_kernel(head_prod p)
{
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tokens = __builtin_amdgcn_readfirstlane(p.held[0]);
    if (NU > 0) {
        p.kt = max(8, ((tokens + 63) >> 6) * 2);
        hp_run<NU ? NU : 2, EPI, NSEG>(smem, p, wave);
        return;
    }
    const int n = __builtin_amdgcn_readfirstlane(p.held[EPI < HEAD_ACC ? 1 : 2]);
    p.M = tokens;
    if (EPI == HEAD_P && tokens <= 192) {  // (dW has eight steps at least: rows of P that no tile reaches)
        const int KTp = p.nt * (HP_TILE / HP_BK), b0 = (tokens + 63) >> 6 << 2, per = 16 - b0;
        for (int i = blockIdx.x * 4 + wave; i < KTp * per; i += gridDim.x * 4)
#pragma unroll
            for (int q = 0; q < (NSEG > 1 ? 3 : 1); ++q) {
                const int kb = i / per, b = b0 + i - kb * per;
                *(uint4 *)(p.P + q * p.planeP + ((((size_t)(b >> 3) * KTp + kb) * 8 + (b & 7)) << 10) + hp_lane() * 16) = make_uint4(0, 0, 0, 0);
            }
    }
    if (n == 4) {
        p.mt = (tokens + 255) >> 8;
        hp_run<8, EPI, NSEG>(smem, p, wave);
    } else if (n == 3) {
        p.mt = (tokens + 191) / 192;
        hp_run<6, EPI, NSEG>(smem, p, wave);
    } else if (n == 2) {
        p.mt = (tokens + 127) >> 7;
        hp_run<4, EPI, NSEG>(smem, p, wave);
    } else {
        p.mt = (tokens + 63) >> 6;
        hp_run<2, EPI, NSEG>(smem, p, wave);
    }
}

// ---- tile images ----
// Parts of 8 columns from c on of row `row` of a row-major matrix of K columns, zero from K on
template <bool BF>
__device__ __forceinline__ void head_chunk(const void *__restrict__ src, size_t row, int K, int c, int vec, uint4 (&part)[BF ? 1 : 3])
{
    constexpr int NP = BF ? 1 : 3;
    uint32_t w[NP][4];
    const size_t at = row * K + c;
    if (BF) {
        const bf16_t *s = (const bf16_t *)src + at;
        if (vec) {
            part[0] = *(const uint4 *)s;
            return;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) w[0][k] = (c + 2 * k < K ? (uint32_t)s[2 * k] : 0u) | (c + 2 * k + 1 < K ? (uint32_t)s[2 * k + 1] : 0u) << 16;
    } else {
        const float *s = (const float *)src + at;
        float v[8];
        if (vec) {
            *(float4 *)&v[0] = *(const float4 *)s;
            *(float4 *)&v[4] = *(const float4 *)(s + 4);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = c + k < K ? s[k] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t two[3];
            hp_split2<true>(v[2 * k], v[2 * k + 1], two);
#pragma unroll
            for (int q = 0; q < NP; ++q) w[q][k] = two[q];
        }
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) part[q] = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
}

// Rows 64 bx .., columns 64 by .. of W [R,K] as parts of a tile image (KTi k steps a row group), zero outside the matrix
template <bool BF>
__global__ __launch_bounds__(256) void head_images_kernel(const void *__restrict__ src, int R, int K, int vec, unsigned char *__restrict__ img, int KTi, size_t plane)
{
    constexpr int NP = BF ? 1 : 3;
    const int tid = threadIdx.x, r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int idx = tid + u * 256, row = r0 + (idx >> 3), c = c0 + (idx & 7) * 8;
        uint4 part[NP] = {};
        if (row < R && c < K) head_chunk<BF>(src, row, K, c, vec, part);
#pragma unroll
        for (int q = 0; q < NP; ++q) *(uint4 *)(img + q * plane + pk_chunk_off(row, c >> 5, (c & 31) >> 3, KTi)) = part[q];
    }
}

// The tokens that have a target, moved together in their order: x's image, their targets and (where the backward pass wants them) statistics,
// slot[t] = a token's place or -1, held = their number n, the tile heights of the products over them.  The products work on n rows, whatever the others hold; the image's rows from n on are
// zeros.  A workgroup takes 64 tokens and counts for itself how many of those before have a target: a launch less than a scan of its own
// (T / 64 workgroups read T targets each, a few us for thousands of tokens).
template <bool BF>
__global__ __launch_bounds__(256) void head_tokens_kernel(const void *__restrict__ x, int T, int d, int vec, const int32_t *__restrict__ targets, int V,
                                                          const float *__restrict__ row_stats, unsigned char *__restrict__ img, int KTi, size_t plane,
                                                          int32_t *__restrict__ held, int32_t *__restrict__ slot, int32_t *__restrict__ tok_target,
                                                          float *__restrict__ tok_stats, int nt_v, int slices_v, int nt_d, int slices_d, int cus)
{
    constexpr int NP = BF ? 1 : 3;
    __shared__ int counts[2][4], place[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r0 = blockIdx.x * 64;
    int before = 0, all = 0;
#pragma unroll 4
    for (int t = tid; t < T; t += 256) {
        const int y = targets[t], h = y >= 0 && y < V;
        all += h;
        before += t < r0 ? h : 0;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        all += __shfl_xor(all, o, 64);
        before += __shfl_xor(before, o, 64);
    }
    if (lane == 0) counts[0][wave] = before, counts[1][wave] = all;
    __syncthreads();
    before = counts[0][0] + counts[0][1] + counts[0][2] + counts[0][3];
    const int n = counts[1][0] + counts[1][1] + counts[1][2] + counts[1][3];
    if (wave == 0) {
        const int t = r0 + lane, y = t < T ? targets[t] : -1;
        const bool h = y >= 0 && y < V;
        const uint64_t mask = __ballot(h);
        const int at = h ? before + __popcll(mask & ((1ull << lane) - 1)) : -1;
        place[lane] = at;
        if (blockIdx.y == 0) {
            if (t < T) slot[t] = at;
            if (h) {
                tok_target[at] = y;
                if (tok_stats) {
                    tok_stats[at] = row_stats[t];
                    tok_stats[T + at] = row_stats[T + t];
                }
            }
            if (t == 0) {
                held[0] = n;
                held[1] = head_rows(n, nt_v, slices_v, cus, NP);
                held[2] = head_rows(n, nt_d, slices_d, cus, NP);
            }
        }
    }
    __syncthreads();
    for (int c0 = blockIdx.y * 64; c0 < KTi * 32; c0 += gridDim.y * 64) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int idx = tid + u * 256, rr = idx >> 3, row = r0 + rr, c = c0 + (idx & 7) * 8, at = place[rr];
            uint4 part[NP] = {};
            if (row >= n)
#pragma unroll
                for (int q = 0; q < NP; ++q) *(uint4 *)(img + q * plane + pk_chunk_off(row, c >> 5, (c & 31) >> 3, KTi)) = part[q];
            if (at < 0) continue;
            if (c < d) head_chunk<BF>(x, row, d, c, vec, part);
#pragma unroll
            for (int q = 0; q < NP; ++q) *(uint4 *)(img + q * plane + pk_chunk_off(at, c >> 5, (c & 31) >> 3, KTi)) = part[q];
        }
    }
}

// ---- a few tokens: W streams through registers ----
// A workgroup takes 16 NF rows of W; its four waves share k.  Lane l holds 16 bytes (8 or 4 k) of row l % 16 and of token l % 16, k
// chunk l / 16: a fragment of v_mfma_f32_16x16x32_bf16, or four of v_mfma_f32_16x16x4_f32 (any order of k serves, as long as both
// operands have it).  The waves' sums are added in LDS in wave order; (max, sum) of each token over the rows go to `part`.
// 16 bytes from element k of a row of K elements at p on (at the alignment of an element), zero from element K on
typedef uint32_t u32x4_el __attribute__((ext_vector_type(4), aligned(2)));
template <bool BF>
__device__ __forceinline__ u32x4_t head_few_load(const unsigned char *p, int k, int K)
{
    constexpr int W = BF ? 8 : 4, ES = BF ? 2 : 4;
    u32x4_t v = {0u, 0u, 0u, 0u};
    if (k + W <= K) {
        const u32x4_el u = *(const u32x4_el *)(p + (size_t)k * ES);
        v = u32x4_t{u[0], u[1], u[2], u[3]};
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (k + j < K) {
                if (BF) v[j >> 1] |= (uint32_t)((const bf16_t *)p)[k + j] << (16 * (j & 1));
                else v[j & 3] = ((const uint32_t *)p)[k + j];
            }
    }
    return v;
}
// 16 rows of W and 16 tokens, 16 bytes of k a lane
template <bool BF>
__device__ __forceinline__ void head_few_mfma(const u32x4_t &w, const u32x4_t &x, f32x4_t &acc)
{
    if (BF) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8_t *)&w, *(const bf16x8_t *)&x, acc, 0, 0, 0);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[j]), __uint_as_float(x[j]), acc, 0, 0, 0);
    }
}
// The end of both streaming kernels: the four waves' sums added in wave order, (max, sum) of each token over the workgroup's rows of W.
template <bool BF, int NF, int TF>
__device__ __forceinline__ void head_few_end(f32x4_t (&acc)[TF][NF], f32x4_t (*sums)[TF][NF][64], int t0, int T, int V, int v0, const int32_t *__restrict__ targets,
                                             float2 *__restrict__ part, float *__restrict__ tlogit)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, lq = lane >> 4;
    if (wave > 0)
#pragma unroll
        for (int q = 0; q < TF; ++q)
#pragma unroll
            for (int f = 0; f < NF; ++f) sums[wave - 1][q][f][lane] = acc[q][f];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int q = 0; q < TF; ++q) {
        const int t = t0 + 16 * q + l16;
        float m = -INFINITY, s = 0.0f;
        const int y = t < T ? targets[t] : -1;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            f32x4_t &a = acc[q][f];
            a = ((a + sums[0][q][f][lane]) + sums[1][q][f][lane]) + sums[2][q][f][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int v = v0 + 16 * f + 4 * lq + r;
                if (v >= V) a[r] = -INFINITY;
                else if (v == y && t < T) tlogit[t] = a[r];
                m = fmaxf(m, a[r]);
            }
        }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float m0 = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) s += hp_exp<BF ? 1 : 6>(acc[q][f][r] - m0);
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (t < T && lq == 0) part[(size_t)blockIdx.x * T + t] = make_float2(m, s);
    }
}

template <bool BF, int NF, int TF>
__global__ __launch_bounds__(256) void head_few_kernel(const void *__restrict__ x, const void *__restrict__ w, int T, int V, int K, const int32_t *__restrict__ targets,
                                                       float2 *__restrict__ part, float *__restrict__ tlogit)
{
    __shared__ f32x4_t sums[3][TF][NF][64];
    constexpr int KS = BF ? 32 : 16, ES = BF ? 2 : 4, UN = 8 / NF;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, lq = lane >> 4;
    const int v0 = blockIdx.x * 16 * NF, t0 = blockIdx.y * 16 * TF;
    const unsigned char *xr[TF], *wr[NF];
#pragma unroll
    for (int q = 0; q < TF; ++q) xr[q] = (const unsigned char *)x + (size_t)min(t0 + 16 * q + l16, T - 1) * K * ES;
#pragma unroll
    for (int f = 0; f < NF; ++f) wr[f] = (const unsigned char *)w + (size_t)min(v0 + 16 * f + l16, V - 1) * K * ES;
    f32x4_t acc[TF][NF];
#pragma unroll
    for (int q = 0; q < TF; ++q)
#pragma unroll
        for (int f = 0; f < NF; ++f) acc[q][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (K + KS - 1) / KS, first = wave * steps / 4, last = (wave + 1) * steps / 4;
    const int whole = min(last, K / KS);  // steps that are all there
    int at = first;
    for (; at + UN <= whole; at += UN) {
        u32x4_t xv[UN][TF], wv[UN][NF];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const size_t k = ((size_t)(at + u) * KS + lq * (KS / 4)) * ES;
#pragma unroll
            for (int q = 0; q < TF; ++q) {
                const u32x4_el a = *(const u32x4_el *)(xr[q] + k);
                xv[u][q] = u32x4_t{a[0], a[1], a[2], a[3]};
            }
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const u32x4_el b = *(const u32x4_el *)(wr[f] + k);
                wv[u][f] = u32x4_t{b[0], b[1], b[2], b[3]};
            }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int q = 0; q < TF; ++q)
#pragma unroll
                for (int f = 0; f < NF; ++f) head_few_mfma<BF>(wv[u][f], xv[u][q], acc[q][f]);
    }
    for (; at < last; ++at) {
        const int k = at * KS + lq * (KS / 4);
        u32x4_t wv[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) wv[f] = head_few_load<BF>(wr[f], k, K);
#pragma unroll
        for (int q = 0; q < TF; ++q) {
            const u32x4_t xv = head_few_load<BF>(xr[q], k, K);
#pragma unroll
            for (int f = 0; f < NF; ++f) head_few_mfma<BF>(wv[f], xv, acc[q][f]);
        }
    }
    head_few_end<BF, NF, TF>(acc, sums, t0, T, V, v0, targets, part, tlogit);
}

// The same for rows of whole 16-byte pieces: a wave brings 64 rows of W and the tokens' rows, 128 bytes of each, into a ring of LDS of
// its own by direct loads, whole lines at a time (loads of 16 rows x 64 bytes straight into registers ask for every line twice: one
// token x 4096, vocabulary 128000: 188 us, so 164, 6.4 TB/s).  A block of 8 rows is 1 KiB; chunk c of row r lies at slot c ^ r.
#define HS_STAGES 2   // (80 KiB up to 16 tokens: two workgroups a compute unit; one with three or four stages: 164 -> 168 us)
#define HS_LOADS(TF) (8 + 2 * (TF))  // 8 of W, 2 of 16 tokens each
template <bool BF, int TF>
__global__ __launch_bounds__(256) void head_stream_kernel(const unsigned char *__restrict__ x, const unsigned char *__restrict__ w, int T, int V, int row_bytes,
                                                          const int32_t *__restrict__ targets, float2 *__restrict__ part, float *__restrict__ tlogit)
{
    constexpr int STAGE = HS_LOADS(TF) * 1024;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];  // [4 waves][HS_STAGES][STAGE]; then the waves' sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, lq = lane >> 4;
    const int v0 = blockIdx.x * 64, t0 = blockIdx.y * 16 * TF;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem + wave * (HS_STAGES * STAGE);
    const unsigned char *mine = smem + wave * (HS_STAGES * STAGE);
    const int steps = (row_bytes + 127) / 128, first = wave * steps / 4, n = (wave + 1) * steps / 4 - first;
    const int last = wave == 3 ? row_bytes - (steps - 1) * 128 : 128;  // bytes of the wave's last step that are there
    const uint32_t r8 = lane >> 3, ch = ((lane & 7) ^ r8) * 16;
    const unsigned char *wb = hp_uniform(w + (size_t)v0 * row_bytes + (size_t)first * 128), *xb = hp_uniform(x + (size_t)t0 * row_bytes + (size_t)first * 128);
    uint32_t vw[8], vx[2 * TF];
#pragma unroll
    for (int i = 0; i < 8; ++i) vw[i] = (uint32_t)min(8 * i + (int)r8, V - 1 - v0) * (uint32_t)row_bytes + ch;
#pragma unroll
    for (int i = 0; i < 2 * TF; ++i) vx[i] = (uint32_t)min(8 * i + (int)r8, T - 1 - t0) * (uint32_t)row_bytes + ch;
    auto ask = [&](int step, int stage) {
        const uint32_t sb = lds0 + stage * STAGE;
        if (step == n - 1 && last < 128) {  // the row's end: what is behind it is read from before it, and counts as zero below
            const uint32_t back = max((int)ch + 16 - last, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) vw[i] -= back;
#pragma unroll
            for (int i = 0; i < 2 * TF; ++i) vx[i] -= back;
        }
        hp_dma16_nt<0>(wb, vw[0], sb); hp_dma16_nt<1 * 1024>(wb, vw[1], sb); hp_dma16_nt<2 * 1024>(wb, vw[2], sb); hp_dma16_nt<3 * 1024>(wb, vw[3], sb);
        hp_dma16_nt<4 * 1024>(wb, vw[4], sb); hp_dma16_nt<5 * 1024>(wb, vw[5], sb); hp_dma16_nt<6 * 1024>(wb, vw[6], sb); hp_dma16_nt<7 * 1024>(wb, vw[7], sb);
        hp_dma16<8 * 1024>(xb, vx[0], sb); hp_dma16<9 * 1024>(xb, vx[1], sb);
        if constexpr (TF > 1) { hp_dma16<10 * 1024>(xb, vx[2], sb); hp_dma16<11 * 1024>(xb, vx[3], sb); }
        if constexpr (TF > 2) { hp_dma16<12 * 1024>(xb, vx[4], sb); hp_dma16<13 * 1024>(xb, vx[5], sb); hp_dma16<14 * 1024>(xb, vx[6], sb); hp_dma16<15 * 1024>(xb, vx[7], sb); }
        wb += 128;
        xb += 128;
    };
    f32x4_t acc[TF][4];
#pragma unroll
    for (int q = 0; q < TF; ++q)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[q][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < HS_STAGES - 1 && i < n; ++i) ask(i, i);
    int stage = 0;
    for (int i = 0; i < n; ++i) {
        // this step's loads have landed (the next steps' may be in flight), and what was read from the stage that is filled next is here
        if (i + HS_STAGES - 1 <= n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((HS_STAGES - 2) * HS_LOADS(TF)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (i + HS_STAGES - 1 < n) ask(i + HS_STAGES - 1, stage == 0 ? HS_STAGES - 1 : stage - 1);
        const unsigned char *p = mine + stage * STAGE + (l16 >> 3) * 1024 + (l16 & 7) * 128;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = ((4 * h + lq) ^ (l16 & 7)) * 16;
            const bool none = i == n - 1 && (4 * h + lq) * 16 >= last;
            const u32x4_t zero = {0u, 0u, 0u, 0u};
            u32x4_t xv[TF];
#pragma unroll
            for (int q = 0; q < TF; ++q) {
                xv[q] = *(const u32x4_t *)(p + 8192 + q * 2048 + at);
                if (none) xv[q] = zero;
            }
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                u32x4_t wv = *(const u32x4_t *)(p + f * 2048 + at);
                if (none) wv = zero;
#pragma unroll
                for (int q = 0; q < TF; ++q) head_few_mfma<BF>(wv, xv[q], acc[q][f]);
            }
        }
        stage = stage + 1 == HS_STAGES ? 0 : stage + 1;
    }
    __syncthreads();  // (the rings are done with: the sums take their place)
    head_few_end<BF, 4, TF>(acc, (f32x4_t(*)[TF][4][64])smem, t0, T, V, v0, targets, part, tlogit);
}

// ---- joins ----
__device__ __forceinline__ float2 head_join2(float2 a, float2 b)
{
    const float m = fmaxf(a.x, b.x), m0 = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * expf(a.x - m0) + b.y * expf(b.x - m0));
}
// mean[0] = sum of the losses / n, mean[1] = n, by one workgroup (sums in double: a large batch's do not lose the small losses)
__device__ void head_mean(const float *loss, const int32_t *targets, int T, int V, float *mean)
{
    __shared__ double sd[16];
    __shared__ int sn[16];
    double a = 0.0;
    int n = 0;
    for (int t = threadIdx.x; t < T; t += blockDim.x) {
        const bool held = targets[t] >= 0 && targets[t] < V;
        n += held;
        if (held) a += (double)loss[t];
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        a += __shfl_xor(a, m, 64);
        n += __shfl_xor(n, m, 64);
    }
    if ((threadIdx.x & 63) == 0) sd[threadIdx.x >> 6] = a, sn[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < (int)(blockDim.x >> 6); ++w) a += sd[w], n += sn[w];
        mean[0] = n > 0 ? (float)(a / n) : 0.0f;
        mean[1] = (float)n;
    }
}
// (max, sum) of a token over nb column blocks: TL tokens (a power of two) a workgroup, 1024 / TL threads each, joined in a fixed order.
// A launch of one workgroup forms the mean too.  (By the last of several, behind a counter and the fences that takes: 5 us more than none,
// a launch of its own 3 to 4.)
__global__ __launch_bounds__(1024) void head_join_kernel(const float2 *__restrict__ part, int nb, const float *__restrict__ tlogit, const int32_t *__restrict__ targets,
                                                         const int32_t *__restrict__ slot, int T, int V, int TL, float *__restrict__ loss, float *__restrict__ row_stats, float *__restrict__ mean)
{
    __shared__ float2 red[1024];
    const int tid = threadIdx.x, sub = tid / TL, n_sub = 1024 / TL, t = blockIdx.x * TL + (tid & (TL - 1));
    // the maximum first: one exp a block instead of two
    float m = -INFINITY, s = 0.0f;
    const int at = t < T ? (slot ? slot[t] : t) : -1;  // (a token without a target has no place)
    if (at >= 0) {
#pragma unroll 8
        for (int b = sub; b < nb; b += n_sub) m = fmaxf(m, part[(size_t)b * T + at].x);
        const float m0 = m == -INFINITY ? 0.0f : m;
#pragma unroll 8
        for (int b = sub; b < nb; b += n_sub) {
            const float2 v = part[(size_t)b * T + at];
            s += v.y * expf(v.x - m0);
        }
    }
    red[tid] = make_float2(m, s);
    __syncthreads();
    for (int h = 512; h >= TL; h >>= 1) {
        if (tid < h) red[tid] = head_join2(red[tid], red[tid + h]);
        __syncthreads();
    }
    if (tid < TL && t < T) {
        const float2 v = red[tid];
        const int y = targets[t];
        loss[t] = y >= 0 && y < V ? (v.x - tlogit[at]) + logf(v.y) : 0.0f;
        if (row_stats) {
            row_stats[t] = at >= 0 ? v.x : 0.0f;
            row_stats[T + t] = at >= 0 ? v.y : 1.0f;
        }
    }
    if (gridDim.x == 1) {
        __syncthreads();
        head_mean(loss, targets, T, V, mean);
    }
}
__global__ __launch_bounds__(1024) void head_mean_kernel(const float *loss, const int32_t *__restrict__ targets, int T, int V, float *__restrict__ mean)
{
    head_mean(loss, targets, T, V, mean);
}

// ---- logits in slabs of k slices ----
__device__ __forceinline__ f32x4_t head_logits4(const float *at, int slices, size_t slab)
{
    f32x4_t l = *(const f32x4_t *)at;
#pragma unroll 4
    for (int k = 1; k < slices; ++k) l += *(const f32x4_t *)(at + k * slab);
    return l;
}

// Loss and statistics of token blockIdx.x: every thread a maximum and a sum of its own columns, joined in a fixed order
template <int NSEG>
__global__ __launch_bounds__(256) void head_slab_loss_kernel(const float *__restrict__ slabs, int slices, size_t slab, int ld, const int32_t *__restrict__ slot,
                                                             const int32_t *__restrict__ targets, int T, int V, float *__restrict__ loss, float *__restrict__ row_stats)
{
    __shared__ float2 red[256];
    const int t = blockIdx.x, at = slot[t], tid = threadIdx.x;
    if (at < 0) {
        if (tid == 0) {
            loss[t] = 0.0f;
            if (row_stats) row_stats[t] = 0.0f, row_stats[T + t] = 1.0f;
        }
        return;
    }
    const float *row = slabs + (size_t)at * ld;
    float m = -INFINITY, s = 0.0f;
    for (int c = 4 * tid; c < V; c += 1024) {
        f32x4_t l = head_logits4(row + c, slices, slab);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k >= V) l[k] = -INFINITY;
        const float m1 = fmaxf(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), m), m0 = m1 == -INFINITY ? 0.0f : m1;
        s = s * hp_exp<NSEG>(m - m0) + ((hp_exp<NSEG>(l[0] - m0) + hp_exp<NSEG>(l[1] - m0)) + (hp_exp<NSEG>(l[2] - m0) + hp_exp<NSEG>(l[3] - m0)));
        m = m1;
    }
    red[tid] = make_float2(m, s);
    __syncthreads();
    for (int h = 128; h; h >>= 1) {
        if (tid < h) red[tid] = head_join2(red[tid], red[tid + h]);
        __syncthreads();
    }
    if (tid == 0) {
        const float2 v = red[0];
        float l = 0.0f;
        for (int k = 0; k < slices; ++k) l = k ? l + row[k * slab + targets[t]] : row[targets[t]];
        loss[t] = (v.x - l) + logf(v.y);
        if (row_stats) row_stats[t] = v.x, row_stats[T + t] = v.y;
    }
}

// Gradient of the logits as tile images, row blockIdx.x: zeros behind the tokens with a target and behind the vocabulary
template <int NSEG>
__global__ __launch_bounds__(256) void head_slab_p_kernel(const float *__restrict__ slabs, int slices, size_t slab, int ld, const int32_t *__restrict__ held,
                                                          const int32_t *__restrict__ targets, const float *__restrict__ stats, int T, int V,
                                                          unsigned char *__restrict__ P, int KTp, size_t plane)
{
    constexpr int NP = NSEG > 1 ? 3 : 1;
    const int row = blockIdx.x, c = 8 * (blockIdx.y * 256 + threadIdx.x);
    if (c >= 32 * KTp) return;
    float v[8] = {};
    if (row < held[0] && c < V) {
        const int y = targets[row];
        const float m = stats[row], f = 1.0f / stats[T + row];
        const float *at = slabs + (size_t)row * ld + c;
        const f32x4_t a = head_logits4(at, slices, slab), b = head_logits4(at + 4, slices, slab);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < V ? hp_exp<NSEG>((k < 4 ? a[k & 3] : b[k & 3]) - m) * f - (c + k == y ? 1.0f : 0.0f) : 0.0f;
    }
    uint32_t w[NP][4];
    if (NSEG == 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[0][k] = hp_pack2(v[2 * k], v[2 * k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t two[3];
            hp_split2<false>(v[2 * k], v[2 * k + 1], two);
#pragma unroll
            for (int q = 0; q < NP; ++q) w[q][k] = two[q];
        }
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) *(uint4 *)(P + q * plane + pk_chunk_off(row, c >> 5, (c & 31) >> 3, KTp)) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
}

// dx: the slabs added in slice order, rounded once; rows without a target are zero.  Rows from `first` on
template <bool BF>
__global__ __launch_bounds__(256) void head_dx_kernel(const float *__restrict__ slabs, int slices, size_t slab, int ld, const int32_t *__restrict__ slot, int first,
                                                      int d, int vec, const float *__restrict__ mean, const float *dloss, void *__restrict__ dx)
{
    const float g = head_scale(mean, dloss);
    const int t = first + blockIdx.x, at = slot[t];
    for (int c = 4 * (blockIdx.y * 256 + threadIdx.x); c < d; c += 4 * gridDim.y * 256) {
        f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
        if (at >= 0) {
#pragma unroll 4
            for (int k = 0; k < slices; ++k) s += *(const f32x4_t *)(slabs + (size_t)k * slab + (size_t)at * ld + c);
            s *= g;
        }
        const size_t o = (size_t)t * d + c;
        if (vec) {
            if (BF) *(uint2 *)((bf16_t *)dx + o) = make_uint2(hp_pack2(s[0], s[1]), hp_pack2(s[2], s[3]));
            else *(f32x4_t *)((float *)dx + o) = s;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c + k < d) {
                    if (BF) ((bf16_t *)dx)[o + k] = f32_to_bf16(s[k]);
                    else ((float *)dx)[o + k] = s[k];
                }
        }
    }
}
__global__ __launch_bounds__(256) void head_zero_kernel(void *p, size_t bytes)  // (memset nodes are not for captured graphs)
{
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (size_t)gridDim.x * 256) ((unsigned char *)p)[i] = 0;
}

// ---- host side ----
static size_t up_to(size_t x, size_t m) { return (x + m - 1) / m * m; }
#define HEAD_DX_ROWS (1 << 18)  // rows of a launch of head_dx_kernel (lanes in x are counted in 32 bits)
static int k_pad(int n) { return std::max(256, (int)up_to(n, 64)); }  // k of a product: whole pairs of steps, eight steps or more

// Sizes of a call and where its parts lie in the workspace
struct head_plan {
    int planes, dp, Tp, piece, pieces;  // k of d, k of T, columns of a piece (a multiple of 256)
    int nb;                             // column blocks of the forward pass
    int slices, lslices;                // k slices of dx; of the logits, 0: their tiles are enough
    bool direct, few;
    size_t x_img, w_img, p_img, slabs, part, tlogit, held, slot, tok_target, tok_stats, bytes;
    size_t x_plane, w_plane, p_plane, slab, lslab, lslabs;
};

static head_plan head_plan_of(const omega_ctx *ctx, const head_args &a, bool backward)
{
    head_plan h = {};
    h.planes = a.dtype == OMEGA_DTYPE_BF16 ? 1 : 3;
    h.few = !backward && a.T <= HEAD_FEW(a.dtype) && a.V <= 1 << 29;  // (256 lanes for 64 rows of W: counted in 32 bits)
    h.dp = k_pad(a.d);
    h.Tp = k_pad(a.T);
    // W in place: bf16 rows of whole pairs of k steps, 16-byte aligned (tile offsets within 32 bits)
    h.direct = h.planes == 1 && a.d == h.dp && (uintptr_t)a.w % 16 == 0 && a.d <= (1 << 20);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += up_to(bytes, 1024);
        return o;
    };
    if (h.few) {
        h.nb = a.V > 0 ? ceil_div(a.V, 16) : 0;  // (an upper bound: workgroups of 16 rows)
        h.part = take((size_t)h.nb * a.T * sizeof(float2));
        h.tlogit = take((size_t)a.T * 4);
        h.bytes = at;
        return h;
    }
    // what a column of the vocabulary needs while its piece is worked on
    const size_t per = (size_t)h.planes * 2 * ((backward ? h.Tp : 0) + (h.direct ? 0 : h.dp));
    const size_t budget = (size_t)1 << 30;
    const int all = (int)up_to(a.V, 256);
    h.piece = per == 0 ? all : (int)std::min<size_t>(all, std::max<size_t>(256, budget / per / 256 * 256));
    h.pieces = ceil_div(a.V, h.piece);
    h.piece = (int)up_to(ceil_div(a.V, h.pieces), 256);
    h.x_plane = up_to(backward ? h.Tp : a.T, 128) * (size_t)h.dp * 2;
    h.x_img = take(h.x_plane * h.planes);
    h.held = take(12);
    h.slot = take((size_t)a.T * 4);
    h.tok_target = take((size_t)a.T * 4);
    if (backward) h.tok_stats = take((size_t)a.T * 8);
    if (!h.direct) {
        h.w_plane = (size_t)h.piece * h.dp * 2;
        h.w_img = take(h.w_plane * h.planes);
    }
    // Few tiles of the logits, as a small vocabulary has: d is shared out to k slices, whose sums head_slab_loss_kernel and
    // head_slab_p_kernel add, where that saves 24 steps or more.  Training steps, bf16 343 x 3904, vocabulary 2036: 143 -> 97 us, 250 x 2048,
    // 6000: 110 -> 99; fp32 252 x 2082, 2535, half masked: 294 -> 174; with 16 steps saved, bf16 2000 x 1024, 1000: 94 -> 99.
    const long long ltiles = (long long)ceil_div(a.T, 64) * ceil_div(a.V, 256);
    if (h.pieces == 1 && ltiles <= ctx->num_cus / 2) {
        const int n = std::min(ctx->num_cus / (int)ltiles, h.dp / 256), steps = h.dp / 32 * (h.planes == 1 ? 1 : 6);
        if (n > 1 && steps - steps / n >= 24) h.lslices = n;
    }
    if (h.lslices) {
        h.lslab = (up_to(a.T, 64) + 192) * up_to(a.V, 256);  // whole tiles
        h.lslabs = take(h.lslab * h.lslices * 4);
    }
    if (backward) {
        h.p_plane = up_to(h.Tp, 128) * (size_t)h.piece * 2;
        h.p_img = take(h.p_plane * h.planes);
        // few tiles of dx: the vocabulary is shared out to k slices, a slab of sums each
        const int tiles = ceil_div(a.T, 256) * ceil_div(a.d, 256);
        h.slices = tiles < ctx->num_cus ? std::max(1, std::min(ctx->num_cus / std::max(tiles, 1), h.piece / 32 / 16)) : 1;
        h.slab = (up_to(a.T, 64) + 192) * up_to(h.dp, 256);  // whole tiles
        h.slabs = take(h.slab * h.slices * 4);
    } else {
        h.nb = ceil_div(a.V, 256) * 2;
        h.part = take((size_t)h.nb * a.T * sizeof(float2));
        h.tlogit = take((size_t)a.T * 4);
    }
    h.bytes = at;
    return h;
}

size_t head_workspace(const omega_ctx *ctx, const head_args &a, bool backward) { return a.T > 0 ? head_plan_of(ctx, a, backward).bytes : 0; }

static const void *head_kernel_of(int epi, int planes, int rows)
{
#define HEAD_K(NU, E) (planes == 1 ? (const void *)head_product_kernel<NU, E, 1> : (const void *)head_product_kernel<NU, E, 6>)
    return epi == HEAD_LSE   ? HEAD_K(0, HEAD_LSE)
           : epi == HEAD_P   ? HEAD_K(0, HEAD_P)
           : epi == HEAD_LOG ? HEAD_K(0, HEAD_LOG)
           : epi == HEAD_ACC ? HEAD_K(0, HEAD_ACC)
           : epi == HEAD_ADD ? HEAD_K(0, HEAD_ADD)
           : rows == 4       ? HEAD_K(8, HEAD_OUT)
           : rows == 3       ? HEAD_K(6, HEAD_OUT)
           : rows == 2       ? HEAD_K(4, HEAD_OUT)
                             : HEAD_K(2, HEAD_OUT);
#undef HEAD_K
}
hipError_t head_init(void)
{
    for (const void *f : {(const void *)head_stream_kernel<true, 1>, (const void *)head_stream_kernel<true, 2>, (const void *)head_stream_kernel<true, 4>,
                          (const void *)head_stream_kernel<false, 1>, (const void *)head_stream_kernel<false, 2>, (const void *)head_stream_kernel<false, 4>}) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, HP_SMEM);
        if (e != hipSuccess) return e;
    }
    for (int epi = HEAD_LSE; epi <= HEAD_OUT; ++epi)
        for (int rows = 1; rows <= (epi == HEAD_OUT ? 4 : 1); ++rows)
            for (int planes = 1; planes <= 3; planes += 2) {
                const hipError_t e = hipFuncSetAttribute(head_kernel_of(epi, planes, rows), hipFuncAttributeMaxDynamicSharedMemorySize, HP_SMEM);
                if (e != hipSuccess) return e;
            }
    return hipSuccess;
}

static hipError_t head_product(const omega_ctx *ctx, int epi, head_prod p, int planes, hipStream_t s)
{
    p.nt = ceil_div(p.N, HP_TILE);
    const int rows = epi == HEAD_OUT ? head_rows(p.M, p.nt, p.slices, ctx->num_cus, planes) : 1;  // (1: the lowest, which makes the most items)
    p.mt = ceil_div(p.M, 64 * rows);
    const long long items = (long long)p.mt * p.nt * p.slices;
    if (items > 0x3fffffff) return hipErrorInvalidValue;
    const int grid = (int)std::min<long long>(up_to(items, 8), ctx->num_cus);
    void *args[] = {&p};
    return hipLaunchKernel(head_kernel_of(epi, planes, rows), dim3(grid), dim3(256), args, HP_SMEM, s);
}
#define HEAD_TRY(expr)                          \
    do {                                        \
        const hipError_t _e = (expr);           \
        if (_e != hipSuccess) return _e;        \
    } while (0)

// Images of rows [R,K] at src: rows up to Rp (a multiple of 64), columns up to Kp
static void head_images(const head_args &a, const void *w, int R, int Rp, int Kp, unsigned char *img, size_t plane, hipStream_t s)
{
    const int vec = a.d % 8 == 0 && (uintptr_t)w % 16 == 0;
    const dim3 grid(Rp / 64, Kp / 64);
    if (a.dtype == OMEGA_DTYPE_BF16) hipLaunchKernelGGL(head_images_kernel<true>, grid, dim3(256), 0, s, w, R, a.d, vec, img, Kp / 32, plane);
    else hipLaunchKernelGGL(head_images_kernel<false>, grid, dim3(256), 0, s, w, R, a.d, vec, img, Kp / 32, plane);
}

// k steps of dx over `vc` rows of W (P has zeros up to a multiple of 256)
static int head_dx_steps(int vc) { return std::max(8, (int)up_to(ceil_div(vc, 32), 2)); }
// ... and k slices over a piece
static int head_dx_slices(const head_args &a, const head_plan &h) { return std::max(1, std::min(h.slices, head_dx_steps(std::min(h.piece, a.V)) / 8)); }

static void head_tokens(const omega_ctx *ctx, const head_args &a, const head_plan &h, unsigned char *base, int Rp, const float *row_stats, hipStream_t s)
{
    const int vec = a.d % 8 == 0 && (uintptr_t)a.x % 16 == 0;
    // (as many workgroups a row of tiles as fill the machine; more would only count again)
    const dim3 grid(Rp / 64, std::min(h.dp / 64, std::max(1, 4096 / (Rp / 64))));
    const auto k = a.dtype == OMEGA_DTYPE_BF16 ? head_tokens_kernel<true> : head_tokens_kernel<false>;
    hipLaunchKernelGGL(k, grid, dim3(256), 0, s, a.x, a.T, a.d, vec, a.targets, a.V, row_stats, base + h.x_img, h.dp / 32, h.x_plane, (int32_t *)(base + h.held),
                       (int32_t *)(base + h.slot), (int32_t *)(base + h.tok_target), row_stats ? (float *)(base + h.tok_stats) : nullptr, ceil_div(std::min(h.piece, a.V), HP_TILE), std::max(1, h.lslices), ceil_div(a.d, HP_TILE),
                       head_dx_slices(a, h), ctx->num_cus);
}


static void head_zero(void *p, size_t bytes, hipStream_t s)
{
    if (bytes > 0) hipLaunchKernelGGL(head_zero_kernel, dim3((unsigned)std::min<size_t>((bytes + 255) / 256, 4096)), dim3(256), 0, s, p, bytes);
}

hipError_t launch_head_forward(const omega_ctx *ctx, const head_args &a, void *ws, hipStream_t s)
{
    if (a.T == 0) {
        head_zero(a.mean, 8, s);
        return hipGetLastError();
    }
    const head_plan h = head_plan_of(ctx, a, false);
    unsigned char *base = (unsigned char *)ws;
    float2 *part = (float2 *)(base + h.part);
    float *tlogit = (float *)(base + h.tlogit);
    const bool bf = a.dtype == OMEGA_DTYPE_BF16;
    const size_t es = bf ? 2 : 4;
    int nb = h.nb;
    if (h.few) {
        // 64 rows of W a workgroup read x a quarter as often as 16; vocabularies that would leave compute units idle take 16
        const int nf = a.V >= 64 * ctx->num_cus ? 4 : 1;
        nb = ceil_div(a.V, 16 * nf);
        const int row_bytes = a.d * (int)es, tf = a.T <= 16 ? 1 : a.T <= 32 ? 2 : 4;
        const dim3 grid(nb, ceil_div(a.T, 16 * tf));
        const unsigned char *x = (const unsigned char *)a.x, *w = (const unsigned char *)a.w;
#define HEAD_STREAM_K(B, TF)                                                                                                                             \
    hipLaunchKernelGGL((head_stream_kernel<B, TF>), grid, dim3(256), 4 * HS_STAGES * HS_LOADS(TF) * 1024, s, x, w, a.T, a.V, row_bytes, a.targets, part, \
                       tlogit)
#define HEAD_FEW_K(B, F, TF) hipLaunchKernelGGL((head_few_kernel<B, F, TF>), grid, dim3(256), 0, s, a.x, a.w, a.T, a.V, a.d, a.targets, part, tlogit)
#define HEAD_FEW_T(K, ...)                  \
    do {                                    \
        if (tf == 1) K(__VA_ARGS__, 1);     \
        else if (tf == 2) K(__VA_ARGS__, 2); \
        else K(__VA_ARGS__, 4);             \
    } while (0)
        if (nf == 4 && row_bytes % 16 == 0 && row_bytes >= 128 && ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0) {
            if (bf) HEAD_FEW_T(HEAD_STREAM_K, true);
            else HEAD_FEW_T(HEAD_STREAM_K, false);
        } else if (bf) {
            if (nf == 4) HEAD_FEW_T(HEAD_FEW_K, true, 4);
            else HEAD_FEW_T(HEAD_FEW_K, true, 1);
        } else {
            if (nf == 4) HEAD_FEW_T(HEAD_FEW_K, false, 4);
            else HEAD_FEW_T(HEAD_FEW_K, false, 1);
        }
#undef HEAD_FEW_T
#undef HEAD_FEW_K
#undef HEAD_STREAM_K
    } else {
        head_tokens(ctx, a, h, base, (int)up_to(a.T, 64), nullptr, s);
        for (int v0 = 0; v0 < a.V; v0 += h.piece) {
            const int vc = std::min(h.piece, a.V - v0);
            const unsigned char *w = (const unsigned char *)a.w + (size_t)v0 * a.d * es;
            if (!h.direct) head_images(a, w, vc, (int)up_to(vc, 64), h.dp, base + h.w_img, h.w_plane, s);
            head_prod p = {};
            p.A = base + h.x_img;
            p.planeA = h.x_plane;
            p.B = h.direct ? w : base + h.w_img;
            p.planeB = h.w_plane;
            p.b_ld = h.direct ? (size_t)a.d * 2 : 0;
            p.kt = p.ktA = p.ktB = h.dp / 32;
            p.M = p.rowsA = a.T;
            p.N = vc;
            p.slices = 1;
            p.held = (const int32_t *)(base + h.held);
            p.targets = (const int32_t *)(base + h.tok_target);
            p.T = a.T;
            p.v0 = v0;
            p.part = part;
            p.tlogit = tlogit;
            if (h.lslices) {
                p.slices = h.lslices;
                p.C = (float *)(base + h.lslabs);
                p.slab = h.lslab;
                p.ld = (int)up_to(a.V, 256);
            }
            HEAD_TRY(head_product(ctx, h.lslices ? HEAD_LOG : HEAD_LSE, p, h.planes, s));
        }
        if (h.lslices) {
            const auto k = bf ? head_slab_loss_kernel<1> : head_slab_loss_kernel<6>;
            hipLaunchKernelGGL(k, dim3(a.T), dim3(256), 0, s, (const float *)(base + h.lslabs), h.lslices, h.lslab, (int)up_to(a.V, 256),
                               (const int32_t *)(base + h.slot), a.targets, a.T, a.V, a.loss, a.row_stats);
            hipLaunchKernelGGL(head_mean_kernel, dim3(1), dim3(1024), 0, s, a.loss, a.targets, a.T, a.V, a.mean);
            return hipGetLastError();
        }
    }
    int TL = 1;
    while (TL < 64 && TL < a.T) TL *= 2;
    const int32_t *slot = h.few ? nullptr : (const int32_t *)(base + h.slot);
    hipLaunchKernelGGL(head_join_kernel, dim3(ceil_div(a.T, TL)), dim3(1024), 0, s, part, nb, tlogit, a.targets, slot, a.T, a.V, TL, a.loss, a.row_stats, a.mean);
    if (a.T > TL) hipLaunchKernelGGL(head_mean_kernel, dim3(1), dim3(1024), 0, s, a.loss, a.targets, a.T, a.V, a.mean);
    return hipGetLastError();
}

hipError_t launch_head_backward(const omega_ctx *ctx, const head_args &a, void *ws, hipStream_t s)
{
    const bool bf = a.dtype == OMEGA_DTYPE_BF16;
    const size_t es = bf ? 2 : 4;
    if (a.T == 0) {
        if (a.dw) head_zero(a.dw, (size_t)a.V * a.d * es, s);
        return hipGetLastError();
    }
    const head_plan h = head_plan_of(ctx, a, true);
    unsigned char *base = (unsigned char *)ws;
    head_tokens(ctx, a, h, base, h.Tp, a.row_stats, s);
    const int32_t *held = (const int32_t *)(base + h.held);
    for (int v0 = 0; v0 < a.V; v0 += h.piece) {
        const int vc = std::min(h.piece, a.V - v0), vp = (int)up_to(vc, 256);
        const unsigned char *w = (const unsigned char *)a.w + (size_t)v0 * a.d * es;
        if (!h.direct) head_images(a, w, vc, vp, h.dp, base + h.w_img, h.w_plane, s);
        head_prod p = {};
        p.A = base + h.x_img;
        p.planeA = h.x_plane;
        p.B = h.direct ? w : base + h.w_img;
        p.planeB = h.w_plane;
        p.b_ld = h.direct ? (size_t)a.d * 2 : 0;
        p.kt = p.ktA = p.ktB = h.dp / 32;
        p.M = a.T;
        p.rowsA = h.Tp;
        p.N = vc;
        p.slices = 1;
        p.held = held;
        p.targets = (const int32_t *)(base + h.tok_target);
        p.row_stats = (const float *)(base + h.tok_stats);
        p.T = a.T;
        p.v0 = v0;
        p.P = base + h.p_img;
        p.planeP = h.p_plane;
        if (h.lslices) {
            p.slices = h.lslices;
            p.C = (float *)(base + h.lslabs);
            p.slab = h.lslab;
            p.ld = vp;
            HEAD_TRY(head_product(ctx, HEAD_LOG, p, h.planes, s));
            const auto k = bf ? head_slab_p_kernel<1> : head_slab_p_kernel<6>;
            hipLaunchKernelGGL(k, dim3(h.Tp, ceil_div(vp, 2048)), dim3(256), 0, s, (const float *)p.C, h.lslices, h.lslab, vp, held, p.targets, p.row_stats, a.T, a.V, p.P,
                               vp / 32, h.p_plane);
        } else {
            HEAD_TRY(head_product(ctx, HEAD_P, p, h.planes, s));
        }
        if (a.dx) {
            head_prod q = {};
            q.A = base + h.p_img;
            q.planeA = h.p_plane;
            q.B = p.B;
            q.planeB = h.w_plane;
            q.b_ld = p.b_ld;
            q.kt = head_dx_steps(vc);
            q.ktA = vp / 32;
            q.ktB = h.dp / 32;
            q.held = held;
            q.M = q.rowsA = a.T;
            q.N = a.d;
            q.rowsB = vc;
            q.slices = std::max(1, std::min(h.slices, q.kt / 8));
            q.C = (float *)(base + h.slabs);
            q.slab = h.slab;
            q.ld = (int)up_to(h.dp, 256);
            if (v0 == 0) HEAD_TRY(head_product(ctx, HEAD_ACC, q, h.planes, s));
            else HEAD_TRY(head_product(ctx, HEAD_ADD, q, h.planes, s));
        }
        if (a.dw) {
            head_prod q = {};
            q.A = base + h.p_img;
            q.planeA = h.p_plane;
            q.B = base + h.x_img;
            q.planeB = h.x_plane;
            q.held = held;
            q.kt = h.Tp / 32;
            q.ktA = vp / 32;
            q.ktB = h.dp / 32;
            q.M = vc;
            q.N = a.d;
            q.slices = 1;
            q.out = (unsigned char *)a.dw + (size_t)v0 * a.d * es;
            q.out_bf = bf;
            q.mean = a.mean;
            q.dloss = a.dloss;
            q.out_vec = a.d % (bf ? 8 : 4) == 0 && (uintptr_t)q.out % 16 == 0;
            HEAD_TRY(head_product(ctx, HEAD_OUT, q, h.planes, s));
        }
    }
    if (a.dx) {
        const int slices = head_dx_slices(a, h);
        const int vec = a.d % 4 == 0 && (uintptr_t)a.dx % (bf ? 8 : 16) == 0;
        const auto k = bf ? head_dx_kernel<true> : head_dx_kernel<false>;
        for (int first = 0; first < a.T; first += HEAD_DX_ROWS) {
            const dim3 grid(std::min(a.T - first, HEAD_DX_ROWS), std::min(ceil_div(a.d, 1024), 1024));
            hipLaunchKernelGGL(k, grid, dim3(256), 0, s, (const float *)(base + h.slabs), slices, h.slab, (int)up_to(h.dp, 256), (const int32_t *)(base + h.slot), first, a.d, vec,
                               a.mean, a.dloss, a.dx);
        }
    }
    return hipGetLastError();
}
