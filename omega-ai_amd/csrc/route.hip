// Routing to experts from their logits z [T,E] (an operator of its own, and the selection of MoE layers that ask for it).
//
//   scores   softmax(z) over a token's open experts, or 1 / (1 + e^-z);  an expert is closed to a token where z is -infinity or no number
//   worth    score + bias (no bias: the score; a sum that is -infinity or no number closes the expert)
//   groups   E / groups consecutive experts each; a group's worth is the sum of its group_best best; the top_groups best stay
//   choice   the K best of what stays, by worth, without a bias by z; equal ones, experts and groups, in the order of their numbers
//   weights  w_j = scale s_j, with renorm divided by the sum of the chosen scores
//   back     renorm: dz_j = w_j sum_k (w_k / scale)(dw_j - dw_k) (1 - s_j for sigmoid); else sigmoid: w_j dw_j (1 - s_j), softmax: [chosen] w_j dw_j - s_e sum_k w_k dw_k
//
// The choice is that of worths in 64 bits.  They are formed in fp32, a few instructions an expert, and where two that the choice tells apart are nearer
// to each other than their errors, or equal, those few are formed in double and put in order; where they are not few, or it is groups, the whole token is
// chosen for again in double, by a wave of its workgroup at the end (route_exact).
// L lanes share a token, V experts a lane.  What is compared of an expert is one word: its worth as a whole number of the same order, the last bits
// replaced by the expert's place in its lane.  A lane sorts its words by minima and maxima and leaves them in LDS; a round of the choice is the largest of
// the lanes' first ones, found in the lanes' own pipeline, and a step in the list of the lane that holds it.
// Bound: waiting.  16384 x 256 with bias and groups takes 13 us, and 4 to 5 more where a token is chosen for again; 1086 vector instructions a wave, four
// waves a SIMD, are 7 of them, the bytes 3; a wave makes one round of its loop, and its fetch, its sort and its K + 2 rounds follow each other.  16384 x 128
// with neither: 6.5 us, 377 instructions (2.5), the bytes 2.  Logits that are equal or next to each other at the edge of the choice cost what is done in
// double: rounded to bf16 13.2 us a call in place of 8.7 (128 experts, softmax), a tenth of the rows at the lowest number 20.9, all of them equal 44.4.
#include <float.h>

#include <algorithm>

#include "common.h"
#include "rows.h"

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define ROUTE_MAX_E 512
#define ROUTE_TOKENS 1024     // of a workgroup, at most
#define ROUTE_NONE (-1)
#define ROUTE_FILL (1 << 16)  // chosen only because a layer's token has K experts whatever is open: weight 0

// what other lanes of a row of 16 hold, then across the rows
template <int CTRL>
__device__ __forceinline__ uint32_t lane_of(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float lane_of(float v)
{
    return __uint_as_float(lane_of<CTRL>(__float_as_uint(v)));
}
// `meet` of a value in the lanes of a token, the same in all of them
template <int L, class F>
__device__ __forceinline__ uint32_t over_token(uint32_t v, F meet)
{
    v = meet(v, lane_of<0x128>(v));  // row_ror 8, 4, 2, 1
    v = meet(v, lane_of<0x124>(v));
    v = meet(v, lane_of<0x122>(v));
    v = meet(v, lane_of<0x121>(v));
    if (L >= 32) {
        const u32x2 u = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = meet(u[0], u[1]);
    }
    if (L == 64) {
        const u32x2 u = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = meet(u[0], u[1]);
    }
    return v;
}
// the bits of a ballot that a token's lanes have
template <int L>
__device__ __forceinline__ unsigned long long token_bits(unsigned long long lanes)
{
    return L == 64 ? lanes : (lanes >> (threadIdx.x & (64 - L))) & ((1ull << (L & 63)) - 1);
}
// the first lane of each token's of a ballot that every token has a lane in
template <int L>
__device__ __forceinline__ unsigned long long first_lanes(unsigned long long lanes)
{
    return lanes & ((L == 64 ? 1ull : L == 32 ? 0x0000000100000001ull : 0x0001000100010001ull) + ~lanes);
}
template <int L>
__device__ __forceinline__ float token_max(float v)
{
    return __uint_as_float(over_token<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int L>
__device__ __forceinline__ float token_sum(float v)
{
    return __uint_as_float(over_token<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
template <int L>
__device__ __forceinline__ uint32_t token_max(uint32_t v)
{
    return over_token<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// e^x for x <= 0 to 2 units in the last place: 2^(x log2 e), what the product's rounding cuts off added to the result; 0 below 2^-126
__device__ __forceinline__ float exp_neg(float x)
{
    const float t = x * 0x1.715476p+0f, lo = fmaf(x, 0x1.715476p+0f, -t) + x * 0x1.4ae0cp-26f;
    const float e = __builtin_amdgcn_exp2f(t);
    return t < -126.0f ? 0.0f : fmaf(e, lo * 0x1.62e43p-1f, e);
}
// ... with the relative error |x| 2^-24 of the product: of a score that is some 2^-26, where e^x is large enough to matter x is small
__device__ __forceinline__ float exp_near(float x) { return __builtin_amdgcn_exp2f(x * 0x1.715476p+0f); }
__device__ __forceinline__ float sigmoid_near(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_near(-z)); }
__device__ __forceinline__ float sigmoid(float z)
{
    const float e = exp_neg(-fabsf(z));
    return (z >= 0.0f ? 1.0f : e) / (1.0f + e);
}
// the larger of v and -infinity: no number becomes -infinity.  v is a result of arithmetic: of a signalling NaN, which only memory holds, the instruction
// makes a quiet one (written out: the compiler would quiet v again in front of it)
__device__ __forceinline__ float or_closed(float v)
{
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(v), "s"(0xff800000u));
    return r;
}
// a logit as it is compared: closed ones -infinity, infinite ones the largest number (v from memory: quieted first, as fmaxf does)
__device__ __forceinline__ float open_logit(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX); }

// A float as a whole number of the same order; and back
#define ROUTE_OPEN 0x00800000u  // that of the lowest number: -infinity's is below, and so is 0
__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t u = __float_as_uint(v);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ unsigned long long ordered(double v)
{
    const unsigned long long u = *(const unsigned long long *)&v;
    return u ^ ((unsigned long long)((long long)u >> 63) | 1ull << 63);
}
__device__ __forceinline__ float of_ordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// element i of p, the same p in a wave
__device__ __forceinline__ float ld_at(const float *p, uint32_t i) { return *(const float *)((const char *)p + (i << 2)); }

// the lanes of a wave see each other's LDS writes
__device__ __forceinline__ void wave_lds()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct route_args {
    const float *logits, *bias;
    int T, E, K, sigmoid, renorm, groups, top_groups, group_best;
    int per_group, group_magic, group_shift;  // experts of a group; e / per_group = e magic >> 20; 1 << shift lanes look at a group
    float scale;
    int tokens;      // of a workgroup
    int fill;        // a layer's routing: every token gets K experts
    int vec;         // rows are 16-byte aligned and whole 16-byte pieces
    int32_t *ids;
    float *w;
    int32_t *part;   // [workgroups][E]: tokens that chose an expert
};

template <int CTRL>
__device__ __forceinline__ double lane_of(double v)
{
    const u32x2 u = *(const u32x2 *)&v;
    const u32x2 o = {lane_of<CTRL>(u[0]), lane_of<CTRL>(u[1])};
    return *(const double *)&o;
}
// `meet` of a double over a wave
template <class F>
__device__ __forceinline__ double over_wave(double v, F meet)
{
    v = meet(v, lane_of<0x128>(v));
    v = meet(v, lane_of<0x124>(v));
    v = meet(v, lane_of<0x122>(v));
    v = meet(v, lane_of<0x121>(v));
#define ACROSS(swap)                                                                              \
    do {                                                                                          \
        const u32x2 u = *(const u32x2 *)&v;                                                       \
        const u32x2 lo = swap(u[0], u[0], false, false), hi = swap(u[1], u[1], false, false);     \
        const u32x2 x = {lo[0], hi[0]}, y = {lo[1], hi[1]};                                       \
        v = meet(*(const double *)&x, *(const double *)&y);                                       \
    } while (0)
    ACROSS(__builtin_amdgcn_permlane16_swap);
    ACROSS(__builtin_amdgcn_permlane32_swap);
#undef ACROSS
    return v;
}

// The choice for one token in double, by a wave: lane j's place.  row: its logits; spare: room for 64 N doubles in LDS, where each lane keeps its experts'
// (loops that are not unrolled: few waves come here, and wait for their instructions most of all); top and recip: of its softmax.
template <int N>
__device__ __forceinline__ int route_exact(const route_args &a, const float *row, const float *bias, double *spare, float *top_out, float *recip_out)
{
    const int lane = threadIdx.x & 63, E = a.E;
    float z[N];  // of experts lane + 64 i
    double *own = spare + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = row[min(lane + 64 * i, E - 1)];
    float top = -FLT_MAX;
    uint32_t left = 0, shut = 0;  // bit i: expert lane + 64 i has not been chosen; it is closed
#pragma unroll
    for (int i = 0; i < N; ++i) {
        left |= lane + 64 * i < E ? 1u << i : 0u;
        z[i] = lane + 64 * i < E ? open_logit(z[i]) : -INFINITY;
        shut |= z[i] == -INFINITY ? 1u << i : 0u;
        top = fmaxf(top, z[i]);
    }
    wave_lds();  // (what the wave had there has been read)
#pragma unroll
    for (int i = 0; i < N; ++i) own[64 * i] = (double)z[i];
    double m = 0.0, sum = 1.0;
    if (!a.sigmoid) {
        m = (double)token_max<64>(top);
        sum = 0.0;
    }
#pragma unroll 1
    for (int i = 0; i < N; ++i) {  // (closed ones: e^-inf = 0)
        const double x = exp(a.sigmoid ? -own[64 * i] : own[64 * i] - m);
        own[64 * i] = x;
        if (!a.sigmoid) sum += x;
    }
    if (!a.sigmoid) sum = over_wave(sum, [](double x, double y) { return x + y; });
    *top_out = (float)m;
    *recip_out = sum > 0.0 ? (float)(1.0 / sum) : 0.0f;
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
        const double x = own[64 * i];
        double v = (a.sigmoid ? 1.0 : x) / (a.sigmoid ? 1.0 + x : sum);
        if (bias != nullptr) v += (double)bias[min(lane + 64 * i, E - 1)];
        own[64 * i] = ((shut >> i) & 1) || !(v == v) ? -INFINITY : v;
    }
    double key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = own[64 * i];
    if (a.groups > 1) {
        wave_lds();
        double best = -INFINITY;
        if (lane < a.groups) {
            double second = -INFINITY;
#pragma unroll 8
            for (int e = lane * a.per_group; e < (lane + 1) * a.per_group; ++e) {
                const double v = spare[e];
                second = fmax(second, fmin(best, v));
                best = fmax(best, v);
            }
            if (a.group_best == 2 && second > -INFINITY) best += second;
        }
        int ahead = 0;
        const u32x2 u = *(const u32x2 *)&best;
        for (int g = 0; g < a.groups; ++g) {
            const u32x2 o = {(uint32_t)__builtin_amdgcn_readlane((int)u[0], g), (uint32_t)__builtin_amdgcn_readlane((int)u[1], g)};
            const double v = *(const double *)&o;
            ahead += v > best || (v == best && g < lane) ? 1 : 0;
        }
        const unsigned long long stay = __ballot(lane < a.groups && ahead < a.top_groups);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!((stay >> (((uint32_t)(lane + 64 * i) * (uint32_t)a.group_magic >> 20) & 63)) & 1)) key[i] = -INFINITY;
        wave_lds();
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (bias == nullptr && key[i] > -INFINITY) key[i] = (double)z[i];
    int place = ROUTE_NONE;
    for (int j = 0; j < a.K; ++j) {
        double bv = -INFINITY;
        int be = INT_MAX;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (((left >> i) & 1) && (be == INT_MAX || key[i] > bv)) bv = key[i], be = lane + 64 * i;
        // the largest of the upper halves of their orders, mostly one lane's, else of the lower ones among those
        const unsigned long long o = be != INT_MAX ? ordered(bv + 0.0) : 0ull;
        const uint32_t hi = (uint32_t)(o >> 32), top = token_max<64>(hi);
        const bool none = top < 0x00100000u;  // (-infinity at best; a layer's token then takes the first of the others)
        if (none && !a.fill) break;
        int e = be != INT_MAX && hi == top ? be : INT_MAX;
        unsigned long long have = __ballot(e != INT_MAX);
        if (have & (have - 1)) {
            const uint32_t lo = e != INT_MAX ? (uint32_t)o : 0u;
            if (lo != token_max<64>(lo)) e = INT_MAX;
            for (int s = 32; s > 0; s >>= 1) e = min(e, __shfl_xor(e, s));  // equal ones: the first
        } else e = __builtin_amdgcn_readlane(e, __ffsll((long long)have) - 1);
        if ((e & 63) == lane) left &= ~(1u << (e >> 6));
        if (lane == j) place = none ? e | ROUTE_FILL : e;
    }
    return place;
}

// Weights of a token's chosen experts, and what is written of them: lane sub of L has the places sub, sub + L, ...
template <int L>
__device__ __forceinline__ void route_write(const route_args &a, const float *row, int t, bool live, int sub, const int (&at)[64 / L], float top, float recip, int *hist)
{
    constexpr int KL = 64 / L;
    float c[KL], zt = -INFINITY;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
        c[i] = at[i] >= 0 && at[i] < ROUTE_FILL ? open_logit(row[at[i]]) : -INFINITY;
        zt = fmaxf(zt, c[i]);
    }
    zt = a.renorm ? token_max<L>(zt) : 0.0f;
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
        if (i * L >= a.K) {
            c[i] = 0.0f;
            continue;
        }
        const float zc = c[i];
        float v;
        if (!a.sigmoid) v = a.renorm ? exp_neg(zc - zt) : exp_neg(zc - top) * recip;
        else {
            // all multiplied by e^-zt where every chosen logit is negative: their ratios stay where the scores themselves vanish
            const float e = exp_neg(-fabsf(zc));
            v = (zc >= 0.0f ? 1.0f : a.renorm && zt < 0.0f ? exp_neg(zc - zt) : e) / (1.0f + e);
        }
        c[i] = zc > -INFINITY ? v : 0.0f;
        total += c[i];
    }
    float by = a.scale;
    if (a.renorm) {
        total = token_sum<L>(total);
        by = total > 0.0f ? a.scale / total : 0.0f;
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
        const int j = sub + i * L;
        if (j < a.K) {
            const int e = at[i] < 0 ? ROUTE_NONE : at[i] & (ROUTE_FILL - 1);
            a.ids[(size_t)t * a.K + j] = e;
            a.w[(size_t)t * a.K + j] = c[i] * by;
            if (e >= 0) atomicAdd(&hist[e], 1);
        }
    }
}

// A token in doubt, by a wave
template <int N>
__device__ __forceinline__ void route_again(const route_args &a, int t, const float *bias, double *spare, int *hist)
{
    const float *row = a.logits + (size_t)t * a.E;
    float top, recip;
    const int at[1] = {route_exact<N>(a, row, bias, spare, &top, &recip)};
    route_write<64>(a, row, t, true, threadIdx.x & 63, at, top, recip, hist);
}

// Words of LDS that a wave needs: the worths of its tokens for their groups (four words of padding behind 32: groups of 32 in different banks) and then two
// words for each group, of which a token has as many as lanes at most; the lanes' lists and one more word each; one token's worths in double
static constexpr int route_worths(int L, int V) { return std::max((L * V + L * V / 8 + 3) & ~3, 2 * L); }
__device__ __forceinline__ int route_padded(int e) { return e + (e >> 5) * 4; }
static constexpr int route_lds(int L, int V) { return std::max(std::max(64 * (V + 1), 2 * L * V), 64 / L * route_worths(L, V)); }
// ... and with the picks of its tokens, all of a wave (pieces of 16 bytes)
__host__ __device__ static constexpr int route_words(int L, int V, int K) { return (route_lds(L, V) + 64 / L * 2 * (K + 2) + 3) & ~3; }

// WORTH: there is a bias or there are groups
template <int L, int V, bool WORTH>
__global__ __launch_bounds__(1024) void route_forward_kernel(const route_args a)
{
    constexpr int TW = 64 / L, EW = L * V, KL = 64 / L;  // tokens of a wave, experts, chosen ones of a lane
    constexpr int C = V < 4 ? V : 4;                     // a lane's experts lie in pieces of C: k is expert (k / C) L C + sub C + k % C
    constexpr uint32_t LOW = V - 1;                      // bits of a word that say which of a lane's experts it is
    static_assert((V & (V - 1)) == 0 && V * L <= ROUTE_MAX_E, "places of a lane's experts in whole bits");
    extern __shared__ __attribute__((aligned(16))) uint32_t spare_all[];
    __shared__ int again[ROUTE_TOKENS], n_again;         // tokens that are chosen for in double
    __shared__ int hist[EW];
    __shared__ __attribute__((aligned(16))) float bias[WORTH ? EW : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane & (L - 1), tok = lane / L;
    const int E = a.E, K = a.K, NT = blockDim.x;
    uint32_t *spare = spare_all + wave * route_words(L, V, K), *list = spare + lane;
    float *uw = (float *)spare + tok * route_worths(L, V);
    u32x2 *picks = (u32x2 *)(spare + route_lds(L, V)) + tok * (K + 2);  // the chosen words and the lanes that held them, and two behind them
    const bool softmax_row = !a.sigmoid && (WORTH || !a.renorm);
    for (int e = threadIdx.x; e < EW; e += NT) {
        hist[e] = 0;
        if (WORTH) bias[e] = a.bias != nullptr && e < E ? a.bias[e] : 0.0f;
    }
    if (threadIdx.x == 0) n_again = 0;
    __syncthreads();
    float span = 0.0f;  // the largest bias that scores, which are 1 at most, compete with: of 16 and more it switches its expert on or off
    if (WORTH && a.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < (EW + 63) / 64; ++k) {
            const float b = fabsf(bias[min(lane + 64 * k, EW - 1)]);
            span = b < 16.0f ? fmaxf(span, b) : span;
        }
        span = token_max<64>(span);
    }
    // What two worths u may differ by although they are equal, of twice the largest score and the larger bias of the two, in units of 2^-24.  Sigmoid: e^-z 2 +
    // 1.22 |z| of itself, a score by 0.8 of that at most (its slope is s (1 - s)), the addition 1, the reciprocal 2, the bias's rounding 1 + |b|: 5 + |b| each,
    // of 2 + |b| 8 in all.  Softmax: e^x 2.5 (|x| e^x is 0.37 at most), the bias's rounding s + |b|, in common the sum's V + 8 and the reciprocal's 1, whose
    // error the biases do not share: (V + 16) s + 2 |b| in all.  Sums of two, by which groups are told apart: twice that, and 8 (s + |b|) for the two additions
    // and for the bounds that each group is given.  Where |u| is below 14 the bias is at most `span`, else at most |u| + s: one that switches an expert off
    // says nothing about the others.
    const float unsure = a.sigmoid ? 0x1p-21f : (float)(V + 24) * 0x1p-25f;
    const int end = min(a.T, (int)(blockIdx.x + 1) * a.tokens);
    for (int t0 = blockIdx.x * a.tokens + wave * TW; t0 < end; t0 += NT / 64 * TW) {
        const int t = t0 + tok;
        const bool live = t < end;
        const float *rows = a.logits + (size_t)t0 * E;  // (the same for the wave: lanes' offsets are of 32 bits)
        const int at0 = live ? tok * E : 0;
        // (few rounds of this loop: what depends on the lane alone is not worth registers across them)
        int lane_first = sub * C;
        asm("" : "+v"(lane_first));
        auto expert = [&](int k) { return (k / C) * (L * C) + lane_first + k % C; };
        float z[V];
        if (a.vec && C == 4) {
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const float4 u = *(const float4 *)((const char *)rows + ((uint32_t)(at0 + min(expert(k), E - 4)) << 2));
                z[k] = u.x, z[(k + 1) % V] = u.y, z[(k + 2) % V] = u.z, z[(k + 3) % V] = u.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) z[k] = ld_at(rows, (uint32_t)(at0 + min(expert(k), E - 1)));
        }
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] = open_logit(z[k]);
        if (E < EW) {
#pragma unroll
            for (int k = 0; k < V; ++k) z[k] = expert(k) < E ? z[k] : -INFINITY;
        }
        // scores, where the choice or the weights need all of them
        float top = 0.0f, recip = 1.0f;
        if (softmax_row) {
            top = z[0];
#pragma unroll
            for (int k = 1; k < V; ++k) top = fmaxf(top, z[k]);
            top = fmaxf(token_max<L>(top), -FLT_MAX);  // (a token without open experts: every score 0)
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < V; ++k) s += exp_near(z[k] - top);
            s = token_sum<L>(s);
            recip = s > 0.0f ? 1.0f / s : 0.0f;
        }
        auto doubtful = [&](float u) { return fmaf(2.0f, recip, u < 14.0f ? span : fminf(u, FLT_MAX) + recip); };  // (sigmoid: scores up to 1)
        bool doubt = false;
        uint32_t word[V];
        if (!WORTH) {
#pragma unroll
            for (int k = 0; k < V; ++k) word[k] = ordered(z[k] + 0.0f);  // (both zeros the same)
        } else {
            float u[V];
#pragma unroll
            for (int k = 0; k < V; ++k) u[k] = 0.0f;
            if (a.bias != nullptr) {
#pragma unroll
                for (int k = 0; k < V; ++k) u[k] = bias[expert(k)];
            }
            if (a.sigmoid) {
#pragma unroll
                for (int k = 0; k < V; ++k) u[k] += sigmoid_near(z[k]);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) u[k] = fmaf(exp_near(z[k] - top), recip, u[k]);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) u[k] = or_closed(fmaf(z[k], 0.0f, u[k]));  // (-infinity times 0 is no number, others' nothing)
            if (a.bias != nullptr) {  // (no sum of a score and a bias is -0)
#pragma unroll
                for (int k = 0; k < V; ++k) word[k] = ordered(u[k]);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) word[k] = ordered(z[k] + 0.0f);
            }
            if (a.groups > 1) {
                wave_lds();  // (what the wave's last tokens left there has been read)
                const bool whole = C == 4 && (a.per_group & 3) == 0;  // a piece of four experts is one group's: its two best are enough
                float2 *ub = (float2 *)uw;
                if (whole) {
#pragma unroll
                    for (int k = 0; k + 3 < V; k += 4) {
                        const float m0 = fmaxf(u[k], u[k + 1]), n0 = fminf(u[k], u[k + 1]), m1 = fmaxf(u[k + 2], u[k + 3]), n1 = fminf(u[k + 2], u[k + 3]);
                        const int at = k / 4 * L + sub;
                        ub[at + (at >> 3)] = make_float2(fmaxf(m0, m1), fmaxf(fmaxf(n0, n1), fminf(m0, m1)));
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k) uw[route_padded(expert(k))] = u[k];
                }
                wave_lds();
                const int q = 1 << a.group_shift, g = sub >> a.group_shift, i = sub & (q - 1);
                float best = -INFINITY, second = -INFINITY;
                auto meet = [&](float b, float s) {
                    second = fmaxf(fmaxf(second, s), fminf(best, b));
                    best = fmaxf(best, b);
                };
                if (g < a.groups) {
                    if (whole) {
                        const int n = a.per_group >> 2;
                        for (int at = g * n + i; at < (g + 1) * n; at += q) {
                            const float2 b = ub[at + (at >> 3)];
                            meet(b.x, b.y);
                        }
                    } else {
                        for (int e = g * a.per_group + i; e < (g + 1) * a.per_group; e += q) meet(uw[route_padded(e)], -INFINITY);
                    }
                }
                // (after each step its lanes hold the same, so that a mirror is a neighbour)
                if (q > 1) meet(lane_of<0xB1>(best), lane_of<0xB1>(second));
                if (q > 2) meet(lane_of<0x4E>(best), lane_of<0x4E>(second));
                if (q > 4) meet(lane_of<0x141>(best), lane_of<0x141>(second));
                if (q > 8) meet(lane_of<0x140>(best), lane_of<0x140>(second));
                if (q > 16) meet(__shfl_xor(best, 16), __shfl_xor(second, 16));
                const bool two = a.group_best == 2 && second > -INFINITY;
                const float mine = two ? fmaxf(best + second, -FLT_MAX) : best;  // (below the lowest number: in doubt, but not closed)
                // what it may be at most and at least, of which every group has its own
                const float off = unsure * doubtful(two ? fmaxf(fabsf(best), fabsf(second)) : fabsf(best)), least = mine - off;
                wave_lds();
                if (i == 0) ((float2 *)uw)[g] = make_float2(mine, mine + off);
                wave_lds();
                int ahead = 0;
                bool near = false;
                for (int o0 = 0; o0 < a.groups; o0 += 4) {
                    const float4 o2[2] = {((const float4 *)uw)[o0 / 2], ((const float4 *)uw)[o0 / 2 + 1]};
                    const float o[4] = {o2[0].x, o2[0].z, o2[1].x, o2[1].z}, at_most[4] = {o2[0].y, o2[0].w, o2[1].y, o2[1].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool there = o0 + k < a.groups, in_front = there & ((o[k] > mine) | ((o[k] == mine) & (o0 + k < g)));
                        ahead += in_front ? 1 : 0;
                        near |= there & !in_front & (o0 + k != g) & (o[k] > -INFINITY) & !(least > at_most[k]);
                    }
                }
                doubt = g < a.groups && near && ahead == a.top_groups - 1;  // (the last group that stays, and one behind it)
                const unsigned long long stay = token_bits<L>(__ballot(i == 0 && g < a.groups && ahead < a.top_groups));
                if ((a.per_group & (C - 1)) == 0) {  // (a piece is one group's)
#pragma unroll
                    for (int k = 0; k < V; k += C) {
                        const bool in = (stay >> ((((uint32_t)expert(k) * (uint32_t)a.group_magic >> 20) << a.group_shift) & (L - 1))) & 1;
#pragma unroll
                        for (int n = 0; n < C; ++n) word[k + n] = in ? word[k + n] : 0u;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        word[k] = (stay >> ((((uint32_t)expert(k) * (uint32_t)a.group_magic >> 20) << a.group_shift) & (L - 1))) & 1 ? word[k] : 0u;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) word[k] = (word[k] & ~LOW) | (LOW - k);
        // descending (Batcher's odd-even merges)
#pragma unroll
        for (int p = 1; p < V; p *= 2)
#pragma unroll
            for (int k = p; k >= 1; k /= 2)
#pragma unroll
                for (int j = k % p; j <= V - 1 - k; j += 2 * k)
#pragma unroll
                    for (int i = 0; i < k; ++i)
                        if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                            const uint32_t x = word[i + j], y = word[i + j + k];
                            word[i + j] = max(x, y);
                            word[i + j + k] = min(x, y);
                        }
        wave_lds();
        uint32_t first = word[0], next = V > 1 ? word[1 % V] : 0u;
#pragma unroll
        for (int k = 2; k < V; ++k) list[64 * k] = word[k];
        list[64 * V] = 0u;
        int taken = 0;
        for (int j = 0; j < K + 2; ++j) {  // (two more: what is left has to be told from what is chosen)
            const uint32_t b = token_max<L>(first);
            if (__builtin_amdgcn_inverse_ballot_w64(first_lanes<L>(__ballot(first == b)))) {  // (two lanes that hold it: their turn one by one)
                picks[j] = u32x2{b, (uint32_t)sub};
                const bool open = b >= ROUTE_OPEN;
                taken += open ? 1 : 0;
                first = open ? next : b;
                next = list[64 * min(taken + 1, V)];
            }
        }
        wave_lds();
        // The chosen and, next to each, the one behind it: lane sub has the places sub, sub + L, ...
        int at[KL];
        bool near = false;
        auto apart = [&](uint32_t b, uint32_t o) {  // b >= o
            if (!WORTH || a.bias == nullptr) return o < ROUTE_OPEN || (b & ~LOW) != (o & ~LOW);
            const float x = of_ordered(b & ~LOW), y = of_ordered(o & ~LOW);
            return o < ROUTE_OPEN || x - y > (unsure + (float)V * 0x1p-23f) * doubtful(fmaxf(fabsf(x), fabsf(y)));  // (the words' last bits besides)
        };
        auto expert_of = [&](u32x2 p) {
            const int k = (int)(LOW - (p[0] & LOW));
            return p[0] >= ROUTE_OPEN ? (k / C) * (L * C) + (int)p[1] * C + k % C : ROUTE_NONE;
        };
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const int j = sub + i * L;
            at[i] = ROUTE_NONE;
            if (i * L >= K) continue;
            if (j < K) {
                const u32x2 p = picks[j];
                at[i] = expert_of(p);
                near |= at[i] >= 0 && !apart(p[0], picks[j + 1][0]);
                if (at[i] < 0 && a.fill) doubt = true;
            }
        }
        if (__ballot(near)) {
            // They and the two behind them once more, a lane each, without a bias as they are, else in double.  Where the last of these is near to the last
            // chosen there may be more.
            if (K + 2 > L) doubt |= near;
            else {
                const u32x2 last = picks[K - 1];
                doubt |= last[0] >= ROUTE_OPEN && !apart(last[0], picks[K + 1][0]);
                const int e = sub < K + 2 ? expert_of(picks[sub]) : ROUTE_NONE;
                const float ze = e >= 0 ? open_logit(ld_at(rows, (uint32_t)(at0 + e))) : -INFINITY;
                int ahead = 0;
                if (WORTH && a.bias != nullptr) {
                    double v = -INFINITY, sum = 0.0;
                    if (!a.sigmoid) {
                        float zo[V];
#pragma unroll
                        for (int k = 0; k < V; ++k) zo[k] = ld_at(rows, (uint32_t)(at0 + min(expert(k), E - 1)));
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            zo[k] = open_logit(expert(k) < E ? zo[k] : -INFINITY);
                            sum += zo[k] == -INFINITY ? 0.0 : exp((double)zo[k] - (double)top);
                            __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
                        }
                        for (int n = L / 2; n > 0; n >>= 1) sum += __shfl_xor(sum, n);
                    }
                    v = exp(a.sigmoid ? -(double)ze : (double)ze - (double)top);
                    v = (a.sigmoid ? 1.0 / (1.0 + v) : v / sum) + (e >= 0 ? (double)bias[e] : 0.0);
                    if (e < 0 || !(v == v)) v = -INFINITY;
                    for (int o = 0; o < K + 2; ++o) {
                        const double x = __shfl(v, o, L);
                        const int y = __shfl(e, o, L);
                        ahead += (x > v) | ((x == v) & (y < e)) ? 1 : 0;
                    }
                } else {
                    for (int o = 0; o < K + 2; ++o) {
                        const float x = __shfl(ze, o, L);
                        const int y = __shfl(e, o, L);
                        ahead += (x > ze) | ((x == ze) & (y < e)) ? 1 : 0;
                    }
                }
                wave_lds();
                if (e >= 0) picks[ahead] = u32x2{(uint32_t)e, 0u};
                wave_lds();
                if (at[0] >= 0) at[0] = (int)picks[sub][0];
            }
        }
        const unsigned long long doubts = token_bits<L>(__ballot(doubt));
        if (doubts && live && sub == 0) again[atomicAdd(&n_again, 1)] = t;
        route_write<L>(a, rows + at0, t, live && !doubts, sub, at, top, recip, hist);
        wave_lds();
    }
    __syncthreads();
    // in double, a wave each
    for (int i = wave; i < n_again; i += NT / 64) route_again<(L * V + 63) / 64>(a, again[i], WORTH && a.bias != nullptr ? bias : nullptr, (double *)spare, hist);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += NT) a.part[(size_t)blockIdx.x * E + e] = hist[e];
}

// counts = sums of n rows of part [n][E]: a workgroup takes 16 experts, 64 rows at a time (512 x 256: 3.8 us, 128 x 128: 2.5; one memory latency
// and the launch)
__global__ __launch_bounds__(1024) void route_counts_kernel(const int32_t *__restrict__ part, int n, int E, int32_t *__restrict__ counts)
{
    __shared__ int red[16][16];
    const int cc = threadIdx.x & 15, k = threadIdx.x >> 4, e = blockIdx.x * 16 + cc;
    int s = 0;
    for (int i0 = k; i0 < n && e < E; i0 += 64 * 8) {  // eight rows asked for together
        int v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i0 + 64 * j < n ? part[(size_t)(i0 + 64 * j) * E + e] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if ((threadIdx.x & 48) == 0) red[threadIdx.x >> 6][cc] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || e >= E) return;
    s = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += red[w][cc];
    counts[e] = s;
}

struct route_back_args {
    const float *logits;
    int T, E, K, sigmoid, renorm, vec;
    float scale;
    const int32_t *ids;
    const float *w, *dw;
    float *dlogits;
};
// L lanes a token; a lane takes the chosen j = sub, sub + L, ... and, as in the forward pass, V experts in pieces of C.  The gradients of the chosen meet
// the row in LDS, so that every element of dlogits is written once, 16 bytes a lane.  Bound: bytes (65536 x 256, all scores: 33 us, 4.1 TB/s; 16384 x 128:
// 5.6 us, a launch and 8 MB).
template <int L, int V>
__global__ __launch_bounds__(256) void route_backward_kernel(const route_back_args a)
{
    constexpr int TW = 64 / L, KL = 64 / L, C = V < 4 ? V : 4;
    __shared__ __attribute__((aligned(16))) float dzs[4][TW][L * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (L - 1), tok = lane / L;
    const int E = a.E, K = a.K, t = (blockIdx.x * 4 + wave) * TW + tok;
    const bool live = t < a.T;
    float *dz = dzs[wave][tok];
    const size_t row = (size_t)t * E, pick = (size_t)t * K;
    auto expert = [&](int k) { return (k / C) * (L * C) + sub * C + k % C; };
    int id[KL];
    float w[KL], g[KL], z[V];
    const bool all = !a.sigmoid && !a.renorm;  // every score has a part in the gradient
#pragma unroll
    for (int i = 0; i < KL; ++i) {
        const int j = sub + i * L;
        id[i] = ROUTE_NONE;
        w[i] = g[i] = 0.0f;
        if (live && j < K) {
            id[i] = a.ids[pick + j];
            w[i] = a.w[pick + j];
            g[i] = a.dw[pick + j];
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = all && live && expert(k) < E ? open_logit(a.logits[row + expert(k)]) : -INFINITY;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
        if (id[i] < 0 || id[i] >= E) w[i] = 0.0f;
        if (w[i] == 0.0f) id[i] = ROUTE_NONE, g[i] = 0.0f;
    }
    float rest[KL];  // 1 - s
#pragma unroll
    for (int i = 0; i < KL; ++i) rest[i] = a.sigmoid && id[i] >= 0 ? sigmoid(-open_logit(a.logits[row + id[i]])) : 1.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) dz[expert(k)] = 0.0f;
    wave_lds();
    float dot = 0.0f;
    if (a.renorm) {
        // by differences: what all chosen have in common has no part in the gradient
        float d[KL];
#pragma unroll
        for (int i = 0; i < KL; ++i) d[i] = 0.0f;
#pragma unroll
        for (int p = 0; p < KL; ++p)
            for (int k = 0; k < min(L, K - p * L); ++k) {
                const float wk = __shfl(w[p], k, L), gk = __shfl(g[p], k, L);
#pragma unroll
                for (int i = 0; i < KL; ++i) d[i] = fmaf(wk, g[i] - gk, d[i]);
            }
#pragma unroll
        for (int i = 0; i < KL; ++i) g[i] = d[i] / a.scale;
    } else if (all) {
#pragma unroll
        for (int i = 0; i < KL; ++i) dot = fmaf(w[i], g[i], dot);
        dot = token_sum<L>(dot);
    }
#pragma unroll
    for (int i = 0; i < KL; ++i)  // (a token's ids differ: one addition a place, of which no order shows)
        if (id[i] >= 0) atomicAdd(&dz[id[i]], w[i] * g[i] * rest[i]);
    wave_lds();
    float top = 0.0f, recip = 0.0f;
    if (all) {
        top = z[0];
#pragma unroll
        for (int k = 1; k < V; ++k) top = fmaxf(top, z[k]);
        top = fmaxf(token_max<L>(top), -FLT_MAX);
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) s += exp_neg(z[k] - top);
        s = token_sum<L>(s);
        recip = s > 0.0f ? 1.0f / s : 0.0f;
    }
    if (!live) return;
    float o[V];
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = dz[expert(k)];
    if (all) {
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = fmaf(-exp_neg(z[k] - top) * recip, dot, o[k]);
    }
#pragma unroll
    for (int k = 0; k < V; k += C) {
        float *p = a.dlogits + row + expert(k);
        if (C == 4 && a.vec) {
            if (expert(k) < E) *(float4 *)p = make_float4(o[k], o[(k + 1) % V], o[(k + 2) % V], o[(k + 3) % V]);
        } else {
#pragma unroll
            for (int n = 0; n < C; ++n)
                if (expert(k) + n < E) p[n] = o[k + n];
        }
    }
}

// bias[e] += rate where an expert was chosen less often than the mean, -= rate where more often
__global__ __launch_bounds__(256) void route_balance_kernel(const int32_t *__restrict__ counts, int E, float rate, float *__restrict__ bias)
{
    __shared__ long long red[256];
    long long s = 0;
    for (int e = threadIdx.x; e < E; e += 256) s += counts[e];
    red[threadIdx.x] = s;
    for (int n = 128; n > 0; n >>= 1) {
        __syncthreads();
        if (threadIdx.x < n) red[threadIdx.x] += red[threadIdx.x + n];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 256) {
        const long long over = (long long)counts[e] * E - red[0];
        if (over != 0) bias[e] += over < 0 ? rate : -rate;
    }
}

// How a batch is cut.  Few lanes a token do the least work for it (16; above 256 experts 32: 65536 x 512, softmax, 41 us, with a wave a token 78), a wave ends
// soonest: sixteen tokens a compute unit and fewer have one each (E = 256, sigmoid, 8 groups: 4096 tokens 13.0 us, with 16 lanes 13.8; 8192 tokens 17.4 and
// 14.0; at 64 experts and fewer half of it is idle).  What one workgroup takes at once it does alone, without a second launch for the counts (64
// tokens of 128 experts 5.4 us a call, in several workgroups 6.3; 64 of 256 experts, two rounds of its waves, 7.9 and 6.4).  Groups: one lane for each at
// least.
struct route_cut {
    int lanes, threads, tokens;  // of a token; of a workgroup
};
static int route_per_lane(int E, int lanes)
{
    if (lanes == 64) return E <= 64 ? 1 : E <= 128 ? 2 : E <= 256 ? 4 : 8;
    return lanes == 32 ? 16 : E <= 16 ? 1 : E <= 64 ? 4 : E <= 128 ? 8 : 16;
}
static int route_wave_words(int E, int K, int lanes) { return route_words(lanes, route_per_lane(E, lanes), K); }
static int route_lanes(const omega_route_config &c, bool few)
{
    const int least = c.E <= 256 ? 16 : 32;
    return c.groups > least || (few && c.E > 64) ? 64 : least;
}
static route_cut route_cut_of(const omega_ctx *ctx, const omega_route_config &c, int T)
{
    const bool must = c.groups > 16 || c.E > 256;
    if (!must) {
        // one workgroup of sixteen waves, of eight where their LDS would not be within 64 KB, beside the workgroup's own: its tokens at once
        const int lanes = T <= 16 ? 64 : 16, threads = 16 * 4 * route_wave_words(c.E, c.K, lanes) <= 56 << 10 ? 1024 : 512;
        if (T <= threads / lanes) return {lanes, threads, 64};
    }
    const int lanes = route_lanes(c, T <= 16 * ctx->num_cus);
    const int round = 8 * (64 / lanes);  // tokens that the waves of a workgroup take at once
    return {lanes, 512, std::min(std::max(1, ceil_div(ceil_div(T, 2 * ctx->num_cus), round)) * round, ROUTE_TOKENS)};
}

static route_args route_arguments(const omega_route_config &c, const float *logits, int T, const float *bias, int tokens, int L, int32_t *ids, float *w)
{
    const int E = c.E, vec = E % 4 == 0 && (uintptr_t)logits % 16 == 0;
    int shift = 0;  // lanes of a group: as many as the next power of two of groups leaves
    while (c.groups > 1 && (2 << shift) * c.groups <= L) ++shift;
    return {logits, bias, T, E, c.K, c.score == OMEGA_ROUTE_SIGMOID, c.renorm, c.groups, c.top_groups, c.group_best, E / c.groups, (1 << 20) / (E / c.groups) + 1,
            shift, c.scale, tokens, 0, vec, ids, w, nullptr};
}
static hipError_t route_launch(const route_args &a, int lanes, int threads, hipStream_t s)
{
    const int E = a.E, T = a.T, tokens = a.tokens;
    const bool worth = a.bias != nullptr || a.groups > 1;
#define ROUTE_FORWARD(LL, V)                                                                                                                     \
    do {                                                                                                                                         \
        const dim3 grid(ceil_div(T, tokens));                                                                                                    \
        const size_t lds = (size_t)threads / 64 * route_wave_words(E, a.K, lanes) * sizeof(float);                                                \
        if (worth) hipLaunchKernelGGL((route_forward_kernel<LL, V, true>), grid, dim3(threads), lds, s, a);                                      \
        else hipLaunchKernelGGL((route_forward_kernel<LL, V, false>), grid, dim3(threads), lds, s, a);                                           \
    } while (0)
    if (lanes == 64) {
        if (E <= 64) ROUTE_FORWARD(64, 1);
        else if (E <= 128) ROUTE_FORWARD(64, 2);
        else if (E <= 256) ROUTE_FORWARD(64, 4);
        else ROUTE_FORWARD(64, 8);
    } else if (lanes == 32) {
        ROUTE_FORWARD(32, 16);
    } else {
        if (E <= 16) ROUTE_FORWARD(16, 1);
        else if (E <= 64) ROUTE_FORWARD(16, 4);
        else if (E <= 128) ROUTE_FORWARD(16, 8);
        else ROUTE_FORWARD(16, 16);
    }
#undef ROUTE_FORWARD
    return hipGetLastError();
}

size_t route_workspace(const omega_ctx *ctx, const omega_route_config &c, int T) { return (size_t)std::max(1, ceil_div(T, route_cut_of(ctx, c, T).tokens)) * c.E * sizeof(int32_t); }

hipError_t launch_route_forward(const omega_ctx *ctx, const omega_route_config &c, const float *logits, int T, const float *bias, int32_t *ids, float *w,
                                int32_t *counts, void *ws, hipStream_t s)
{
    int n = 0;
    if (T > 0) {
        const route_cut cut = route_cut_of(ctx, c, T);
        n = ceil_div(T, cut.tokens);
        route_args a = route_arguments(c, logits, T, bias, cut.tokens, cut.lanes, ids, w);
        a.part = n == 1 && counts ? counts : (int32_t *)ws;
        const hipError_t e = route_launch(a, cut.lanes, cut.threads, s);
        if (e != hipSuccess || n == 1 || !counts) return e;
    }
    hipLaunchKernelGGL(route_counts_kernel, dim3(ceil_div(c.E, 16)), dim3(1024), 0, s, (const int32_t *)ws, n, c.E, counts);
    return hipGetLastError();
}

// (workgroups of as many tokens as a row of the layer's histogram has: sixteen lanes a token are one round of four waves)
hipError_t launch_route_layer(const omega_route_config &c, const float *logits, int T, const float *bias, int tokens, int32_t *ids, float *w, int32_t *tile_counts,
                              hipStream_t s)
{
    const int lanes = route_lanes(c, false);
    route_args a = route_arguments(c, logits, T, bias, tokens, lanes, ids, w);
    a.fill = 1;
    a.part = tile_counts;
    return route_launch(a, lanes, 256, s);
}

#define ROUTE_RUN(K, grid, s, ...)                                                                       \
    do {                                                                                                 \
        if (E <= 16) hipLaunchKernelGGL((K<16, 1>), dim3(grid), dim3(256), 0, s, __VA_ARGS__);            \
        else if (E <= 64) hipLaunchKernelGGL((K<16, 4>), dim3(grid), dim3(256), 0, s, __VA_ARGS__);       \
        else if (E <= 128) hipLaunchKernelGGL((K<16, 8>), dim3(grid), dim3(256), 0, s, __VA_ARGS__);      \
        else if (E <= 256) hipLaunchKernelGGL((K<16, 16>), dim3(grid), dim3(256), 0, s, __VA_ARGS__);     \
        else hipLaunchKernelGGL((K<64, 8>), dim3(grid), dim3(256), 0, s, __VA_ARGS__);                    \
    } while (0)

hipError_t launch_route_backward(const omega_route_config &c, const float *logits, int T, const int32_t *ids, const float *w, const float *dw, float *dlogits,
                                 hipStream_t s)
{
    const int E = c.E, round = E <= 256 ? 16 : 4, most = round << 22;  // (a launch holds fewer than 2^32 lanes: tokens in several)
    for (int t = 0; t < T; t += most) {
        const int n = std::min(most, T - t);
        const size_t row = (size_t)t * E, pick = (size_t)t * c.K;
        const route_back_args a = {logits ? logits + row : nullptr, n, E, c.K, c.score == OMEGA_ROUTE_SIGMOID, c.renorm, E % 4 == 0 && (uintptr_t)dlogits % 16 == 0, c.scale, ids + pick, w + pick, dw + pick, dlogits + row};
        ROUTE_RUN(route_backward_kernel, ceil_div(n, round), s, a);
    }
    return hipGetLastError();
}

hipError_t launch_route_balance(const int32_t *counts, int E, float rate, float *bias, hipStream_t s)
{
    hipLaunchKernelGGL(route_balance_kernel, dim3(1), dim3(256), 0, s, counts, E, rate, bias);
    return hipGetLastError();
}
