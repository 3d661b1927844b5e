// lg_sample.h — tokens drawn from logits rows by given random numbers: temperature, top-k, top-p, min-p.
//
// The definition is in whole numbers, so that no sum depends on an order and any split of a row gives the same token:
//   M = the row's largest logit (NaN counts as -inf), w_i = 2^44 exp((l_i - M) / T) rounded to a whole number; every token with w_i > 0 is in question
//   (less than 2^-45 of the likeliest token's probability is none).
//   Order: larger logit first, of equal ones the lower index.  top_k keeps the first k; top_p of those the shortest prefix whose sum reaches
//   ceil(p W), W their sum; min_p of those w_i >= min_p 2^44.  All three are prefixes of the order, so what is kept is a border: a logit, and how many of
//   the tokens that have exactly it.
//   S = sum of the kept, r = min(floor(u S), S - 1); the token is the first in index order whose running sum of kept weights passes r.
// Rows of up to 2^19 tokens: a sum is at most 2^63.
//
// A row is read by many workgroups and finished by one, in four launches (one for rows of at most LG_SAMPLE_WHOLE tokens):
//   lg_k_sample_max     the largest logit of every group of 256
//   lg_k_sample_bins    rows whose border is to be found: 2048 bins of equal width from the largest logit down, how many tokens and about what sum each holds
//   lg_k_sample_sums    the exact sum of every group above the bins that can hold the border, and the tokens in those (candidates)
//   lg_k_sample_finish  one workgroup a row: the border among the candidates, the draw by the groups' sums and the tokens of one group.
//                       Rows of a small top-k come here at once: the k-th largest of the groups' largest logits is at most the k-th largest logit, so
//                       the tokens not below it, few more than k, are the candidates.
// What the second and third find only narrows down: the border is taken from whole-number sums, and where the candidates turn out not to hold
// it (too many, as with a top-p near 1; a bin's sum estimated too far off) lg_sample_row finds it from the row alone, as it does where f32 does not hold the logits' distances.
//
// A row is 4 bytes a token and is read once (a small top-k, greedy), twice (no top-k and no top-p) or three times, from the second time on mostly from caches: 64 rows of 262144
// have 67 MB, which a bare read takes 11.8 us for.  Launches of them with rows of all kinds: 14.6 us (4.6 TB/s), 10.8, 22.3 and 19.9 us.  Few rows are bound by
// the chain of launches, loads and barriers: one with top-k 64 and top-p 0.95 3.8, 1.8, 1.7 and 10.2 us (the second and third have nothing to do), 5 with top-p alone 4.7, 7.3,
// 11.1 and 9.3.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "lg_block.h"

#define LG_SAMPLE_WG     1024
#define LG_SAMPLE_VOCAB  (1 << 19)
#define LG_SAMPLE_ONE    17592186044416.0        // 2^44

struct SampleRow { float temperature; int32_t top_k; float top_p, min_p; };     // struct lg_hip_sampling
struct SampleArgs {
    const float *logits; long long stride;
    const SampleRow *params;
    const float *u;
    int32_t *tok; float *prob; int32_t *kept;   // the last two may be null
    int n_vocab, slices;                // workgroups of lg_k_sample_sums to a row
};

// A number that is larger for a larger logit; NaN and -inf give 0x007FFFFF, -0 what +0 gives
__device__ __forceinline__ uint32_t lg_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    if (l != l) return 0x007FFFFFu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lg_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// 2^(j / 32)
__device__ const double lg_exp2_32nds[32] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002,
};
// What a row's weights need: M, 32 / (T ln 2) (0 for a T of infinity), the table in LDS
struct Weigh { double top, inv; const double *tab; };
// 2^44 e^((l - top) / T), rounded.  With y = 32 (l - top) / (T ln 2) = n + r, n whole, it is 2^(44 + n / 32) times the power series of 2^(r / 32) (|r| <= 1/2: what
// comes after r^5 is 2e-15).  Adding 1.5 2^52 leaves n in the low bits, adding 2^52 the result.  Beyond LG_SAMPLE_REACH it is 0.  (The series of e^r to r^12
// without the table would be 25 operations in place of 14.)
#define LG_SAMPLE_REACH   31.5
__device__ __forceinline__ lg_u64 lg_weight_at(const Weigh &w, double y) {          // y of -LG_SAMPLE_REACH 32 / ln 2 .. 0
    const double t = y + 6755399441055744.0, r = y - (t - 6755399441055744.0);
    const int n = (int)(uint32_t)(lg_u64)__double_as_longlong(t);
    double p = 3.9737099845494161e-11;
    p = __builtin_fma(p, r, 9.172562701824643e-09);
    p = __builtin_fma(p, r, 1.6938509724371821e-06);
    p = __builtin_fma(p, r, 0.0002345961982022468);
    p = __builtin_fma(p, r, 0.02166084939249829);
    p = __builtin_fma(p, r, 1.0);
    const double scale = __longlong_as_double(__double_as_longlong(w.tab[n & 31]) + ((long long)(44 + (n >> 5)) << 52));
    return (lg_u64)__double_as_longlong(__builtin_fma(p, scale, 4503599627370496.0)) & 0x000FFFFFFFFFFFFFull;
}
__device__ __forceinline__ lg_u64 lg_weigh(const Weigh &w, float l) {
    const double y = l == (float)w.top ? 0.0 : ((double)l - w.top) * w.inv;
    return y >= -LG_SAMPLE_REACH * 46.166241308446828384 && l != -INFINITY ? lg_weight_at(w, y) : 0;
}
// The same for a finite maximum and a logit whose exponent is known to be above LG_SAMPLE_FLOOR (in base 2, to an f32's accuracy; a weight is 0 below -45)
#define LG_SAMPLE_FLOOR   -45.2f
__device__ __forceinline__ lg_u64 lg_weight(const Weigh &w, float l) { return lg_weight_at(w, ((double)l - w.top) * w.inv); }
__device__ __forceinline__ Weigh lg_weigher(float top, float T, const double *tab) { return { (double)top, T > 0 ? 46.166241308446828384 / (double)T : 0.0, tab }; }
// The table on its way: asked for first, stored once the kernel's other loads are asked for (the caller's next barrier is the table's)
__device__ __forceinline__ double lg_table_entry() { return lg_exp2_32nds[threadIdx.x & 31]; }
__device__ __forceinline__ void lg_table_store(double *tab, double entry) { if (threadIdx.x < 32) tab[threadIdx.x] = entry; }

// One workgroup, one row: the border by digits of the key (4 passes of 8 bits each for top-k and top-p), then the draw.
struct SampleLds { lg_u64 bin[256]; lg_u64 part[LG_SAMPLE_WG / 64]; uint32_t key; int idx; lg_u64 rest; };    // (tab: the caller's)

// The key at which a running sum from the largest key down reaches `want` (1..sum of all), among the tokens in question with keys >= low (of key `low`
// itself the first `ties` count); *before = the sum of the tokens with larger keys.  BY_COUNT: every token counts 1, else its weight.
template <bool BY_COUNT>
__device__ __forceinline__ uint32_t lg_border(const SampleArgs &a, const float *row, const Weigh &wg, uint32_t low, int ties, lg_u64 want, lg_u64 *before, SampleLds &s) {
    uint32_t prefix = 0, mask = 0;
    lg_u64 above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += LG_SAMPLE_WG) s.bin[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < a.n_vocab; i += LG_SAMPLE_WG) {
            const uint32_t k = lg_key(row[i]);
            if (k <= low || (k & mask) != prefix) continue;
            const lg_u64 w = lg_weigh(wg, row[i]);
            if (w) atomicAdd(&s.bin[k >> shift & 255], BY_COUNT ? 1ull : w);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            if (low && (low & mask) == prefix) s.bin[low >> shift & 255] += (lg_u64)ties * (BY_COUNT ? 1ull : lg_weigh(wg, lg_unkey(low)));
            int b = 255;
            lg_u64 run = above;
            for (; b > 0 && run + s.bin[b] < want; --b) run += s.bin[b];
            s.key = prefix | (uint32_t)b << shift;
            s.rest = run;
        }
        __syncthreads();
        prefix = s.key; above = s.rest;
        mask |= 255u << shift;
        __syncthreads();
    }
    *before = above;
    return prefix;
}

__device__ __forceinline__ void lg_sample_row(const SampleArgs &a, int r, const SampleRow &p, const double *tab, SampleLds &s) {
    const float *row = a.logits + r * a.stride;
    const int n = a.n_vocab, t = threadIdx.x;
    // the largest logit, and the first token that has it
    uint32_t key = 0; int at = n;
    for (int i = t; i < n; i += LG_SAMPLE_WG) { const uint32_t k = lg_key(row[i]); if (k > key) { key = k; at = i; } }
    if (t == 0) { s.key = 0; s.idx = n; }
    __syncthreads();
    atomicMax(&s.key, key);
    __syncthreads();
    if (key == s.key) atomicMin(&s.idx, at);
    __syncthreads();
    const uint32_t best = s.key;
    const int best_at = s.idx;
    __syncthreads();
    if (best == 0x007FFFFFu || !(p.temperature > 0)) {
        if (t == 0) {
            const bool none = best == 0x007FFFFFu;
            a.tok[r] = none ? -1 : best_at;
            if (a.prob) a.prob[r] = none ? 0.0f : 1.0f;
            if (a.kept) a.kept[r] = none ? 0 : 1;
        }
        return;
    }
    const Weigh wg = lg_weigher(lg_unkey(best), p.temperature, tab);
    uint32_t cut = 0; int ties = 0;                 // kept: keys > cut, and the first `ties` of those with it
    lg_u64 W = 0; unsigned count = 0;
    for (int i = t; i < n; i += LG_SAMPLE_WG) { const lg_u64 w = lg_weigh(wg, row[i]); W += w; count += w != 0; }
    W = lg_block_sum<LG_SAMPLE_WG>(W, s.part);
    count = (unsigned)lg_block_sum<LG_SAMPLE_WG>((lg_u64)count, s.part);
    if (p.top_k > 0 && (unsigned)p.top_k < count) {
        lg_u64 before;
        cut = lg_border<true>(a, row, wg, 0, 0, (lg_u64)p.top_k, &before, s);
        ties = (int)(p.top_k - before);
        lg_u64 sum = 0;
        for (int i = t; i < n; i += LG_SAMPLE_WG) if (lg_key(row[i]) > cut) sum += lg_weigh(wg, row[i]);
        W = lg_block_sum<LG_SAMPLE_WG>(sum, s.part) + (lg_u64)ties * lg_weigh(wg, lg_unkey(cut));
    }
    if (p.top_p < 1) {
        const double want_d = __builtin_ceil((double)p.top_p * (double)W);
        const lg_u64 want = want_d >= 1 ? (lg_u64)want_d : 1;
        lg_u64 before;
        const uint32_t c2 = lg_border<false>(a, row, wg, cut, ties, want < W ? want : W, &before, s);
        const lg_u64 w = lg_weigh(wg, lg_unkey(c2));
        ties = (int)((want - before + w - 1) / w);
        cut = c2;
    }
    // min-p: a whole number or more
    lg_u64 least = 1;
    if (p.min_p > 0) { const double m = __builtin_ceil((double)p.min_p * LG_SAMPLE_ONE); least = m >= 1 ? m < LG_SAMPLE_ONE ? (lg_u64)m : (lg_u64)LG_SAMPLE_ONE : 1; }
    const lg_u64 wcut = cut ? lg_weigh(wg, lg_unkey(cut)) : 0;
    if (wcut < least) ties = 0;
    lg_u64 S = 0; count = 0;
    for (int i = t; i < n; i += LG_SAMPLE_WG) if (lg_key(row[i]) > cut) { const lg_u64 w = lg_weigh(wg, row[i]); if (w >= least) { S += w; ++count; } }
    S = lg_block_sum<LG_SAMPLE_WG>(S, s.part) + (lg_u64)ties * wcut;
    count = (unsigned)lg_block_sum<LG_SAMPLE_WG>((lg_u64)count, s.part) + ties;
    const float u = a.u[r];
    lg_u64 target = u > 0 ? (lg_u64)__builtin_floor((u < 1 ? (double)u : 1.0) * (double)S) : 0;
    if (S && target > S - 1) target = S - 1;
    if (t == 0) { s.idx = -1; }
    // the draw: workgroup-wide pieces of the row in index order
    lg_u64 run = 0; int tied = 0;
    for (int i0 = 0; i0 < n && run <= target; i0 += LG_SAMPLE_WG) {
        const int i = i0 + t;
        const uint32_t k = i < n ? lg_key(row[i]) : 0;
        lg_u64 w = k >= cut && i < n ? lg_weigh(wg, row[i]) : 0;
        if (w < least) w = 0;
        lg_u64 all, all_ties = 0;
        if (cut) { const int mine = k == cut, rank = tied + (int)lg_block_run<LG_SAMPLE_WG>((lg_u64)mine, s.part, &all_ties) - mine; if (mine && rank >= ties) w = 0; }
        const lg_u64 upto = run + lg_block_run<LG_SAMPLE_WG>(w, s.part, &all);
        if (w && upto > target && upto - w <= target) { s.idx = i; s.rest = w; }
        run += all; tied += (int)all_ties;
    }
    __syncthreads();
    if (t == 0) {
        a.tok[r] = s.idx;
        if (a.prob) a.prob[r] = s.idx < 0 ? 0.0f : (float)((double)s.rest / (double)S);
        if (a.kept) a.kept[r] = (int)count;
    }
}


// ---- many workgroups to a row ----------------------------------------------------------------------------------------
#define LG_SAMPLE_GROUP   256                    // tokens of a group: a wavefront's load of 4 each
#define LG_SAMPLE_GROUPS  (LG_SAMPLE_VOCAB / LG_SAMPLE_GROUP)
#define LG_SAMPLE_MAX_WG  256                    // lg_k_sample_max: 16 groups to a workgroup
#define LG_SAMPLE_BINS    2048                   // (half as many are 3% faster and leave twice the candidates)
#define LG_SAMPLE_CAND    4096                   // candidates that a row may have
#define LG_SAMPLE_WHOLE   8192                   // tokens of a row that one workgroup takes by itself: 8 to a thread (16 do not fit its registers)
#define LG_SAMPLE_SMALL_K 400                    // top-k up to which, and up to half as many as there are groups, the groups' maxima bound the candidates well: with
                                                 // 1024 groups the tokens not below the k-th largest maximum are 1.15 k at k = 256 and 1.27 k at 400 where large
                                                 // logits lie anywhere in the row.  One row of 262144 by maxima and by bins: top-k 200 22 and 32 us, 400 29 and 33,
                                                 // 512 (more than LG_SAMPLE_LIST candidates) 37 and 32
#define LG_SAMPLE_SLACK   2048                   // the estimated sum of a row's bins is trusted to 1 / 2048: four times what the comment at lg_k_sample_bins allows, a bound for
                                                 // half a unit of each of 2^19 tokens.  Of a bell's tail that share is thousands of tokens: near a top-p of 1 there are more
                                                 // than LG_SAMPLE_CAND of them, and the row is taken alone.  One row of 262144, normal logits of a spread of 3 with some
                                                 // higher ones, T 1: top-p 0.99 32 us, from 0.995 on 780; of 128000 0.995 33, 0.999 404; of 60000 0.995 31, 0.999 222

// Tokens whose largest logit lg_k_sample_max keeps: a group's, a quarter's where these are no more than LG_SAMPLE_GROUPS (a small top-k is to be half of their number
// at most, and its candidates lie in fewer tokens: a row of 32000, top-k 64, 31.1 -> 17.4 us; of 128000, top-k 200, 22.5 -> 18.2)
__host__ __device__ constexpr int lg_top_shift(int n_vocab) { return n_vocab <= LG_SAMPLE_GROUPS * 64 ? 6 : 8; }
struct SampleWork {                     // per row, in working memory
    uint32_t *gmax;                     // [tops] keys
    uint32_t *smin;                     // [workgroups of lg_k_sample_max] ~key of the smallest logit above -inf, 0: none
    lg_u64 *mass; uint32_t *count;      // [LG_SAMPLE_BINS]
    lg_u64 *gsum;                       // [groups]
    lg_u64 *part;                       // [slices][3]: sum above the candidates, sum that top-p goes by (without the candidates), tokens kept above them
    uint32_t *ncand;                    // candidates; behind it, from word 4 on, the row's SampleRange, from word 8 its largest key and ~key of its smallest logit
    lg_u64 *cand;                       // [LG_SAMPLE_CAND] ~key << 32 | index
};
struct SampleGeo { int groups, tops, maxes, slices; size_t gmax, smin, mass, count, gsum, part, ncand, cand, row; };
__host__ __device__ inline size_t lg_up64(size_t n) { return (n + 63) & ~(size_t)63; }
__host__ __device__ inline SampleGeo lg_sample_geo(int n_vocab) {
    SampleGeo g;
    g.groups = (n_vocab + LG_SAMPLE_GROUP - 1) / LG_SAMPLE_GROUP;
    g.tops = (n_vocab + (1 << lg_top_shift(n_vocab)) - 1) >> lg_top_shift(n_vocab);
    g.maxes = (g.groups + 15) / 16;
    g.slices = (g.groups + 15) / 16;                 // of the passes after it at most: 16 groups or 64 each, as lg_hip_sample chooses
    size_t at = 0;
    g.gmax = at;  at += lg_up64((size_t)g.tops * 4);
    g.smin = at;  at += lg_up64((size_t)g.maxes * 4);
    g.mass = at;  at += LG_SAMPLE_BINS * 8;
    g.count = at; at += LG_SAMPLE_BINS * 4;
    g.gsum = at;  at += lg_up64((size_t)g.groups * 8);
    g.part = at;  at += lg_up64((size_t)g.slices * 24);
    g.ncand = at; at += 64;
    g.cand = at;  at += LG_SAMPLE_CAND * 8;
    g.row = at;
    return g;
}
__device__ __forceinline__ SampleWork lg_sample_work(char *base, const SampleGeo &g, int r) {
    char *const p = base + (size_t)r * g.row;
    return { (uint32_t *)(p + g.gmax), (uint32_t *)(p + g.smin), (lg_u64 *)(p + g.mass), (uint32_t *)(p + g.count), (lg_u64 *)(p + g.gsum), (lg_u64 *)(p + g.part),
             (uint32_t *)(p + g.ncand), (lg_u64 *)(p + g.cand) };
}
// The first largest; a small top-k; no top-k and no top-p; a border to be found; a temperature so small that the estimates' f32 does not hold 1 / T
enum { LG_ROW_FIRST, LG_ROW_SMALL, LG_ROW_FREE, LG_ROW_BORDER, LG_ROW_ALONE };
__device__ __forceinline__ int lg_row_kind(const SampleRow &p, int n_vocab) {
    if (!(p.temperature > 0)) return LG_ROW_FIRST;
    const bool k = p.top_k > 0 && p.top_k < n_vocab;
    if (k && p.top_k <= LG_SAMPLE_SMALL_K && p.top_k <= n_vocab >> (lg_top_shift(n_vocab) + 1)) return LG_ROW_SMALL;
    if (!(p.temperature > 1e-20f)) return LG_ROW_ALONE;
    return k || p.top_p < 1 ? LG_ROW_BORDER : LG_ROW_FREE;
}
__device__ __forceinline__ lg_u64 lg_least(const SampleRow &p) {      // the smallest weight that min-p keeps
    if (!(p.min_p > 0)) return 1;
    const double m = __builtin_ceil((double)p.min_p * LG_SAMPLE_ONE);
    return m >= 1 ? m < LG_SAMPLE_ONE ? (lg_u64)m : (lg_u64)LG_SAMPLE_ONE : 1;
}
// Tokens i .. i + 3; -inf behind the row's end.  VEC: rows aligned to 16 bytes
template <bool VEC>
__device__ __forceinline__ void lg_load4_at(const float *row, int n, int i, float (&l)[4]) {
    if (VEC && i + 3 < n) { const float4 x = *(const float4 *)(row + i); l[0] = x.x; l[1] = x.y; l[2] = x.z; l[3] = x.w; }
    else
        #pragma unroll
        for (int j = 0; j < 4; ++j) l[j] = i + j < n ? row[i + j] : -INFINITY;
}
// Four tokens of a lane in group `grp`
template <bool VEC>
__device__ __forceinline__ void lg_load4(const float *row, int n, int grp, float (&l)[4]) { lg_load4_at<VEC>(row, n, grp * LG_SAMPLE_GROUP + (threadIdx.x & 63) * 4, l); }

template <bool VEC>
__global__ __launch_bounds__(LG_SAMPLE_MAX_WG) void lg_k_sample_max(SampleArgs a, char *base) {
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const int r = blockIdx.y, part = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const SampleWork w = lg_sample_work(base, g, r);
    const float *row = a.logits + r * a.stride;
    __shared__ uint32_t s_min[LG_SAMPLE_MAX_WG / 64];
    float l[4][4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) lg_load4<VEC>(row, a.n_vocab, part * 16 + wave * 4 + j, l[j]);
    // the bins of a row that needs them are cleared on the way
    const SampleRow p = a.params[r];
    if (lg_row_kind(p, a.n_vocab) == LG_ROW_BORDER)
        for (int i = part * LG_SAMPLE_MAX_WG + threadIdx.x; i < LG_SAMPLE_BINS; i += g.maxes * LG_SAMPLE_MAX_WG) { w.mass[i] = 0; w.count[i] = 0; }
    if (part == 0 && threadIdx.x == 0) *w.ncand = 0;
    const bool quarters = lg_top_shift(a.n_vocab) == 6;
    uint32_t least = 0;                                      // as ~key: the largest is the smallest logit
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t m = 0x007FFFFFu;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t k = lg_key(l[j][i]);
            if (k > m) m = k;
            if (k > 0x007FFFFFu && ~k > least) least = ~k;
        }
        const int grp = part * 16 + wave * 4 + j;
        if (quarters) {
            m = lg_row_max(m);
            const int at = grp * 4 + (lane >> 4);
            if ((lane & 15) == 15 && at < g.tops) w.gmax[at] = m;
        } else {
            m = lg_wave_max(m);
            if (lane == 0 && grp < g.tops) w.gmax[grp] = m;
        }
    }
    least = lg_block_max<LG_SAMPLE_MAX_WG>(least, s_min);
    if (threadIdx.x == 0) w.smin[part] = least;
}

// The row's largest logit and the width of its bins
struct SampleSpan { Weigh wg; float top, scale, c; uint32_t key, least; bool wide; };      // key: of the largest logit, 0x007FFFFF: none; least: ~key of the smallest; scale: bins per unit of logit; c: base-2 exponents per unit
__device__ __forceinline__ SampleSpan lg_sample_span_of(const SampleRow &p, uint32_t key, uint32_t least, const double *tab) {
    SampleSpan s;
    s.key = key; s.least = least;
    s.top = lg_unkey(key);
    s.wg = lg_weigher(s.top, p.temperature, tab);
    s.c = -(float)(1.4426950408889634 / (double)p.temperature);
    const float reach = (float)LG_SAMPLE_REACH * p.temperature, width = fminf(s.top - lg_unkey(~least), reach);
    s.scale = width > 0 && width < INFINITY ? (float)LG_SAMPLE_BINS / width : 0;      // (0: all in the first bin)
    // `wide`: distances from the largest logit that f32 does not hold may have weight: an infinite largest logit, or a smallest one further away than f32 holds at a
    // temperature that reaches as far (above 1.08e37).  Bins and sums, which take distances in f32, leave such a row to lg_sample_row, which takes them in f64
    s.wide = s.top == INFINITY || width == INFINITY;
    return s;
}
// From what lg_k_sample_max left: this thread's share, asked for early, and all of it
struct SampleEnds { uint32_t key, least; };
template <int NT>
__device__ __forceinline__ SampleEnds lg_sample_ends(const SampleWork &w, const SampleGeo &g) {
    SampleEnds e{ 0, 0 };
    #pragma unroll
    for (int i = 0; i < LG_SAMPLE_GROUPS / NT; ++i) { const int at = threadIdx.x + i * NT; const uint32_t k = w.gmax[at < g.tops ? at : 0]; if (k > e.key) e.key = k; }
    const uint32_t k = w.smin[(int)threadIdx.x < g.maxes ? threadIdx.x : 0];          // (at most 128)
    e.least = k;
    return e;
}
template <int NT>
__device__ __forceinline__ SampleSpan lg_sample_span(const SampleRow &p, SampleEnds e, const double *tab, uint32_t *part) {
    lg_block_max2<NT>(e.key, e.least, part);
    return lg_sample_span_of(p, e.key, e.least, tab);
}
// Monotone in the logit, also as rounded: a larger logit never has a larger bin
__device__ __forceinline__ int lg_sample_bin(const SampleSpan &s, float l) {
    const float b = (s.top - l) * s.scale;                                            // (top - l is NaN for two infinities: the first bin)
    return b >= 0 ? b < (float)(LG_SAMPLE_BINS - 1) ? (int)b : LG_SAMPLE_BINS - 1 : 0;
}

// (64 groups to a workgroup: with 16, more workgroups add to the row's bins; 5 rows 7.6 -> 10.3 us)
template <bool VEC>
__global__ __launch_bounds__(LG_SAMPLE_WG) void lg_k_sample_bins(SampleArgs a, char *base) {
    constexpr int NT = LG_SAMPLE_WG;
    __shared__ lg_u64 mass[LG_SAMPLE_BINS];
    __shared__ uint32_t count[LG_SAMPLE_BINS], part[NT / 32];
    __shared__ double tab[32];
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const int r = blockIdx.y, slice = blockIdx.x, wave = threadIdx.x >> 6;
    const SampleRow p = a.params[r];
    const int kind = lg_row_kind(p, a.n_vocab);
    if (kind != LG_ROW_BORDER && !(kind == LG_ROW_FREE && slice == 0)) return;
    const SampleWork w = lg_sample_work(base, g, r);
    const float *row = a.logits + r * a.stride;
    const double entry = lg_table_entry();
    const SampleEnds ends = lg_sample_ends<NT>(w, g);
    float l[4][4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) lg_load4<VEC>(row, a.n_vocab, slice * (NT / 16) + j * (NT / 64) + wave, l[j]);
    lg_table_store(tab, entry);
    for (int i = threadIdx.x; i < LG_SAMPLE_BINS; i += NT) { mass[i] = 0; count[i] = 0; }
    const SampleSpan s = lg_sample_span<NT>(p, ends, tab, part);                      // (its barriers are the clearing's too)
    if (slice == 0 && threadIdx.x == 0) { w.ncand[8] = s.key; w.ncand[9] = s.least; }        // for the launches behind this one
    if (kind != LG_ROW_BORDER || s.key == 0x007FFFFFu || s.wide) return;
    const bool by_count = p.top_k > 0 && p.top_k < a.n_vocab, by_mass = p.top_p < 1;
    #pragma unroll
    for (int j = 0; j < 4; ++j)
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = l[j][i], e = x == s.top ? 0.0f : (s.top - x) * s.c;       // base 2; a weight of 0 starts near -45
            if (!(e > -46.0f)) continue;                                              // (NaN too)
            if (e < -44.0f && !lg_weigh(s.wg, x)) continue;
            const int b = lg_sample_bin(s, x);
            // an estimate, to 2^-32 of the largest weight: 2^19 of them are within 2^-13 of their sum.  In whole numbers too: no order changes it
            if (by_mass) atomicAdd(&mass[b], (lg_u64)(uint32_t)(__builtin_amdgcn_exp2f(e + 31.0f) + 0.5f));
            if (by_count) atomicAdd(&count[b], 1u);
        }
    __syncthreads();
    for (int i = threadIdx.x; i < LG_SAMPLE_BINS; i += NT) {
        if (by_mass && mass[i]) atomicAdd(&w.mass[i], mass[i]);
        if (by_count && count[i]) atomicAdd(&w.count[i], count[i]);
    }
}

// The bins that can hold the border, from the row's estimates: the same in every workgroup of a row
struct SampleRange { int first, last, cut; uint32_t above; };        // top-p's border is in bins first..last, top-k's in bin cut (LG_SAMPLE_BINS: none), behind `above` tokens
template <int NT>
struct SampleRangeLds { lg_u64 part[NT / 64]; SampleRange r; lg_u64 lo, hi; };
template <int NT>
struct SampleBins { lg_u64 m[LG_SAMPLE_BINS / NT]; uint32_t c[LG_SAMPLE_BINS / NT]; };           // this thread's, asked for early
template <int NT>
__device__ __forceinline__ SampleBins<NT> lg_sample_bins(const SampleWork &w) {
    constexpr int PT = LG_SAMPLE_BINS / NT;
    SampleBins<NT> b;
    #pragma unroll
    for (int i = 0; i < PT; ++i) { b.m[i] = w.mass[threadIdx.x * PT + i]; b.c[i] = w.count[threadIdx.x * PT + i]; }
    return b;
}
template <int NT>
__device__ __forceinline__ SampleRange lg_sample_range(const SampleArgs &a, const SampleRow &p, const SampleBins<NT> &bins, SampleRangeLds<NT> &s) {
    constexpr int PT = LG_SAMPLE_BINS / NT;
    const int b0 = threadIdx.x * PT;
    const bool by_count = p.top_k > 0 && p.top_k < a.n_vocab, by_mass = p.top_p < 1;
    if (threadIdx.x == 0) s.r = { 0, LG_SAMPLE_BINS - 1, LG_SAMPLE_BINS, 0 };
    const lg_u64 (&m)[PT] = bins.m;
    if (by_count) {
        const uint32_t (&c)[PT] = bins.c;
        lg_u64 sum = 0, all;
        #pragma unroll
        for (int i = 0; i < PT; ++i) sum += c[i];
        lg_u64 run = lg_block_run<NT>(sum, s.part, &all) - sum;
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            if (run < (lg_u64)p.top_k && run + c[i] >= (lg_u64)p.top_k) { s.r.cut = b0 + i; s.r.above = (uint32_t)run; }
            run += c[i];
        }
        __syncthreads();
    }
    if (by_mass) {
        lg_u64 sum = 0, all;
        #pragma unroll
        for (int i = 0; i < PT; ++i) sum += m[i];
        const lg_u64 start = lg_block_run<NT>(sum, s.part, &all) - sum;
        lg_u64 run = start;
        const int cut = s.r.cut;
        if (cut == LG_SAMPLE_BINS) { if (threadIdx.x == 0) { s.lo = all; s.hi = all; } }
        else
            #pragma unroll
            for (int i = 0; i < PT; ++i) { if (b0 + i == cut) { s.lo = run; s.hi = run + m[i]; } run += m[i]; }
        __syncthreads();
        const double slack = (double)s.hi / LG_SAMPLE_SLACK;
        const double lo = (double)p.top_p * (double)s.lo - slack, hi = (double)p.top_p * (double)s.hi + slack;
        run = start;
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            const double before = (double)run, to = (double)(run + m[i]);
            if (before < lo && to >= lo) s.r.first = b0 + i;
            if (before < hi && to >= hi) s.r.last = b0 + i;
            run += m[i];
        }
    } else if (threadIdx.x == 0) s.r.first = s.r.last = s.r.cut;
    __syncthreads();
    SampleRange q = s.r;
    if (q.last > q.cut) q.last = q.cut;
    return q;
}

// NT threads read 16 (256) or 64 (1024) groups
template <bool VEC, int NT>
__global__ __launch_bounds__(NT) void lg_k_sample_sums(SampleArgs a, char *base) {
    __shared__ uint32_t part[NT / 32], s_n;
    __shared__ SampleRangeLds<NT> s_range;
    __shared__ double tab[32];
    __shared__ lg_u64 s_sum[3], s_cand[NT * 2];                            // candidates on their way out
    constexpr uint32_t ROOM = NT * 2;
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const int r = blockIdx.y, slice = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const SampleRow p = a.params[r];
    const int kind = lg_row_kind(p, a.n_vocab);
    if (kind != LG_ROW_BORDER && kind != LG_ROW_FREE) return;
    const SampleWork w = lg_sample_work(base, g, r);
    const float *row = a.logits + r * a.stride;
    const bool border = kind == LG_ROW_BORDER;
    const double entry = lg_table_entry();
    const SampleBins<NT> bins = border ? lg_sample_bins<NT>(w) : SampleBins<NT>{};
    float l[4][4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) lg_load4<VEC>(row, a.n_vocab, slice * (NT / 16) + j * (NT / 64) + wave, l[j]);
    const uint32_t key = w.ncand[8], least_key = w.ncand[9];
    lg_table_store(tab, entry);
    if (threadIdx.x < 3) s_sum[threadIdx.x] = 0;
    if (threadIdx.x == 3) s_n = 0;
    SampleRange q{ LG_SAMPLE_BINS, -1, LG_SAMPLE_BINS, 0 };
    if (border) {
        q = lg_sample_range<NT>(a, p, bins, s_range);
        if (slice == 0 && threadIdx.x == 0) *(SampleRange *)(w.ncand + 4) = q;
    } else __syncthreads();
    const SampleSpan s = lg_sample_span_of(p, key, least_key, tab);
    if (s.key == 0x007FFFFFu || s.wide) return;
    const lg_u64 least = lg_least(p);
    // What is behind top-k's bin, or below min-p where nothing else is asked, needs no weight (a little more than that gets one); a wavefront without such a
    // token goes on, one with some does all of its lanes without branches
    float floor_ = LG_SAMPLE_FLOOR;
    if (border && q.cut < LG_SAMPLE_BINS && s.scale > 0) floor_ = fmaxf(floor_, s.c * ((float)(q.cut + 1) / s.scale) * 1.0001f - 0.01f);
    if (!border && least > 1) floor_ = fmaxf(floor_, __builtin_amdgcn_logf((float)least * 5.684341886080802e-14f) - 0.01f);       // (2^-44; in base 2)
    lg_u64 whole = 0, above = 0;                               // sums of all before top-k's bin and of those above the candidates
    uint32_t kept = 0;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int grp = slice * (NT / 16) + j * (NT / 64) + wave;
        lg_u64 sum = 0, of_group = 0;
        uint32_t cands = 0;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = l[j][i];
            const bool needed = (s.top - x) * s.c > floor_;
            if (!__any(needed)) continue;
            const lg_u64 wt = needed ? lg_weight(s.wg, x) : 0;
            const int b = border ? lg_sample_bin(s, x) : 0;
            const bool in = b < q.first, stays = in && wt >= least;
            whole += b < q.cut ? wt : 0;
            of_group += in ? wt : 0;
            sum += stays ? wt : 0;
            kept += stays;
            cands |= (uint32_t)(border && !in && wt && (b <= q.last || b == q.cut)) << i;
        }
        above += of_group;
        if (cands)
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                if (cands >> i & 1) {
                    const uint32_t at = atomicAdd(&s_n, 1u);
                    if (at < ROOM) s_cand[at] = (lg_u64)~lg_key(l[j][i]) << 32 | (uint32_t)(grp * LG_SAMPLE_GROUP + lane * 4 + i);
                }
        sum = lg_wave_total(sum);
        if (lane == 0 && grp < g.groups) w.gsum[grp] = sum;
    }
    above = lg_wave_total(above); whole = lg_wave_total(whole); kept = lg_wave_total(kept);
    if (lane == 0) { atomicAdd(&s_sum[0], above); atomicAdd(&s_sum[1], whole); atomicAdd(&s_sum[2], (lg_u64)kept); }
    __syncthreads();
    if (threadIdx.x < 3) w.part[slice * 3 + threadIdx.x] = s_sum[threadIdx.x];
    if (border && s_n) {
        // (what did not fit counts all the same: more than the row may have)
        if (threadIdx.x == 0) part[0] = atomicAdd(w.ncand, s_n > ROOM ? LG_SAMPLE_CAND + 1 : s_n);
        __syncthreads();
        const uint32_t at = part[0], n = s_n < ROOM ? s_n : ROOM;
        for (uint32_t i = threadIdx.x; i < n; i += NT) if (at + i < LG_SAMPLE_CAND) w.cand[at + i] = s_cand[i];
    }
}

// One workgroup, one row.  Candidates are ~key << 32 | index: smaller is earlier in the order.  This thread's are in registers, with their measures.
#define LG_SAMPLE_LIST    512                    // what stays of a small top-k, and its candidates that are ordered by parts of their keys
static_assert(LG_SAMPLE_LIST >= LG_SAMPLE_SMALL_K && LG_SAMPLE_LIST <= 512, "room for what stays; sums of 54 bits");
struct SampleFinishLds {
    lg_u64 sum[LG_SAMPLE_GROUPS], bin[1024], list[LG_SAMPLE_LIST], size[64], cand[LG_SAMPLE_CAND], part[LG_SAMPLE_WG / 32], part3[3], last, rest, whole;
    double tab[32];
    uint32_t key[LG_SAMPLE_WG / 32], groups[LG_SAMPLE_GROUPS];
    uint32_t n, n_groups;
    int at, idx;
    SampleLds alone;
};
// The candidate at which the running sum of measures, in order, reaches `want` (1 .. the sum of all); measures of 0 are no candidates.  1024 equal parts
// between the first and the last candidate, the part that holds the border cut again until it has at most 64 of them (once for logits that lie
// anywhere, again for a group of equal ones, by their index then), and a wavefront over these.  The parts are of the candidates as numbers, whose keys are
// logarithms of logits; BINS: the first ones are bins of logits (`bin`, 0..1023), where the candidates are on both sides of 0 and most of the numbers between
// them the keys of tiny logits.
template <int PT, bool BINS, typename C, typename M, typename B>
__device__ __forceinline__ lg_u64 lg_among(C c, M measure, B bin, lg_u64 want, SampleFinishLds &s) {          // c(i), measure(i): of this thread's PT tokens
    const int t = threadIdx.x;
    uint32_t out = 0;                                        // bit i: token i is in none of the parts any more
    auto m = [&](int i) { return out >> i & 1 ? (lg_u64)0 : measure(i); };
    auto round = [&](auto part_of) {                         // false: the part of the border has more than 64
        #pragma unroll
        for (int i = 0; i < PT; ++i) { const lg_u64 x = m(i); if (x) atomicAdd(&s.bin[part_of(i)], x); }
        __syncthreads();
        lg_u64 all;
        const lg_u64 mine = s.bin[t], run = lg_block_run<LG_SAMPLE_WG>(mine, s.part, &all);
        if (run >= want && run - mine < want) { s.at = t; s.rest = run - mine; }
        __syncthreads();
        const uint32_t part = (uint32_t)s.at;
        want -= s.rest;
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            const lg_u64 x = m(i);
            if (!x) continue;
            if (part_of(i) != part) { out |= 1u << i; continue; }
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < 64) { s.list[at] = c(i); s.size[at] = x; }
        }
        __syncthreads();
        return s.n <= 64;
    };
    bool done;
    if constexpr (BINS) {
        s.bin[t] = 0;
        if (t == 0) s.n = 0;
        __syncthreads();
        done = round([&](int i) { return (uint32_t)bin(i); });
    } else {                                                 // by the keys alone
        uint32_t from = 0, to = 0;
        #pragma unroll
        for (int i = 0; i < PT; ++i) if (measure(i)) { const uint32_t x = (uint32_t)(c(i) >> 32); if (~x > from) from = ~x; if (x > to) to = x; }
        s.bin[t] = 0;
        if (t == 0) s.n = 0;
        lg_block_max2<LG_SAMPLE_WG>(from, to, s.key);        // (its barriers are the clearing's too)
        from = ~from;
        const uint32_t span = to - from;
        const int shift = span >= 1024 ? 32 - __builtin_clz(span) - 10 : 0;
        done = round([&](int i) { return ((uint32_t)(c(i) >> 32) - from) >> shift; });
    }
    while (!done) {                                          // by key and index (every round but the last leaves out a candidate: the first and the last lie in different parts)
        lg_u64 from = 0, to = 0;                             // from as its complement
        #pragma unroll
        for (int i = 0; i < PT; ++i) if (m(i)) { const lg_u64 x = c(i); if (~x > from) from = ~x; if (x > to) to = x; }
        lg_block_max2<LG_SAMPLE_WG>(from, to, s.part);       // (its first barrier: s.n and the bins are no longer read)
        s.bin[t] = 0;
        if (t == 0) s.n = 0;
        __syncthreads();
        from = ~from;
        const lg_u64 span = to - from;
        const int shift = span >= 1024 ? 64 - __builtin_clzll(span) - 10 : 0;
        done = round([&](int i) { return (uint32_t)((c(i) - from) >> shift); });
    }
    if (t < 64) {
        const uint32_t n = s.n;
        const lg_u64 me = (uint32_t)t < n ? s.list[t] : ~0ull, own = (uint32_t)t < n ? s.size[t] : 0;
        lg_u64 upto = 0;
        for (uint32_t i = 0; i < n; ++i) { const lg_u64 x = lg_lane(me, i), y = lg_lane(own, i); if (x <= me) upto += y; }
        if (own && upto >= want && upto - own < want) s.last = me;
    }
    __syncthreads();
    return s.last;
}

// Whole rows of up to PT * 1024 tokens (WHOLE: no launch came before), or what the launches before left of longer ones (PT * 1024 = LG_SAMPLE_CAND)
// False: the row is to be taken from its logits alone
template <bool VEC, bool WHOLE, int PT>
__device__ __forceinline__ bool lg_sample_finish(const SampleArgs &a, char *base, const SampleRow &p, SampleFinishLds &s) {
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, n_vocab = a.n_vocab;
    const double entry = lg_table_entry();
    const float *row = a.logits + r * a.stride, u = a.u[r];
    const SampleGeo g = lg_sample_geo(n_vocab);
    const SampleWork w = WHOLE ? SampleWork{} : lg_sample_work(base, g, r);
    const int kind = lg_row_kind(p, n_vocab), top_shift = lg_top_shift(n_vocab);
    const lg_u64 least = lg_least(p);
    auto answer = [&](int tok, double prob, int kept) {
        a.tok[r] = tok;
        if (a.prob) a.prob[r] = (float)prob;
        if (a.kept) a.kept[r] = kept;
    };
    if (t == 0) { s.n = 0; s.n_groups = 0; s.at = n_vocab; s.idx = 0; }
    lg_u64 kept_c[WHOLE ? 1 : PT], m[PT];                    // this thread's candidates and their weights
    float x[WHOLE ? PT : 1];                                 // (of a whole row its tokens: PT in a row to a thread)
    auto c = [&](int i) { if constexpr (WHOLE) return (lg_u64)~lg_key(x[i]) << 32 | (uint32_t)(t * PT + i); else return kept_c[i]; };
    lg_u64 above = 0, total = 0, all;                        // sum of the tokens before the candidates; what top-p goes by
    SampleSpan span;
    SampleRange q{ LG_SAMPLE_BINS, -1, LG_SAMPLE_BINS, 0 };
    uint32_t kept = 0, from = 0;                             // from: a small top-k's candidates are the tokens with this key and larger ones
    int n = 0;
    if (WHOLE) {
        uint32_t key = 0, least_key = 0;
        #pragma unroll
        for (int i = 0; i < PT; i += 4) {
            const int at = t * PT + i;
            if (VEC && at + 3 < n_vocab) { const float4 v = *(const float4 *)(row + at); x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w; }
            else
                #pragma unroll
                for (int j = 0; j < 4; ++j) x[i + j] = at + j < n_vocab ? row[at + j] : -INFINITY;
        }
        #pragma unroll
        for (int i = 0; i < PT; ++i) { const uint32_t k = lg_key(x[i]); if (k > key) key = k; if (k > 0x007FFFFFu && ~k > least_key) least_key = ~k; }
        lg_table_store(s.tab, entry);
        lg_block_max2<LG_SAMPLE_WG>(key, least_key, s.key);  // (its barriers: the table's too)
        span = lg_sample_span_of(p, key, least_key, s.tab);
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            m[i] = kind != LG_ROW_FIRST && key != 0x007FFFFFu ? lg_weigh(span.wg, x[i]) : 0;
            if (kind == LG_ROW_FIRST && lg_key(x[i]) == key && t * PT + i < n_vocab) atomicMin(&s.at, t * PT + i);
        }
    } else {
        if (kind == LG_ROW_ALONE) { lg_table_store(s.tab, entry); return false; }
        // what the launches before left, all requested at once
        uint32_t gk[LG_SAMPLE_GROUPS / LG_SAMPLE_WG];
        #pragma unroll
        for (int i = 0; i < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++i) { const int at = t + i * LG_SAMPLE_WG; gk[i] = w.gmax[at < g.tops ? at : 0]; if (at >= g.tops) gk[i] = 0; }
        if (kind == LG_ROW_BORDER) {
            #pragma unroll
            for (int i = 0; i < PT; ++i) if constexpr (!WHOLE) kept_c[i] = w.cand[t + i * LG_SAMPLE_WG];
            n = (int)*w.ncand;
            q = *(const SampleRange *)(w.ncand + 4);
        }
        if (kind == LG_ROW_BORDER || kind == LG_ROW_FREE) {
            if (wave < 3) {                                  // (at most 128 slices: a wavefront for each sum)
                lg_u64 x = 0;
                for (int i = lane; i < a.slices; i += 64) x += w.part[i * 3 + wave];
                x = lg_wave_total(x);
                if (lane == 0) s.part3[wave] = x;
            }
            for (int i = t; i < LG_SAMPLE_GROUPS; i += LG_SAMPLE_WG) s.sum[i] = i < g.groups ? w.gsum[i] : 0;
        }
        lg_table_store(s.tab, entry);
        uint32_t low = 0;                                    // ~key of the smallest of the groups' largest logits
        if (kind == LG_ROW_SMALL) {
            uint32_t key = 0;
            #pragma unroll
            for (int i = 0; i < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++i) { if (gk[i] > key) key = gk[i]; if (gk[i] > 0x007FFFFFu && ~gk[i] > low) low = ~gk[i]; }
            s.bin[t] = 0;
            lg_block_max2<LG_SAMPLE_WG>(key, low, s.key);
            span = lg_sample_span_of(p, key, low, s.tab);
            low = ~low;
        } else if (kind == LG_ROW_FIRST) span = lg_sample_span<LG_SAMPLE_WG>(p, lg_sample_ends<LG_SAMPLE_WG>(w, g), s.tab, s.key);
        else {
            span = lg_sample_span_of(p, w.ncand[8], w.ncand[9], s.tab);
            __syncthreads();                                 // (the sums and the table)
        }
        if (kind == LG_ROW_BORDER || kind == LG_ROW_FREE) { above = s.part3[0]; total = s.part3[1]; kept = (uint32_t)s.part3[2]; }
        if (span.wide && (kind == LG_ROW_BORDER || kind == LG_ROW_FREE)) return false;      // (the launches before left nothing)
        if (span.key != 0x007FFFFFu && kind == LG_ROW_FIRST) {
            #pragma unroll
            for (int i = 0; i < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++i) if (gk[i] == span.key) atomicMin(&s.at, t + i * LG_SAMPLE_WG);
            __syncthreads();
            const int grp = s.at;
            __syncthreads();
            if (t == 0) s.at = n_vocab;
            __syncthreads();
            const int first = (grp << top_shift) + lane * 4;
            if (wave == 0 && lane < 1 << (top_shift - 2)) {
                float l[4];
                lg_load4_at<VEC>(row, n_vocab, first, l);
                #pragma unroll
                for (int i = 0; i < 4; ++i) if (lg_key(l[i]) == span.key) atomicMin(&s.at, first + i);
            }
        } else if (kind == LG_ROW_SMALL) {
            // a logit that at least top_k groups reach: the lower edge of one of 1024 equal parts between the groups' smallest and largest maxima
            const uint32_t wide = span.key - low;
            const int shift = wide >= 1024 ? 32 - __builtin_clz(wide) - 10 : 0;
            #pragma unroll
            for (int i = 0; i < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++i) if (gk[i] > 0x007FFFFFu) atomicAdd(&s.bin[(gk[i] - low) >> shift], 1ull);
            __syncthreads();
            const lg_u64 mine = s.bin[1023 - t], run = lg_block_run<LG_SAMPLE_WG>(mine, s.part, &all);
            if (run >= (lg_u64)p.top_k && run - mine < (lg_u64)p.top_k) s.idx = 1023 - t;
            __syncthreads();
            s.bin[t] = 0;
            from = all >= (lg_u64)p.top_k ? low + ((uint32_t)s.idx << shift) : 0x00800000u;      // (fewer groups than top_k: every token)
            #pragma unroll
            for (int i = 0; i < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++i) if (gk[i] >= from) s.groups[atomicAdd(&s.n_groups, 1u)] = t + i * LG_SAMPLE_WG;
            __syncthreads();
            const int n_groups = (int)s.n_groups;
            constexpr int AT_ONCE = 6;
            const int each = 8 - top_shift;                          // a wavefront's load is one group, or four quarters
            for (int at = wave; at << each < n_groups; at += AT_ONCE * (LG_SAMPLE_WG / 64)) {      // groups of a wavefront on their way together: k = 64 takes 66 to 80 in all
                float l[AT_ONCE][4];
                int tok[AT_ONCE];
                #pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    const int b = ((at + j * (LG_SAMPLE_WG / 64)) << each) + (lane >> (top_shift - 2));
                    tok[j] = b < n_groups ? (int)(s.groups[b] << top_shift) + (lane & ((1 << (top_shift - 2)) - 1)) * 4 : n_vocab;         // (behind the row's end: -inf)
                    lg_load4_at<VEC>(row, n_vocab, tok[j], l[j]);
                }
                uint32_t found = 0;
                #pragma unroll
                for (int j = 0; j < AT_ONCE; ++j)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) found += lg_key(l[j][i]) >= from;
                uint32_t to = lg_wave_run(found);
                const uint32_t of_all = lg_last_lane(to);
                uint32_t first = 0;
                if (lane == 0) first = atomicAdd(&s.n, of_all);
                to += lg_lane(first, 0) - found;
                #pragma unroll
                for (int j = 0; j < AT_ONCE; ++j)
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t k = lg_key(l[j][i]);
                        if (k < from) continue;
                        if (to < LG_SAMPLE_CAND) s.cand[to] = (lg_u64)~k << 32 | (uint32_t)(tok[j] + i);
                        ++to;
                    }
            }
            __syncthreads();
            n = (int)s.n;
            #pragma unroll
            for (int i = 0; i < PT; ++i) if constexpr (!WHOLE) { const int at = t + i * LG_SAMPLE_WG; kept_c[i] = at < n && at < LG_SAMPLE_CAND ? s.cand[at] : 0; }
        }
        if (n > LG_SAMPLE_CAND) return false;
        #pragma unroll
        for (int i = 0; i < PT; ++i) m[i] = t + i * LG_SAMPLE_WG < n ? lg_weigh(span.wg, lg_unkey(~(uint32_t)(c(i) >> 32))) : 0;
    }
    if (span.key == 0x007FFFFFu) { if (t == 0) answer(-1, 0, 0); return true; }
    if (kind == LG_ROW_FIRST) {
        __syncthreads();
        if (t == 0) answer(s.at, 1, 1);
        return true;
    }
    auto target_of = [&](lg_u64 S) {
        const lg_u64 x = u > 0 ? (lg_u64)__builtin_floor((u < 1 ? (double)u : 1.0) * (double)S) : 0;
        return x > S - 1 ? S - 1 : x;
    };
    auto bin = [&](int i) { if constexpr (WHOLE) return lg_sample_bin(span, x[i]) * 1024 / LG_SAMPLE_BINS; else return 0; };
    // top-k, then top-p: `last` is the last token in the order that stays
    lg_u64 last = ~0ull;
    bool lost = false;                                       // the candidates do not hold the border after all
    const bool small = !WHOLE && kind == LG_ROW_SMALL;
    constexpr lg_u64 one_more = 1ull << 54, sum_of = one_more - 1;                           // a count above 54 bits of sum: 512 weights of 2^44 are 2^53
    // At most LG_SAMPLE_SMALL_K of R candidates a thread stay: the part of the draw among 1024 of the vocabulary, and pair by pair those in it (each one's
    // running sum from all that stay instead: 58.0 and 36.6 us a row where 490 stay).  The parts and s.n are 0
    auto small_draw = [&](auto regs, lg_u64 last) {
        constexpr int R = decltype(regs)::value;
        auto stays = [&](int i) { return m[i] >= least && c(i) <= last; };
        auto piece = [&](int i) { return (int)((uint32_t)c(i) / (LG_SAMPLE_VOCAB / 1024)); };
        #pragma unroll
        for (int i = 0; i < R; ++i) if (stays(i)) atomicAdd(&s.bin[piece(i)], one_more | m[i]);
        __syncthreads();
        const lg_u64 here = s.bin[t], upto = lg_block_run<LG_SAMPLE_WG>(here, s.part, &all), S = all & sum_of, target = target_of(S), before = (upto - here) & sum_of;
        if ((upto & sum_of) > target && before <= target) { s.at = t; s.rest = before; }
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < R; ++i) if (stays(i) && piece(i) == s.at) { const uint32_t at = atomicAdd(&s.n, 1u); s.list[at] = c(i); s.cand[at] = m[i]; }
        __syncthreads();
        const uint32_t in = s.n;
        if ((uint32_t)t >= in) return;
        const uint32_t me = (uint32_t)s.list[t];
        const lg_u64 own = s.cand[t];
        lg_u64 to = s.rest;
        for (uint32_t i = 0; i < in; ++i) if ((uint32_t)s.list[i] <= me) to += s.cand[i];
        if (to > target && to - own <= target) answer((int)me, (double)own / (double)S, (int)(all >> 54));
    };
    if (small && n <= LG_SAMPLE_LIST) {
        // a few hundred: each one's place in the order and the sum up to it from 1024 equal parts of the keys, and pair by pair within its part.
        // (All pairs instead, in a third of the barriers: 16.6 and 17.2 us at top-k 20, even at 40, 21.1 and 18.7 at 100.)
        const lg_u64 me = c(0), own = m[0];
        const uint32_t wide = span.key - from;
        const int shift = wide >= 1024 ? 32 - __builtin_clz(wide) - 10 : 0;
        const uint32_t part = (span.key - ~(uint32_t)(me >> 32)) >> shift;
        if (own) atomicAdd(&s.bin[part], one_more | own);
        __syncthreads();
        const lg_u64 mine = s.bin[t], before = lg_block_run<LG_SAMPLE_WG>(mine, s.part, &all) - mine;
        s.sum[t] = before;
        s.groups[t] = (uint32_t)(before >> 54);              // where the next one of the part goes
        __syncthreads();
        if (own) { const uint32_t at = atomicAdd(&s.groups[part], 1u); s.list[at] = me; s.cand[at] = own; }
        __syncthreads();
        lg_u64 upto = 0;
        uint32_t place = 0;
        if (own) {
            const lg_u64 first = s.sum[part];
            place = (uint32_t)(first >> 54); upto = first & sum_of;
            for (uint32_t i = place, to = place + (uint32_t)(s.bin[part] >> 54); i < to; ++i) if (s.list[i] <= me) { upto += s.cand[i]; ++place; }
        }
        const uint32_t count = (uint32_t)(all >> 54), k = (uint32_t)p.top_k < count ? (uint32_t)p.top_k : count;
        if (own && place == k) s.whole = upto;
        __syncthreads();
        const lg_u64 W = s.whole;
        s.bin[t] = 0;
        if (t == 0) s.n = 0;
        lg_u64 want = W;
        if (p.top_p < 1) { const double want_d = __builtin_ceil((double)p.top_p * (double)W); want = want_d >= 1 ? (lg_u64)want_d < W ? (lg_u64)want_d : W : 1; }
        if (own && upto >= want && upto - own < want) s.last = me;
        __syncthreads();
        small_draw(std::integral_constant<int, 1>{}, s.last);
        return true;
    }
    const bool longer = !WHOLE && !small;      // the candidates are a part of what stays
    if (WHOLE || small || q.cut < LG_SAMPLE_BINS) {
        // (top-k counts tokens; of a longer row those of its bin)
        auto one = [&](int i) { return (lg_u64)(m[i] && (!longer || lg_sample_bin(span, lg_unkey(~(uint32_t)(c(i) >> 32))) == q.cut)); };
        lg_u64 mine = 0;
        #pragma unroll
        for (int i = 0; i < PT; ++i) mine += one(i);
        const lg_u64 have = lg_block_sum<LG_SAMPLE_WG>(mine, s.part), want = p.top_k > 0 ? (lg_u64)p.top_k - (longer ? q.above : 0) : have + 1;
        if (want <= have) last = lg_among<PT, WHOLE>(c, one, bin, want, s);         // (also where all of them stay: what comes behind them does not)
        else lost = longer;
        lg_u64 sum = 0;
        #pragma unroll
        for (int i = 0; i < PT; ++i) { if (c(i) > last) m[i] = 0; else if (one(i)) sum += m[i]; }
        if (p.top_p < 1) total += lg_block_sum<LG_SAMPLE_WG>(sum, s.part);
    }
    if (p.top_p < 1 && kind != LG_ROW_FREE && !lost) {
        const double want_d = __builtin_ceil((double)p.top_p * (double)total);
        const lg_u64 want = want_d >= 1 ? (lg_u64)want_d < total ? (lg_u64)want_d : total : 1;
        // (bins between top-p's and top-k's hold tokens that are no candidates: those of top-k's are not counted behind them)
        const bool gap = longer && q.cut < LG_SAMPLE_BINS && q.last < q.cut - 1;
        auto in = [&](int i) { return gap && lg_sample_bin(span, lg_unkey(~(uint32_t)(c(i) >> 32))) > q.last ? (lg_u64)0 : m[i]; };
        lg_u64 sum = 0;
        #pragma unroll
        for (int i = 0; i < PT; ++i) sum += in(i);
        const lg_u64 have = lg_block_sum<LG_SAMPLE_WG>(sum, s.part);
        if (above >= want || above + have < want) lost = true;
        else last = lg_among<PT, WHOLE>(c, in, bin, want - above, s);
    }
    if (lost) return false;
    lg_u64 sum = 0;
    uint32_t mine = 0;
    #pragma unroll
    for (int i = 0; i < PT; ++i) { if (c(i) > last || m[i] < least) m[i] = 0; sum += m[i]; mine += m[i] != 0; }
    if (!small) kept += (uint32_t)lg_block_sum<LG_SAMPLE_WG>((lg_u64)mine, s.part);
    if (WHOLE) {                                             // the candidates lie in index order
        lg_u64 run = lg_block_run<LG_SAMPLE_WG>(sum, s.part, &all) - sum;
        const lg_u64 target = target_of(all);
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            if (m[i] && run <= target && run + m[i] > target) answer(t * PT + i, (double)m[i] / (double)all, (int)kept);
            run += m[i];
        }
        return true;
    }
    if (small) {
        s.bin[t] = 0;
        if (t == 0) s.n = 0;
        __syncthreads();
        small_draw(std::integral_constant<int, PT>{}, last);
        return true;
    }
    // the groups' sums with the candidates that stay, the group of the draw, and the token in it
    #pragma unroll
    for (int i = 0; i < PT; ++i) if (m[i]) atomicAdd(&s.sum[(uint32_t)c(i) / LG_SAMPLE_GROUP], m[i]);
    __syncthreads();
    constexpr int GT = LG_SAMPLE_GROUPS / LG_SAMPLE_WG;
    lg_u64 gs[GT];
    sum = 0;
    #pragma unroll
    for (int i = 0; i < GT; ++i) { gs[i] = s.sum[t * GT + i]; sum += gs[i]; }
    lg_u64 run = lg_block_run<LG_SAMPLE_WG>(sum, s.part, &all) - sum;
    const lg_u64 target = target_of(all);
    #pragma unroll
    for (int i = 0; i < GT; ++i) {
        if (run <= target && run + gs[i] > target) { s.at = t * GT + i; s.rest = target - run; }
        run += gs[i];
    }
    __syncthreads();
    if (wave == 0) {
        const int grp = s.at;
        const lg_u64 rest = s.rest;
        float l[4];
        lg_load4<VEC>(row, n_vocab, grp, l);
        lg_u64 wt[4];
        sum = 0;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            wt[i] = ((lg_u64)~lg_key(l[i]) << 32 | (uint32_t)(grp * LG_SAMPLE_GROUP + lane * 4 + i)) <= last ? lg_weigh(span.wg, l[i]) : 0;
            if (wt[i] < least) wt[i] = 0;
            sum += wt[i];
        }
        lg_u64 at = lg_wave_run(sum) - sum;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (wt[i] && at <= rest && at + wt[i] > rest) answer(grp * LG_SAMPLE_GROUP + lane * 4 + i, (double)wt[i] / (double)all, (int)kept);
            at += wt[i];
        }
    }
    return true;
}
template <bool VEC, bool WHOLE, int PT>
__global__ __launch_bounds__(LG_SAMPLE_WG) void lg_k_sample_finish(SampleArgs a, char *base) {
    __shared__ SampleFinishLds s;
    const SampleRow p = a.params[blockIdx.x];
    if (lg_sample_finish<VEC, WHOLE, PT>(a, base, p, s)) return;
    __syncthreads();
    lg_sample_row(a, blockIdx.x, p, s.tab, s.alone);
}
