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
// A row is read by many workgroups and finished by one, in four launches (one for rows of at most LG_SAMPLE_CAND tokens):
//   lg_k_sample_max     the largest logit of every group of 256
//   lg_k_sample_bins    rows whose border is to be found: 2048 bins of equal width from the largest logit down, how many tokens and about what sum each holds
//   lg_k_sample_sums    the exact sum of every group above the bins that can hold the border, and the tokens in those (candidates)
//   lg_k_sample_finish  one workgroup a row: the border among the candidates, the draw by the groups' sums and the tokens of one group.
//                       Rows of a small top-k come here at once: the k-th largest of the groups' largest logits is at most the k-th largest logit, so
//                       the tokens not below it, few more than k, are the candidates.
// What the second and third find only narrows down: the border is taken from whole-number sums, and where the candidates turn out not to hold
// it (too many, a bin's sum estimated too far off) lg_sample_row finds it from the row alone.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#define LG_SAMPLE_WG     1024
#define LG_SAMPLE_VOCAB  (1 << 19)
#define LG_SAMPLE_ONE    17592186044416.0        // 2^44
typedef unsigned long long lg_u64;

struct SampleRow { float temperature; int32_t top_k; float top_p, min_p; };     // struct lg_hip_sampling
struct SampleArgs {
    const float *logits; long long stride;
    const SampleRow *params;
    const float *u;
    int32_t *tok; float *prob; int32_t *kept;   // the last two may be null
    int n_vocab;
};

// A number that is larger for a larger logit; NaN and -inf give 0x007FFFFF, -0 what +0 gives
__device__ __forceinline__ uint32_t lg_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    if (l != l) return 0x007FFFFFu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lg_unkey(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// What a row's weights need: M and 1 / T (0 for a T of infinity)
struct Weigh { double top, inv; };
// 2^44 e^((l - top) inv), rounded.  e^x by n = rint(x / ln 2), r = x - n ln 2 and its power series up to r^12 (|r| <= 0.35: the next term is 2e-16);
// adding 2^52 leaves the whole number in the low bits.  Below -31.5 it is 0.
__device__ __forceinline__ lg_u64 lg_weigh(const Weigh &w, float l) {
    const double x = l == (float)w.top ? 0.0 : ((double)l - w.top) * w.inv;
    if (!(x >= -31.5) || l == -INFINITY) return 0;
    const double n = __builtin_rint(x * 1.4426950408889634074);
    double r = __builtin_fma(n, -6.93147180369123816490e-01, x);
    r = __builtin_fma(n, -1.90821492927058770002e-10, r);
    double p = 1.0 / 479001600.0;
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    const double y = __builtin_fma(p, __longlong_as_double((lg_u64)(1023 + 44 + (int)n) << 52), 4503599627370496.0);
    return (lg_u64)__double_as_longlong(y) & 0x000FFFFFFFFFFFFFull;
}
__device__ __forceinline__ Weigh lg_weigher(float top, float T) { return { (double)top, T > 0 ? 1.0 / (double)T : 0.0 }; }

template <typename T>
__device__ __forceinline__ T lg_block_sum(T v, T *part) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    T all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) all += part[w];
    return all;
}
template <typename T>
__device__ __forceinline__ T lg_block_run(T v, T *part, T *total) {          // inclusive
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int o = 1; o < 64; o <<= 1) { const T u = __shfl_up(v, o); if (lane >= o) v += u; }
    __syncthreads();
    if (lane == 63) part[wave] = v;
    __syncthreads();
    T before = 0, all = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) { const T p = part[w]; if (w < wave) before += p; all += p; }
    *total = all;
    return v + before;
}

// One workgroup, one row: the border by digits of the key (4 passes of 8 bits each for top-k and top-p), then the draw.
struct SampleLds { lg_u64 bin[256]; lg_u64 part[LG_SAMPLE_WG / 64]; uint32_t key; int idx; lg_u64 rest; };

// The key at which a running sum from the largest key down reaches `want` (1..sum of all), among the tokens in question with keys >= low (of key `low`
// itself the first `ties` count); *before = the sum of the tokens with larger keys.  BY_COUNT: every token counts 1, else its weight.
template <bool BY_COUNT>
__device__ uint32_t lg_border(const SampleArgs &a, const float *row, const Weigh &wg, uint32_t low, int ties, lg_u64 want, lg_u64 *before, SampleLds &s) {
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

__device__ void lg_sample_row(const SampleArgs &a, int r, SampleLds &s) {
    const float *row = a.logits + r * a.stride;
    const SampleRow p = a.params[r];
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
    const Weigh wg = lg_weigher(lg_unkey(best), p.temperature);
    uint32_t cut = 0; int ties = 0;                 // kept: keys > cut, and the first `ties` of those with it
    lg_u64 W = 0; unsigned count = 0;
    for (int i = t; i < n; i += LG_SAMPLE_WG) { const lg_u64 w = lg_weigh(wg, row[i]); W += w; count += w != 0; }
    W = lg_block_sum(W, s.part);
    count = (unsigned)lg_block_sum((lg_u64)count, s.part);
    if (p.top_k > 0 && (unsigned)p.top_k < count) {
        lg_u64 before;
        cut = lg_border<true>(a, row, wg, 0, 0, (lg_u64)p.top_k, &before, s);
        ties = (int)(p.top_k - before);
        lg_u64 sum = 0;
        for (int i = t; i < n; i += LG_SAMPLE_WG) if (lg_key(row[i]) > cut) sum += lg_weigh(wg, row[i]);
        W = lg_block_sum(sum, s.part) + (lg_u64)ties * lg_weigh(wg, lg_unkey(cut));
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
    S = lg_block_sum(S, s.part) + (lg_u64)ties * wcut;
    count = (unsigned)lg_block_sum((lg_u64)count, s.part) + ties;
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
        if (cut) { const int mine = k == cut, rank = tied + (int)lg_block_run((lg_u64)mine, s.part, &all_ties) - mine; if (mine && rank >= ties) w = 0; }
        const lg_u64 upto = run + lg_block_run(w, s.part, &all);
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
#define LG_SAMPLE_SLICE   64                     // groups of a workgroup of the two passes after it
#define LG_SAMPLE_BINS    2048
#define LG_SAMPLE_CAND    4096                   // candidates that a row may have
#define LG_SAMPLE_SMALL_K 512                    // top-k up to which the groups' maxima bound the candidates well: with 1024 groups the tokens not below the
                                                 // k-th largest maximum are 1.15 k at k = 256 and 1.39 k at 512 where large logits lie anywhere in the row
#define LG_SAMPLE_SLACK   2048                   // the estimated sum of a row's bins is trusted to 1 / 2048: four times what the comment at lg_k_sample_bins allows
#define LG_SAMPLE_REACH   31.5                   // (max - l) / T beyond which a weight is 0

struct SampleWork {                     // per row, in working memory
    uint32_t *gmax;                     // [groups] keys
    float *smin;                        // [workgroups of lg_k_sample_max] smallest logit above -inf
    lg_u64 *mass; uint32_t *count;      // [LG_SAMPLE_BINS]
    lg_u64 *gsum;                       // [groups]
    lg_u64 *part;                       // [slices][3]: sum above the candidates, sum that top-p goes by (without the candidates), tokens kept above them
    uint32_t *ncand; lg_u64 *cand;      // [LG_SAMPLE_CAND] ~key << 32 | index
};
struct SampleGeo { int groups, maxes, slices; size_t gmax, smin, mass, count, gsum, part, ncand, cand, row; };
__host__ __device__ inline size_t lg_up64(size_t n) { return (n + 63) & ~(size_t)63; }
__host__ __device__ inline SampleGeo lg_sample_geo(int n_vocab) {
    SampleGeo g;
    g.groups = (n_vocab + LG_SAMPLE_GROUP - 1) / LG_SAMPLE_GROUP;
    g.maxes = (g.groups + 15) / 16;
    g.slices = (g.groups + LG_SAMPLE_SLICE - 1) / LG_SAMPLE_SLICE;
    size_t at = 0;
    g.gmax = at;  at += lg_up64((size_t)g.groups * 4);
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
    return { (uint32_t *)(p + g.gmax), (float *)(p + g.smin), (lg_u64 *)(p + g.mass), (uint32_t *)(p + g.count), (lg_u64 *)(p + g.gsum), (lg_u64 *)(p + g.part),
             (uint32_t *)(p + g.ncand), (lg_u64 *)(p + g.cand) };
}
// The first largest; a small top-k; no top-k and no top-p; a border to be found; a temperature so small that the estimates' f32 does not hold 1 / T
enum { LG_ROW_FIRST, LG_ROW_SMALL, LG_ROW_FREE, LG_ROW_BORDER, LG_ROW_ALONE };
__device__ __forceinline__ int lg_row_kind(const SampleRow &p, int n_vocab) {
    if (!(p.temperature > 0)) return LG_ROW_FIRST;
    const bool k = p.top_k > 0 && p.top_k < n_vocab;
    if (k && p.top_k <= LG_SAMPLE_SMALL_K) return LG_ROW_SMALL;
    if (!(p.temperature > 1e-20f)) return LG_ROW_ALONE;
    return k || p.top_p < 1 ? LG_ROW_BORDER : LG_ROW_FREE;
}
__device__ __forceinline__ lg_u64 lg_least(const SampleRow &p) {      // the smallest weight that min-p keeps
    if (!(p.min_p > 0)) return 1;
    const double m = __builtin_ceil((double)p.min_p * LG_SAMPLE_ONE);
    return m >= 1 ? m < LG_SAMPLE_ONE ? (lg_u64)m : (lg_u64)LG_SAMPLE_ONE : 1;
}
// Four tokens of a lane in group `grp`; -inf behind the row's end.  VEC: rows aligned to 16 bytes
template <bool VEC>
__device__ __forceinline__ void lg_load4(const float *row, int n, int grp, float (&l)[4]) {
    const int i = grp * LG_SAMPLE_GROUP + (threadIdx.x & 63) * 4;
    if (VEC && i + 3 < n) { const float4 x = *(const float4 *)(row + i); l[0] = x.x; l[1] = x.y; l[2] = x.z; l[3] = x.w; }
    else
        #pragma unroll
        for (int j = 0; j < 4; ++j) l[j] = i + j < n ? row[i + j] : -INFINITY;
}

template <bool VEC>
__global__ __launch_bounds__(LG_SAMPLE_MAX_WG) void lg_k_sample_max(SampleArgs a, char *base) {
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const int r = blockIdx.x / g.maxes, part = blockIdx.x % g.maxes, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const SampleWork w = lg_sample_work(base, g, r);
    const float *row = a.logits + r * a.stride;
    __shared__ float s_min[LG_SAMPLE_MAX_WG / 64];
    float l[4][4], least = INFINITY;
    #pragma unroll
    for (int j = 0; j < 4; ++j) lg_load4<VEC>(row, a.n_vocab, part * 16 + wave * 4 + j, l[j]);
    // the bins of the row are cleared on the way
    for (int i = part * LG_SAMPLE_MAX_WG + threadIdx.x; i < LG_SAMPLE_BINS; i += g.maxes * LG_SAMPLE_MAX_WG) { w.mass[i] = 0; w.count[i] = 0; }
    if (part == 0 && threadIdx.x == 0) *w.ncand = 0;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        float m = -INFINITY;
        #pragma unroll
        for (int i = 0; i < 4; ++i) { m = fmaxf(m, l[j][i]); if (l[j][i] > -INFINITY) least = fminf(least, l[j][i]); }    // (fmaxf passes over NaN)
        for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        const int grp = part * 16 + wave * 4 + j;
        if (lane == 0 && grp < g.groups) w.gmax[grp] = lg_key(m);
    }
    for (int o = 1; o < 64; o <<= 1) least = fminf(least, __shfl_xor(least, o));
    if (lane == 0) s_min[wave] = least;
    __syncthreads();
    if (threadIdx.x == 0) w.smin[part] = fminf(fminf(s_min[0], s_min[1]), fminf(s_min[2], s_min[3]));
}

// The row's largest logit and the width of its bins, in every workgroup anew (1024 keys and 64 minima: less than a launch of their own)
struct SampleSpan { Weigh wg; float top, scale; bool none; };      // scale: bins per unit of logit
__device__ __forceinline__ SampleSpan lg_sample_span(const SampleRow &p, const SampleWork &w, const SampleGeo &g, uint32_t *s_key, float *s_min) {
    uint32_t key = 0; float least = INFINITY;
    for (int i = threadIdx.x; i < g.groups; i += LG_SAMPLE_WG) { const uint32_t k = w.gmax[i]; if (k > key) key = k; }
    for (int i = threadIdx.x; i < g.maxes; i += LG_SAMPLE_WG) least = fminf(least, w.smin[i]);
    for (int o = 1; o < 64; o <<= 1) { const uint32_t k = __shfl_xor((int)key, o); if (k > key) key = k; least = fminf(least, __shfl_xor(least, o)); }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { s_key[threadIdx.x >> 6] = key; s_min[threadIdx.x >> 6] = least; }
    __syncthreads();
    key = 0; least = INFINITY;
    for (int i = 0; i < LG_SAMPLE_WG / 64; ++i) { if (s_key[i] > key) key = s_key[i]; least = fminf(least, s_min[i]); }
    SampleSpan s;
    s.none = key == 0x007FFFFFu;
    s.top = lg_unkey(key);
    s.wg = lg_weigher(s.top, p.temperature);
    const float reach = (float)LG_SAMPLE_REACH * p.temperature, width = fminf(s.top - least, reach);
    s.scale = width > 0 && width < INFINITY ? (float)LG_SAMPLE_BINS / width : 0;      // (0: all in the first bin)
    return s;
}
// Monotone in the logit, also as rounded: a larger logit never has a larger bin
__device__ __forceinline__ int lg_sample_bin(const SampleSpan &s, float l) {
    const float b = (s.top - l) * s.scale;                                            // (top - l is NaN for two infinities: the first bin)
    return b >= 0 ? b < (float)(LG_SAMPLE_BINS - 1) ? (int)b : LG_SAMPLE_BINS - 1 : 0;
}

template <bool VEC>
__global__ __launch_bounds__(LG_SAMPLE_WG) void lg_k_sample_bins(SampleArgs a, char *base) {
    __shared__ lg_u64 mass[LG_SAMPLE_BINS];
    __shared__ uint32_t count[LG_SAMPLE_BINS], s_key[16];
    __shared__ float s_min[16];
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const int r = blockIdx.x / g.slices, slice = blockIdx.x % g.slices, wave = threadIdx.x >> 6;
    const SampleRow p = a.params[r];
    if (lg_row_kind(p, a.n_vocab) != LG_ROW_BORDER) return;
    const SampleWork w = lg_sample_work(base, g, r);
    const float *row = a.logits + r * a.stride;
    float l[4][4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) lg_load4<VEC>(row, a.n_vocab, slice * LG_SAMPLE_SLICE + j * 16 + wave, l[j]);
    for (int i = threadIdx.x; i < LG_SAMPLE_BINS; i += LG_SAMPLE_WG) { mass[i] = 0; count[i] = 0; }
    const SampleSpan s = lg_sample_span(p, w, g, s_key, s_min);                       // (its barriers are the clearing's too)
    if (s.none) return;
    const bool by_count = p.top_k > 0 && p.top_k < a.n_vocab, by_mass = p.top_p < 1;
    const float c = -(float)(1.0 / (double)p.temperature * 1.4426950408889634);
    #pragma unroll
    for (int j = 0; j < 4; ++j)
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = l[j][i], d = x == s.top ? 0.0f : s.top - x;
            const float e = d * c;                                                    // in base 2; a weight of 0 starts near -45
            if (!(e > -46.0f)) continue;                                              // (NaN too)
            if (e < -44.0f && !lg_weigh(s.wg, x)) continue;
            const int b = lg_sample_bin(s, x);
            // an estimate, to 2^-32 of the largest weight: 2^19 of them are within 2^-13 of their sum.  In whole numbers too: no order changes it
            if (by_mass) atomicAdd(&mass[b], (lg_u64)(uint32_t)(__builtin_amdgcn_exp2f(e + 31.0f) + 0.5f));
            if (by_count) atomicAdd(&count[b], 1u);
        }
    __syncthreads();
    for (int i = threadIdx.x; i < LG_SAMPLE_BINS; i += LG_SAMPLE_WG) {
        if (by_mass && mass[i]) atomicAdd(&w.mass[i], mass[i]);
        if (by_count && count[i]) atomicAdd(&w.count[i], count[i]);
    }
}

// The bins that can hold the border, from the row's estimates: the same in every workgroup of a row
struct SampleRange { int first, last, cut; uint32_t above; };        // top-p's border is in bins first..last, top-k's in bin cut (LG_SAMPLE_BINS: none), behind `above` tokens
struct SampleRangeLds { lg_u64 part[LG_SAMPLE_WG / 64]; SampleRange r; lg_u64 lo, hi; };
__device__ SampleRange lg_sample_range(const SampleArgs &a, const SampleRow &p, const SampleWork &w, SampleRangeLds &s) {
    constexpr int PT = LG_SAMPLE_BINS / LG_SAMPLE_WG;
    const int b0 = threadIdx.x * PT;
    const bool by_count = p.top_k > 0 && p.top_k < a.n_vocab, by_mass = p.top_p < 1;
    if (threadIdx.x == 0) s.r = { 0, LG_SAMPLE_BINS - 1, LG_SAMPLE_BINS, 0 };
    if (by_count) {
        lg_u64 c[PT], sum = 0, all;
        #pragma unroll
        for (int i = 0; i < PT; ++i) { c[i] = w.count[b0 + i]; sum += c[i]; }
        lg_u64 run = lg_block_run(sum, s.part, &all) - sum;
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            if (run < (lg_u64)p.top_k && run + c[i] >= (lg_u64)p.top_k) { s.r.cut = b0 + i; s.r.above = (uint32_t)run; }
            run += c[i];
        }
        __syncthreads();
    }
    if (by_mass) {
        __syncthreads();
        const int cut = s.r.cut;
        lg_u64 m[PT], sum = 0, all;
        #pragma unroll
        for (int i = 0; i < PT; ++i) { m[i] = w.mass[b0 + i]; sum += m[i]; }
        lg_u64 run = lg_block_run(sum, s.part, &all) - sum;
        const lg_u64 start = run;
        if (threadIdx.x == 0) { s.lo = all; s.hi = all; }
        __syncthreads();
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
        __syncthreads();
    } else if (threadIdx.x == 0) s.r.first = s.r.last = s.r.cut;
    __syncthreads();
    SampleRange q = s.r;
    if (q.last > q.cut) q.last = q.cut;
    __syncthreads();
    return q;
}

template <bool VEC>
__global__ __launch_bounds__(LG_SAMPLE_WG) void lg_k_sample_sums(SampleArgs a, char *base) {
    __shared__ uint32_t s_key[16];
    __shared__ float s_min[16];
    __shared__ SampleRangeLds s_range;
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const int r = blockIdx.x / g.slices, slice = blockIdx.x % g.slices, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const SampleRow p = a.params[r];
    const int kind = lg_row_kind(p, a.n_vocab);
    if (kind != LG_ROW_BORDER && kind != LG_ROW_FREE) return;
    const SampleWork w = lg_sample_work(base, g, r);
    const float *row = a.logits + r * a.stride;
    float l[4][4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) lg_load4<VEC>(row, a.n_vocab, slice * LG_SAMPLE_SLICE + j * 16 + wave, l[j]);
    const SampleSpan s = lg_sample_span(p, w, g, s_key, s_min);
    if (s.none) return;
    const bool border = kind == LG_ROW_BORDER, by_mass = border && p.top_p < 1;
    SampleRange q{ LG_SAMPLE_BINS, -1, LG_SAMPLE_BINS, 0 };
    if (border) q = lg_sample_range(a, p, w, s_range);
    const lg_u64 least = lg_least(p);
    const float c = -(float)(1.0 / (double)p.temperature * 1.4426950408889634);
    const float floor_ = !border && least > 1 ? __builtin_amdgcn_logf((float)least * 5.684341886080802e-14f) - 0.01f : -46.0f;       // (2^-44; in base 2)
    lg_u64 above = 0, total = 0, kept = 0;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        lg_u64 sum = 0;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = l[j][i], d = x == s.top ? 0.0f : s.top - x;
            lg_u64 wt = 0;
            bool cand = false;
            if (d * c > floor_) {
                const int b = border ? lg_sample_bin(s, x) : 0;
                cand = border && ((b >= q.first && b <= q.last) || b == q.cut);
                if (b < q.first || cand || (by_mass && b < q.cut)) wt = lg_weigh(s.wg, x);
                if (by_mass && b < q.cut) total += wt;
                if (b < q.first) { above += wt; if (wt >= least) { sum += wt; ++kept; } }
                cand = cand && wt;
            }
            if (border) {
                const unsigned long long all = __ballot(cand);
                if (all) {
                    uint32_t at = 0;
                    if (lane == 0) at = atomicAdd(w.ncand, (uint32_t)__popcll(all));
                    at = __shfl((int)at, 0) + (uint32_t)__popcll(all & ((1ull << lane) - 1));
                    if (cand && at < LG_SAMPLE_CAND)
                        w.cand[at] = (lg_u64)~lg_key(x) << 32 | (uint32_t)((slice * LG_SAMPLE_SLICE + j * 16 + wave) * LG_SAMPLE_GROUP + lane * 4 + i);
                }
            }
        }
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
        const int grp = slice * LG_SAMPLE_SLICE + j * 16 + wave;
        if (lane == 0 && grp < g.groups) w.gsum[grp] = sum;
    }
    above = lg_block_sum(above, s_range.part);
    total = lg_block_sum(total, s_range.part);
    kept = lg_block_sum(kept, s_range.part);
    if (threadIdx.x == 0) { w.part[slice * 3] = above; w.part[slice * 3 + 1] = total; w.part[slice * 3 + 2] = kept; }
}

// LDS of n words sorted, smallest first; padded to a power of two with the largest
__device__ void lg_sample_sort(lg_u64 *v, int n) {
    int m = 64;
    while (m < n) m <<= 1;
    for (int i = n + threadIdx.x; i < m; i += LG_SAMPLE_WG) v[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= m; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            for (int t = threadIdx.x; t < m / 2; t += LG_SAMPLE_WG) {
                const int i = (t & ~(j - 1)) * 2 + (t & (j - 1));
                const lg_u64 x = v[i], y = v[i + j];
                if ((x > y) == !(i & k)) { v[i] = y; v[i + j] = x; }
            }
            __syncthreads();
        }
}

struct SampleFinishLds {
    lg_u64 cand[LG_SAMPLE_CAND], sum[LG_SAMPLE_GROUPS], part[LG_SAMPLE_WG / 64], weight, rest;
    uint32_t s_key[16]; float s_min[16];
    uint32_t n, bin[1024];
    int at, idx, before;
    SampleRangeLds range;
    SampleLds alone;
};
// Whole rows of up to LG_SAMPLE_CAND tokens (WHOLE: no launch came before), or what the launches before left of longer ones
template <bool VEC, bool WHOLE>
__global__ __launch_bounds__(LG_SAMPLE_WG) void lg_k_sample_finish(SampleArgs a, char *base) {
    __shared__ SampleFinishLds s;
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, n_vocab = a.n_vocab;
    const SampleRow p = a.params[r];
    const float *row = a.logits + r * a.stride;
    const SampleGeo g = lg_sample_geo(n_vocab);
    const SampleWork w = WHOLE ? SampleWork{} : lg_sample_work(base, g, r);
    const int kind = lg_row_kind(p, n_vocab);
    const lg_u64 least = lg_least(p);
    auto answer = [&](int tok, double prob, int kept) {
        a.tok[r] = tok;
        if (a.prob) a.prob[r] = (float)prob;
        if (a.kept) a.kept[r] = kept;
    };
    if (!WHOLE && kind == LG_ROW_ALONE) { lg_sample_row(a, r, s.alone); return; }
    int n = 0;                                               // candidates, sorted: larger logit first, then lower index
    lg_u64 above = 0, total = 0;                             // sum of the tokens above them; what top-p goes by, as far as it is not theirs
    int limit = -1, open = 0;                                // candidates from `limit` on are beyond top-k; those before `open` continue the tokens above
    int kept = 0;
    Weigh wg;
    if (WHOLE) {
        for (int i = t; i < n_vocab; i += LG_SAMPLE_WG) s.cand[i] = (lg_u64)~lg_key(row[i]) << 32 | (uint32_t)i;
        n = n_vocab;
        lg_sample_sort(s.cand, n);
        const uint32_t best = ~(uint32_t)(s.cand[0] >> 32);
        if (best == 0x007FFFFFu) { if (t == 0) answer(-1, 0, 0); return; }
        if (kind == LG_ROW_FIRST) { if (t == 0) answer((int)(uint32_t)s.cand[0], 1, 1); return; }
        wg = lg_weigher(lg_unkey(best), p.temperature);
        // those with a weight are a prefix
        lg_u64 mine = 0;
        for (int i = t; i < n; i += LG_SAMPLE_WG) mine += lg_weigh(wg, lg_unkey(~(uint32_t)(s.cand[i] >> 32))) != 0;
        n = (int)lg_block_sum(mine, s.part);
        limit = p.top_k > 0 && p.top_k < n ? p.top_k : n;
        open = n;
    } else {
        const SampleSpan span = lg_sample_span(p, w, g, s.s_key, s.s_min);
        if (span.none) { if (t == 0) answer(-1, 0, 0); return; }
        wg = span.wg;
        const uint32_t best = lg_key(span.top);
        if (kind == LG_ROW_FIRST) {
            if (t == 0) s.at = n_vocab;
            __syncthreads();
            for (int i = t; i < g.groups; i += LG_SAMPLE_WG) if (w.gmax[i] == best) { atomicMin(&s.at, i); break; }
            __syncthreads();
            if (wave == 0) {
                float l[4];
                lg_load4<VEC>(row, n_vocab, s.at, l);
                int first = 4;
                #pragma unroll
                for (int i = 3; i >= 0; --i) if (lg_key(l[i]) == best) first = i;
                const unsigned long long any = __ballot(first < 4);
                if (any && lane == (int)__builtin_ctzll(any)) answer(s.at * LG_SAMPLE_GROUP + lane * 4 + first, 1, 1);
            }
            return;
        }
        if (kind == LG_ROW_SMALL) {
            // a logit that at least top_k groups reach: the lower edge of one of 1024 equal parts between the groups' smallest and largest maxima
            if (t == 0) { s.n = 0; s.idx = 0x7FFFFFFF; }
            s.bin[t] = 0;
            __syncthreads();
            uint32_t low = 0xFFFFFFFFu, key[LG_SAMPLE_GROUPS / LG_SAMPLE_WG];
            #pragma unroll
            for (int u = 0; u < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++u) {
                const int i = t + u * LG_SAMPLE_WG;
                key[u] = i < g.groups ? w.gmax[i] : 0;
                if (key[u] > 0x007FFFFFu && key[u] < low) low = key[u];
            }
            for (int o = 1; o < 64; o <<= 1) { const uint32_t k = __shfl_xor((int)low, o); if (k < low) low = k; }
            if (lane == 0) s.s_key[wave] = low;
            __syncthreads();
            for (int i = 0; i < LG_SAMPLE_WG / 64; ++i) if (s.s_key[i] < low) low = s.s_key[i];
            const int shift = best - low >= 1024 ? 32 - __builtin_clz(best - low) - 10 : 0;
            #pragma unroll
            for (int u = 0; u < LG_SAMPLE_GROUPS / LG_SAMPLE_WG; ++u) if (key[u] >= low && key[u] > 0x007FFFFFu) atomicAdd(&s.bin[(key[u] - low) >> shift], 1u);
            __syncthreads();
            lg_u64 all;
            const uint32_t mine = s.bin[1023 - t];
            const lg_u64 run = lg_block_run((lg_u64)mine, s.part, &all);
            if (run >= (lg_u64)p.top_k && run - mine < (lg_u64)p.top_k) s.idx = 1023 - t;
            __syncthreads();
            const uint32_t from = all >= (lg_u64)p.top_k ? low + ((uint32_t)s.idx << shift) : 0;        // (fewer groups than top_k: every token)
            for (int grp = wave; grp < g.groups; grp += LG_SAMPLE_WG / 64) {
                if (w.gmax[grp] < from || w.gmax[grp] == 0x007FFFFFu) continue;
                float l[4];
                lg_load4<VEC>(row, n_vocab, grp, l);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t k = lg_key(l[i]);
                    if (k < from || !lg_weigh(wg, l[i])) continue;
                    const uint32_t at = atomicAdd(&s.n, 1u);
                    if (at < LG_SAMPLE_CAND) s.cand[at] = (lg_u64)~k << 32 | (uint32_t)(grp * LG_SAMPLE_GROUP + lane * 4 + i);
                }
            }
            __syncthreads();
            n = (int)s.n;
            if (n > LG_SAMPLE_CAND) { __syncthreads(); lg_sample_row(a, r, s.alone); return; }
            lg_sample_sort(s.cand, n);
            limit = p.top_k < n ? p.top_k : n;
            open = n;
        } else {
            SampleRange q{ LG_SAMPLE_BINS, -1, LG_SAMPLE_BINS, 0 };
            lg_u64 part[3] = { 0, 0, 0 };
            for (int i = t; i < g.slices; i += LG_SAMPLE_WG)
                #pragma unroll
                for (int u = 0; u < 3; ++u) part[u] += w.part[i * 3 + u];
            above = lg_block_sum(part[0], s.part);
            total = lg_block_sum(part[1], s.part);
            kept = (int)lg_block_sum(part[2], s.part);
            for (int i = t; i < LG_SAMPLE_GROUPS; i += LG_SAMPLE_WG) s.sum[i] = i < g.groups ? w.gsum[i] : 0;
            if (kind == LG_ROW_BORDER) {
                q = lg_sample_range(a, p, w, s.range);
                const uint32_t found = *w.ncand;
                if (found > LG_SAMPLE_CAND) { lg_sample_row(a, r, s.alone); return; }
                n = (int)found;
                for (int i = t; i < n; i += LG_SAMPLE_WG) s.cand[i] = w.cand[i];
                __syncthreads();
                lg_sample_sort(s.cand, n);
                lg_u64 mine = 0;
                for (int i = t; i < n; i += LG_SAMPLE_WG) mine += lg_sample_bin(span, lg_unkey(~(uint32_t)(s.cand[i] >> 32))) < q.cut;
                const int i0 = (int)lg_block_sum(mine, s.part);
                limit = q.cut < LG_SAMPLE_BINS ? i0 + p.top_k - (int)q.above : n;
                open = q.cut < LG_SAMPLE_BINS && q.last < q.cut - 1 ? i0 : n;
                if (limit > n) { lg_sample_row(a, r, s.alone); return; }
                if (q.cut < LG_SAMPLE_BINS) {
                    lg_u64 v = 0;
                    for (int i = i0 + t; i < limit; i += LG_SAMPLE_WG) v += lg_weigh(wg, lg_unkey(~(uint32_t)(s.cand[i] >> 32)));
                    total += lg_block_sum(v, s.part);
                }
            } else limit = 0;
        }
    }
    __syncthreads();
    // the border among the candidates: this thread's are 4 in a row
    constexpr int PT = LG_SAMPLE_CAND / LG_SAMPLE_WG;
    lg_u64 wt[PT], sum = 0, all;
    #pragma unroll
    for (int i = 0; i < PT; ++i) { const int at = t * PT + i; wt[i] = at < limit ? lg_weigh(wg, lg_unkey(~(uint32_t)(s.cand[at] >> 32))) : 0; sum += wt[i]; }
    int keep = limit;                                        // candidates that stay
    if (p.top_p < 1 && kind != LG_ROW_FREE) {
        lg_u64 run = above + lg_block_run(sum, s.part, &all) - sum;
        const lg_u64 W = WHOLE || kind == LG_ROW_SMALL ? all : total;
        const double want_d = __builtin_ceil((double)p.top_p * (double)W);
        const lg_u64 want = want_d >= 1 ? (lg_u64)want_d < W ? (lg_u64)want_d : W : 1;
        if (t == 0) s.before = -1;
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            if (wt[i] && run < want && run + wt[i] >= want) s.before = t * PT + i;
            run += wt[i];
        }
        __syncthreads();
        keep = s.before + 1;
        if (above >= want || keep == 0 || keep > open) { __syncthreads(); lg_sample_row(a, r, s.alone); return; }
    }
    const lg_u64 last = keep ? s.cand[keep - 1] : ~0ull;     // tokens up to this one stay
    lg_u64 S = 0, mine = 0;
    #pragma unroll
    for (int i = 0; i < PT; ++i) {
        const int at = t * PT + i;
        if (at >= keep || wt[i] < least) wt[i] = 0;
        if (wt[i]) { S += wt[i]; ++mine; }
    }
    kept += (int)lg_block_sum(mine, s.part);
    const float u = a.u[r];
    auto target_of = [&](lg_u64 S_) {
        lg_u64 x = u > 0 ? (lg_u64)__builtin_floor((u < 1 ? (double)u : 1.0) * (double)S_) : 0;
        return x > S_ - 1 ? S_ - 1 : x;
    };
    if (WHOLE || kind == LG_ROW_SMALL) {
        S = lg_block_sum(S, s.part);
        const lg_u64 target = target_of(S);
        if (!WHOLE) {
            // index order: index << 32 | key
            __syncthreads();
            for (int i = t; i < keep; i += LG_SAMPLE_WG) { const lg_u64 c = s.cand[i]; s.cand[i] = c << 32 | (uint32_t)~(c >> 32); }
            lg_sample_sort(s.cand, keep);
        }
        sum = 0;
        uint32_t idx[PT];
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int at = t * PT + i;
            wt[i] = 0;
            if (WHOLE) {
                idx[i] = at;
                if (at < n_vocab) { const uint32_t k = lg_key(row[at]); if (((lg_u64)~k << 32 | (uint32_t)at) <= last) wt[i] = lg_weigh(wg, lg_unkey(k)); }
            } else if (at < keep) { idx[i] = (uint32_t)(s.cand[at] >> 32); wt[i] = lg_weigh(wg, lg_unkey((uint32_t)s.cand[at])); }
            if (wt[i] < least) wt[i] = 0;
            sum += wt[i];
        }
        lg_u64 run = lg_block_run(sum, s.part, &all) - sum;
        #pragma unroll
        for (int i = 0; i < PT; ++i) {
            if (wt[i] && run <= target && run + wt[i] > target) answer((int)idx[i], (double)wt[i] / (double)S, kept);
            run += wt[i];
        }
        return;
    }
    // the groups' sums with the candidates that stay, the group of the draw, and the token in it
    #pragma unroll
    for (int i = 0; i < PT; ++i) if (wt[i]) atomicAdd(&s.sum[(uint32_t)s.cand[t * PT + i] / LG_SAMPLE_GROUP], wt[i]);
    __syncthreads();
    constexpr int GT = LG_SAMPLE_GROUPS / LG_SAMPLE_WG;
    lg_u64 gs[GT];
    sum = 0;
    #pragma unroll
    for (int i = 0; i < GT; ++i) { gs[i] = s.sum[t * GT + i]; sum += gs[i]; }
    lg_u64 run = lg_block_run(sum, s.part, &all) - sum;
    S = all;
    const lg_u64 target = target_of(S);
    #pragma unroll
    for (int i = 0; i < GT; ++i) {
        if (run <= target && run + gs[i] > target) { s.at = t * GT + i; s.rest = target - run; }
        run += gs[i];
    }
    __syncthreads();
    if (wave == 0) {
        float l[4];
        lg_load4<VEC>(row, n_vocab, s.at, l);
        sum = 0;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t k = lg_key(l[i]), idx = s.at * LG_SAMPLE_GROUP + lane * 4 + i;
            wt[i] = kind == LG_ROW_FREE || ((lg_u64)~k << 32 | idx) <= last ? lg_weigh(wg, l[i]) : 0;
            if (wt[i] < least) wt[i] = 0;
            sum += wt[i];
        }
        lg_u64 at = sum;
        for (int o = 1; o < 64; o <<= 1) { const lg_u64 v = __shfl_up(at, o); if (lane >= o) at += v; }
        at -= sum;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (wt[i] && at <= s.rest && at + wt[i] > s.rest) answer(s.at * LG_SAMPLE_GROUP + lane * 4 + i, (double)wt[i] / (double)S, kept);
            at += wt[i];
        }
    }
}
