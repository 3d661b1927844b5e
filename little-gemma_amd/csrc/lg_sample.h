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

__global__ __launch_bounds__(LG_SAMPLE_WG) void lg_k_sample_row(SampleArgs a) {
    __shared__ SampleLds s;
    lg_sample_row(a, blockIdx.x, s);
}
