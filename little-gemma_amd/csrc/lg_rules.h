// lg_rules.h — what logits are held to ahead of sampling: penalties for the tokens of a text, biases, and the tokens that a grammar allows.
#pragma once

#include "lg_block.h"

#define LG_RULES_VOCAB 524288
#define LG_RULES_WG 256
#define LG_RULES_AHEAD 4
#define LG_RULES_SLICE 2048         // tokens of a workgroup: their counts lie in LDS

struct RulesPenalty { float repetition, presence, frequency; int32_t prompt; };       // struct lg_hip_penalty
struct RulesArgs {
    const float *logits; long long stride;
    float *out; long long out_stride;
    const int32_t *seq;
    const RulesPenalty *penalty;
    const int32_t *hist, *hist_len; long long hist_stride;
    const lg_u64 *tree_mask; const int32_t *tree_start, *tree_tok;
    const int32_t *bias_start, *bias_tok; const float *bias;
    const uint32_t *allow; const int32_t *allow_row; long long allow_stride;
    int rows, n_vocab, n_seq, n_bias, n_allow;
};

// A workgroup takes SLICE tokens of one row's vocabulary.  It asks for their logits, goes over the whole text of the row's sequence and counts its own tokens in LDS (whole numbers:
// the order does not matter), then writes the slice.  Bound by memory where rows are many: 8 bytes a logit; a text is read once for every slice of every row, but from the L2.
// 64 rows of 262144 with penalties, biases and sets, 135 MB: 28 us, 4.8 TB/s; one row with a text of 3001 tokens 4.8 us, the launch and the chain of parameters, text and logits.  Slices of 2048 at all sizes: of 4096 64
// rows took 34.6, one row 5.1.  Rows that are not aligned to 16 bytes (VEC false): 39.6 and 5.2.
// Long texts take longer, for each slice goes over all of its row's text: one row with 32768 and 100000 tokens 10.9 and 25.4 us; 64 rows with texts of their own, penalties alone, 3001, 32768 and 100000 tokens 23.0, 36.6
// and 62.4.
// Logits that a rule changes are computed in 64 bits and rounded once.
template <bool VEC>
__global__ __launch_bounds__(LG_RULES_WG) void lg_k_rules(RulesArgs a) {
    extern __shared__ uint32_t s_word[];            // [SLICE] counts: bit 31 a token of the text, below it how often it was generated; [SLICE] 1 + the bias of a token, where there are any
    constexpr uint32_t SEEN = 1u << 31;
    constexpr int SLICE = LG_RULES_SLICE, EACH = SLICE / (4 * LG_RULES_WG);
    const int t = threadIdx.x, row = blockIdx.y, base = blockIdx.x * SLICE;
    const int size = a.n_vocab - base < SLICE ? a.n_vocab - base : SLICE;
    // (logits first: what is asked for later arrives later)
    const float *in = a.logits + row * a.stride + base;
    float *out = a.out + row * a.out_stride + base;
    float4 x[EACH];
    #pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int i = (k * LG_RULES_WG + t) * 4;
        if (VEC && i + 4 <= size) x[k] = *(const float4 *)(in + i);
        else { float *v = (float *)&x[k]; for (int j = 0; j < 4; ++j) v[j] = i + j < size ? in[i + j] : 0.0f; }
    }
    const int s = a.seq ? a.seq[row] : row;
    const bool named = s >= 0 && s < a.n_seq;
    RulesPenalty p = { 1.0f, 0.0f, 0.0f, 0 };
    if (a.penalty && named) p = a.penalty[s];
    if (!(p.repetition > 0)) p.repetition = 1.0f;             // (NaN as well)
    if (p.presence != p.presence) p.presence = 0;
    if (p.frequency != p.frequency) p.frequency = 0;
    const bool text = p.repetition != 1.0f || p.presence != 0 || p.frequency != 0;
    int b0 = 0, b1 = 0;
    if (a.bias_start && named) {
        b0 = a.bias_start[s]; b1 = a.bias_start[s + 1];
        if (b0 < 0) b0 = 0;
        if (b1 > a.n_bias) b1 = a.n_bias;
    }
    const bool biased = b1 > b0;
    const int grammar = a.n_allow ? a.allow_row ? a.allow_row[row] : row : -1;
    const uint32_t *allow = grammar >= 0 && grammar < a.n_allow ? a.allow + grammar * a.allow_stride : nullptr;
    if (in == out && !text && !biased && !allow) return;
    uint32_t *const s_bias = s_word + SLICE;
    if (text || biased) {
        #pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int i = (k * LG_RULES_WG + t) * 4;
            *(uint4 *)(s_word + i) = make_uint4(0, 0, 0, 0);
            if (biased) *(uint4 *)(s_bias + i) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        if (text && a.hist) {
            const int32_t *h = a.hist + s * a.hist_stride;
            int n = a.hist_len[s], prompt = p.prompt;
            if (n > a.hist_stride) n = (int)a.hist_stride;
            auto count = [&](int i, int tok) {
                const uint32_t at = (uint32_t)tok - (uint32_t)base;
                if (at < (uint32_t)size) { if (i < prompt) atomicOr(&s_word[at], SEEN); else atomicAdd(&s_word[at], 1u); }
            };
            const int head = (int)((16 - ((uintptr_t)h & 15)) & 15) / 4, lead = head < n ? head : n;
            if (t < lead) count(t, h[t]);
            // fours of tokens, LG_RULES_AHEAD of them asked for at once
            const int fours = (n - lead) / 4;
            typedef int32_t four __attribute__((ext_vector_type(4)));
            const four *const f = (const four *)(h + lead);
            for (int k0 = t; k0 < fours; k0 += LG_RULES_AHEAD * LG_RULES_WG) {
                four q[LG_RULES_AHEAD];
                #pragma unroll
                for (int k = 0; k < LG_RULES_AHEAD; ++k) q[k] = f[k0 + k * LG_RULES_WG < fours ? k0 + k * LG_RULES_WG : k0];
                #pragma unroll
                for (int k = 0; k < LG_RULES_AHEAD; ++k) {
                    const int x = k0 + k * LG_RULES_WG;
                    if (x < fours)
                        #pragma unroll
                        for (int j = 0; j < 4; ++j) count(lead + 4 * x + j, q[k][j]);
                }
            }
            const int end = lead + 4 * fours;
            if (end + t < n) count(end + t, h[end + t]);       // (up to three)
        }
        if (text && a.tree_mask && t < 64 && (a.tree_mask[row] >> t & 1)) {
            const long long at = (long long)a.tree_start[s] + t;
            if (at >= 0 && at < a.rows) {
                const uint32_t tok = (uint32_t)a.tree_tok[at] - (uint32_t)base;
                if (tok < (uint32_t)size) atomicAdd(&s_word[tok], 1u);
            }
        }
        for (int e = b0 + t; e < b1; e += LG_RULES_WG) {
            const uint32_t at = (uint32_t)a.bias_tok[e] - (uint32_t)base;
            if (at < (uint32_t)size) atomicMax(&s_bias[at], (uint32_t)e + 1);
        }
        __syncthreads();
    }
    #pragma unroll
    for (int k = 0; k < EACH; ++k) {
        const int i = (k * LG_RULES_WG + t) * 4;
        if (i >= size) continue;
        float *v = (float *)&x[k];
        if (text || biased) {
            const uint4 w = *(const uint4 *)(s_word + i), b = biased ? *(const uint4 *)(s_bias + i) : make_uint4(0, 0, 0, 0);
            const uint32_t ws[4] = { w.x, w.y, w.z, w.w }, bs[4] = { b.x, b.y, b.z, b.w };
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!(ws[j] | bs[j])) continue;
                double y = v[j];
                if (ws[j] && p.repetition != 1.0f) y = y > 0 ? y / (double)p.repetition : y * (double)p.repetition;
                const uint32_t made = ws[j] & ~SEEN;
                if (made) { y -= p.presence; if (p.frequency != 0) y -= (double)p.frequency * made; }
                if (bs[j]) y += a.bias[bs[j] - 1];
                v[j] = (float)y;
            }
        }
        if (allow) {
            const uint32_t bits = allow[(base + i) >> 5] >> (i & 31);
            #pragma unroll
            for (int j = 0; j < 4; ++j) if (!(bits >> j & 1)) v[j] = -INFINITY;
        }
        if (VEC && i + 4 <= size) *(float4 *)(out + i) = x[k];
        else for (int j = 0; j < 4; ++j) if (i + j < size) out[i + j] = v[j];
    }
}
