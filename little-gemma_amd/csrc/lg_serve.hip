// lg_serve.hip — the operators of a batched decode step behind include/lg_hip.h: pages of a shared KV cache, attention over them, sampling.
//
// Every entry takes device pointers of the caller, allocates nothing, launches on the caller's stream and returns without waiting: a stream under
// capture can take it.  What the host can see is checked here; what lies in device memory (lengths, page ids, slots) is checked by the kernels.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "../../include/lg_hip.h"
#include "lg_host.h"
#include "lg_pages.h"
#include "lg_sample.h"
#include "lg_tree.h"
#include "lg_share.h"
#include "lg_rules.h"

static_assert(LG_PLAN_BAD_LEN == LG_HIP_PLAN_BAD_LENGTH && LG_PLAN_NO_PAGES == LG_HIP_PLAN_NO_PAGES && LG_PLAN_NO_SLOTS == LG_HIP_PLAN_NO_SLOTS &&
              LG_PLAN_BAD_STACK == LG_HIP_PLAN_BAD_STACK && LG_PLAN_BAD_PAGE == LG_HIP_PLAN_BAD_PAGE, "status bits of a plan");
static_assert(sizeof(SampleRow) == sizeof(struct lg_hip_sampling), "parameters of a row");
static_assert(LG_TREE_BAD_ROWS == LG_HIP_TREE_BAD_ROWS && LG_TREE_BAD_PARENT == LG_HIP_TREE_BAD_PARENT && LG_TREE_BAD_LEN == LG_HIP_TREE_BAD_LENGTH, "status bits of a tree");
static_assert(LG_FORK_BAD_LEN == LG_HIP_FORK_BAD_LENGTH && LG_FORK_NO_PAGES == LG_HIP_FORK_NO_PAGES && LG_FORK_BAD_SOURCE == LG_HIP_FORK_BAD_SOURCE &&
              LG_FORK_BAD_STACK == LG_HIP_FORK_BAD_STACK && LG_FORK_BAD_PAGE == LG_HIP_FORK_BAD_PAGE && LG_FORK_BAD_SHARES == LG_HIP_FORK_BAD_SHARES, "status bits of a fork");
static_assert(sizeof(RulesPenalty) == sizeof(struct lg_hip_penalty), "penalties of a sequence");

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static int shift_of(int page_size) {                 // page_size = 1 << shift; -1: not served
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return -1;
    return __builtin_ctz((unsigned)page_size);
}
#define LG_MOST_GROUPS ((1 << 24) - 1)                // workgroups of 256 threads in a launch
static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// ---- plan -------------------------------------------------------------------------------------------------------
// Slots that the plan's one workgroup fills itself; more by a launch of their own.  In one launch and in two: 64 sequences with 2112 new tokens 5.8 and 7.5 us, with 8192 7.4 and 7.5,
// with 16384 10.1 and 7.5
#define LG_PLAN_APART 8192
extern "C" size_t lg_hip_paged_plan_workspace(int n_seq) { (void)n_seq; return 0; }

extern "C" int lg_hip_paged_plan(int n_seq, int page_size, int n_pages, int max_blocks, const int32_t *d_len_old, const int32_t *d_len_new,
                                 int32_t *d_table, int32_t *d_free, int32_t *d_n_free, int32_t *d_start, int32_t *d_slots, int n_slots,
                                 int32_t *d_status, void *d_work, size_t work_bytes, void *stream) {
    (void)d_work; (void)work_bytes;
    const int shift = shift_of(page_size);
    if (n_seq < 0 || n_seq > LG_PLAN_SEQS) return lg_fail(-2, "paged_plan: %d sequences (0..%d)", n_seq, LG_PLAN_SEQS);
    if (shift < 0) return lg_fail(-2, "paged_plan: pages of %d positions (a power of two of 16..256)", page_size);
    if (n_pages < 1 || (int64_t)n_pages * page_size > INT32_MAX || max_blocks < 1 || (int64_t)max_blocks * page_size > INT32_MAX)
        return lg_fail(-2, "paged_plan: %d pages and %d blocks of %d positions (slots and positions are 31 bits)", n_pages, max_blocks, page_size);
    if (n_slots < 0) return lg_fail(-2, "paged_plan: %d slots", n_slots);
    if (!d_free || !d_n_free || !d_start || !d_status || (n_seq && (!d_len_old || !d_len_new || !d_table)) || (n_slots && !d_slots))
        return lg_fail(-1, "paged_plan: null argument");
    PlanArgs a{ d_len_old, d_len_new, d_table, d_free, d_n_free, d_start, d_slots, d_status, n_seq, shift, n_pages, max_blocks, n_slots };
    hipStream_t st = (hipStream_t)stream;
    // four wavefronts where they have a thread for every sequence and token, for their barriers are shorter: 64 sequences, a token each, 3.6 us, with 1024 threads 4.4
    const bool apart = n_slots > LG_PLAN_APART;
    if (apart) a.slots = nullptr;
    if (n_seq <= 256 && n_slots <= 256) hipLaunchKernelGGL(lg_k_plan<256>, dim3(1), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(lg_k_plan<1024>, dim3(1), dim3(1024), 0, st, a);
    if (apart) {
        a.slots = d_slots;
        hipLaunchKernelGGL(lg_k_plan_slots, dim3((unsigned)(((int64_t)n_slots + 1023) / 1024)), dim3(256), 0, st, a);
    }
    LG_TRY(hipGetLastError());
    return 0;
}

// ---- pages ------------------------------------------------------------------------------------------------------
static int check_pages(const char *who, const struct lg_hip_pages *p, PageGeo *g) {
    if (!p || !p->k || !p->v) return lg_fail(-1, "%s: null argument", who);
    const int shift = shift_of(p->page_size);
    if (shift < 0) return lg_fail(-2, "%s: pages of %d positions (a power of two of 16..256)", who, p->page_size);
    if (p->n_pages < 1 || (int64_t)p->n_pages * p->page_size > INT32_MAX) return lg_fail(-2, "%s: %d pages of %d positions (slots are 31 bits)", who, p->n_pages, p->page_size);
    const int hd = p->head_dim;
    if (p->n_head_kv < 1 || p->n_head_kv > 1024 || (hd != 64 && hd != 128 && hd != 256 && hd != 512))
        return lg_fail(-2, "%s: %d key heads of %d (heads of 64, 128, 256 or 512)", who, p->n_head_kv, hd);
    const int64_t most = INT64_C(1) << 40;           // products of strides and page ids stay in 64 bits
    if (p->row_stride < (int64_t)p->n_head_kv * hd || p->row_stride % 8 || p->row_stride > most || p->page_stride < p->row_stride * p->page_size ||
        p->page_stride % 8 || p->page_stride > most / p->n_pages * 1024)
        return lg_fail(-2, "%s: strides of %lld values a row and %lld a page (multiples of 8 that hold %d rows of %d)", who, (long long)p->row_stride,
                       (long long)p->page_stride, p->page_size, p->n_head_kv * hd);
    if (!aligned16(p->k) || !aligned16(p->v)) return lg_fail(-2, "%s: pages that are not aligned to 16 bytes", who);
    *g = PageGeo{ p->k, p->v, p->row_stride, p->page_stride, p->n_pages, shift };
    return 0;
}

// ---- write ------------------------------------------------------------------------------------------------------
extern "C" int lg_hip_paged_write(const struct lg_hip_pages *p, const float *d_k, const float *d_v, int64_t stride, const int32_t *d_slots, int n_tok,
                                  void *stream) {
    PageGeo g;
    const int rc = check_pages("paged_write", p, &g);
    if (rc) return rc;
    if (n_tok < 0) return lg_fail(-2, "paged_write: %d tokens", n_tok);
    if (n_tok == 0) return 0;
    if (!d_k || !d_v || !d_slots) return lg_fail(-1, "paged_write: null argument");
    const int width = p->n_head_kv * p->head_dim;
    if (stride < width || stride % 4 || !aligned16(d_k) || !aligned16(d_v))
        return lg_fail(-2, "paged_write: rows of %d values, %lld apart (aligned to 16 bytes)", width, (long long)stride);
    const int64_t groups = ((int64_t)n_tok * (width / 4) + 255) / 256;
    if (groups > LG_MOST_GROUPS) return lg_fail(-2, "paged_write: %d tokens of %d values in one call", n_tok, width);
    hipLaunchKernelGGL(lg_k_page_write, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, g, d_k, d_v, (long long)stride, d_slots, n_tok, width / 8);
    LG_TRY(hipGetLastError());
    return 0;
}

// ---- attend -----------------------------------------------------------------------------------------------------
// Workgroups of lg_k_page_attn at a time: lg_pa_per_simd on each of 256 compute units
static int slots_of(int hd) { return 256 * lg_pa_per_simd(hd); }
// Sequences of up to so many tiles are left whole where none is longer: the cut, the partials and the launch that joins them take longer than what splits save, the more so where
// the sequences' key heads keep the chip at work by themselves.  Whole and in splits, us: one sequence of 512 keys, heads of 64 7.1 and 8.1, 128 8.0 and 9.0, 256 12.7 and 10.3 (320
// keys: 9.7 and 10.2), 512 24.8 and 16.1 (192: 14.0 and 15.9).  Two key heads, all sequences as long as the longest / of all lengths up to it: 64 sequences of 1024, heads of 128 13.5 and
// 19.3 / 13.1 and 13.6; of 768, heads of 256 19.9 and 26.0 / 18.9 and 18.1; 128 of 2047, heads of 128 39.6 and 48.9 / 26.7 and 32.5, heads of 256 91.1 and 113 / 52.7 and 53.1;
// 200 of 2047, heads of 256 151 and 169 / 108 and 95.  One key head of 512: 128 of 512 28.1 and 36.4 / 26.7 and 26.1.
// A limit holds for all numbers of units in its tier and lies where splits begin to gain for some of them; for others, lengths above it take the slower side.  One key head of 512, 1024
// keys (limit 512): 128 sequences 49.8 and 57.7 / 44.5 and 35.0, but 200 75.7 and 94.1 / 47.1 and 51.7.  Two heads of 256, 2047 keys (limit 1536): 150 sequences 138 and 126 / 94.4 and
// 67.6, but the 128 above
static int alone_of(int hd, int64_t units) {
    const int tier = units < 128 ? 0 : units < 256 ? 1 : 2;
    static const int tiles[4][3] = { { 20, 32, 64 }, { 18, 32, 64 }, { 11, 24, 48 }, { 7, 16, 32 } };          // heads of 64, 128, 256, 512
    return tiles[hd == 64 ? 0 : hd == 128 ? 1 : hd == 256 ? 2 : 3][tier];
}
struct AttnCut { int64_t splits, tiles; bool join; int least; };        // tiles: of all sequences, at most
// Splits of all sequences together, at most.  lg_pa_split_tiles makes the full ones of a key head slots / n_head_kv or fewer for every round, the rounds one or 2 units / slots rounded
// up, where splits of min_tiles tiles to LG_PA_CHUNK keys allow; every sequence has one that is not full besides
static AttnCut cut_of(int n_seq, int n_head_kv, int hd, int max_len, int window) {
    // (a window need not start with a tile)
    const int64_t span = window > 0 && window < max_len ? (int64_t)window + LG_PA_TILE - 1 : max_len, tiles = (span + LG_PA_TILE - 1) / LG_PA_TILE;
    const int alone = alone_of(hd, (int64_t)n_seq * n_head_kv), min_tiles = tiles <= alone ? alone : 4;
    const int64_t least = (tiles + min_tiles - 1) / min_tiles, slots = slots_of(hd), units = (int64_t)n_seq * n_head_kv, rounds = std::max<int64_t>(1, (units + slots / 2 - 1) / (slots / 2));
    const int64_t full = std::max<int64_t>(rounds * slots / n_head_kv, n_seq * tiles / (LG_PA_CHUNK / LG_PA_TILE));
    return { std::min<int64_t>(n_seq * std::max<int64_t>(least, 1), full + n_seq), n_seq * tiles, least > 1, min_tiles };
}
static bool attn_shape(int n_seq, int n_head, int n_head_kv, int hd, int max_len) {
    return n_seq >= 0 && n_head_kv >= 1 && n_head_kv <= 1024 && n_head >= 1 && n_head % n_head_kv == 0 && n_head / n_head_kv <= 8 &&
           (hd == 64 || hd == 128 || hd == 256 || hd == 512) && max_len >= 0 && max_len <= (1 << 30);
}
static size_t cut_bytes(int n_seq, const AttnCut &c) { return up256(((size_t)n_seq + 1 + (n_seq > LG_PA_LANES ? 1 + c.splits : 0)) * 4); }
extern "C" size_t lg_hip_paged_attention_workspace(int n_seq, int n_head, int n_head_kv, int hd, int max_len, int window) {
    if (!attn_shape(n_seq, n_head, n_head_kv, hd, max_len)) return 0;
    const AttnCut c = cut_of(n_seq, n_head_kv, hd, max_len, window);
    if (!c.join) return 0;
    const size_t slots = (size_t)c.splits * n_head;
    return cut_bytes(n_seq, c) + 2 * up256(slots * 4) + slots * hd * 4;
}

template <int HD>
static void launch_attn(const PageAttn &a, const AttnCut &c, hipStream_t st) {
    hipLaunchKernelGGL(lg_k_page_attn<HD>, dim3((unsigned)(c.splits * a.nkv)), dim3(LG_PA_WAVES * 64), 0, st, a);
    if (!c.join) return;
    // eight wavefronts to a head, or one where there are hundreds of heads (two are no faster)
    if (a.n_seq > LG_PA_LANES) hipLaunchKernelGGL((lg_k_page_merge<HD, 1, PageAttn>), dim3(a.H, a.n_seq), dim3(64), 0, st, a);
    else hipLaunchKernelGGL((lg_k_page_merge<HD, 8, PageAttn>), dim3(a.H, a.n_seq), dim3(512), 0, st, a);
}

extern "C" int lg_hip_paged_attention(const struct lg_hip_pages *p, const float *d_q, int64_t q_stride, int n_seq, int n_head, const int32_t *d_table,
                                      int max_blocks, const int32_t *d_len, int max_len, int window, float scale, float *d_out, int64_t out_stride,
                                      void *d_work, size_t work_bytes, void *stream) {
    PageGeo g;
    const int rc = check_pages("paged_attention", p, &g);
    if (rc) return rc;
    const int hd = p->head_dim;
    if (!attn_shape(n_seq, n_head, p->n_head_kv, hd, max_len))
        return lg_fail(-2, "paged_attention: %d sequences, %d query heads on %d key heads (at most 8 each), lengths up to %d", n_seq, n_head, p->n_head_kv, max_len);
    if (max_blocks < 1 || (int64_t)max_blocks * p->page_size > INT32_MAX) return lg_fail(-2, "paged_attention: %d blocks of %d positions", max_blocks, p->page_size);
    if (window < 0) return lg_fail(-2, "paged_attention: a window of %d", window);
    if (n_seq == 0) return 0;
    if (!d_q || !d_table || !d_len || !d_out) return lg_fail(-1, "paged_attention: null argument");
    const int64_t qd = (int64_t)n_head * hd;
    if (q_stride < qd || q_stride % 4 || !aligned16(d_q)) return lg_fail(-2, "paged_attention: query rows of %lld values, %lld apart (aligned to 16 bytes)", (long long)qd, (long long)q_stride);
    if (out_stride < qd || ((uintptr_t)d_out & 3)) return lg_fail(-2, "paged_attention: output rows of %lld values, %lld apart", (long long)qd, (long long)out_stride);
    const AttnCut c = cut_of(n_seq, p->n_head_kv, hd, max_len, window);
    // (sums over the sequences are 32 bits on the device, and so are a launch's threads)
    if (n_seq > LG_PA_SEQS || c.tiles > INT32_MAX || c.splits * n_head > LG_MOST_GROUPS)
        return lg_fail(-2, "paged_attention: %d sequences of %d heads in %lld splits in one call (at most %d sequences)", n_seq, n_head, (long long)c.splits, LG_PA_SEQS);
    const size_t need = lg_hip_paged_attention_workspace(n_seq, n_head, p->n_head_kv, hd, max_len, window);
    if (need && (!d_work || work_bytes < need || ((uintptr_t)d_work & 255)))
        return lg_fail(-2, "paged_attention: %zu bytes of working memory (aligned to 256), given %zu", need, d_work ? work_bytes : 0);
    const size_t part = up256((size_t)c.splits * n_head * 4);
    char *const w = need ? (char *)d_work + cut_bytes(n_seq, c) : nullptr;
    const PageAttn a{ g, d_q, (long long)q_stride, d_table, d_len, d_out, (long long)out_stride, (float *)w, need ? (float *)(w + part) : nullptr,
                      need ? (float *)(w + 2 * part) : nullptr, scale, need ? (int32_t *)d_work : nullptr, n_head, p->n_head_kv, n_seq, max_blocks, max_len, window, slots_of(hd), c.least };
    hipStream_t st = (hipStream_t)stream;
    if (c.join && n_seq > LG_PA_LANES) hipLaunchKernelGGL(lg_k_page_cut, dim3(1), dim3(LG_PC_WG), 0, st, a);
    switch (hd) {
        case 64:  launch_attn<64>(a, c, st); break;
        case 128: launch_attn<128>(a, c, st); break;
        case 256: launch_attn<256>(a, c, st); break;
        default:  launch_attn<512>(a, c, st); break;
    }
    LG_TRY(hipGetLastError());
    return 0;
}

// ---- sample -----------------------------------------------------------------------------------------------------
extern "C" size_t lg_hip_sample_workspace(int rows, int n_vocab) {
    if (rows < 0 || n_vocab <= LG_SAMPLE_WHOLE || n_vocab > LG_SAMPLE_VOCAB) return 0;
    return (size_t)rows * lg_sample_geo(n_vocab).row;
}

// Groups of 256 logits in a call from which on lg_k_sample_sums takes workgroups of 64 groups instead of 16, so that fewer read a row's bins again.  Top-p of rows of 262144, 16 groups
// and 64: 5 rows 32.3 and 34.2 us, 33 62.2 and 67.6, 48 73.7 and 73.0; top-k 5000 with it: 33 68.8 and 73.8, 64 96.3 and 94.4
#define LG_SAMPLE_WIDE 40960
template <bool VEC>
static void launch_sample(SampleArgs a, int rows, char *work, hipStream_t st) {
    if (!work) {
        if (a.n_vocab <= 4 * LG_SAMPLE_WG) hipLaunchKernelGGL((lg_k_sample_finish<VEC, true, 4>), dim3(rows), dim3(LG_SAMPLE_WG), 0, st, a, work);
        else hipLaunchKernelGGL((lg_k_sample_finish<VEC, true, LG_SAMPLE_WHOLE / LG_SAMPLE_WG>), dim3(rows), dim3(LG_SAMPLE_WG), 0, st, a, work);
        return;
    }
    const SampleGeo g = lg_sample_geo(a.n_vocab);
    const dim3 maxes((unsigned)g.maxes, rows), few((unsigned)(g.groups + 15) / 16, rows), many((unsigned)(g.groups + 63) / 64, rows);
    hipLaunchKernelGGL(lg_k_sample_max<VEC>, maxes, dim3(LG_SAMPLE_MAX_WG), 0, st, a, work);
    hipLaunchKernelGGL(lg_k_sample_bins<VEC>, many, dim3(LG_SAMPLE_WG), 0, st, a, work);
    const bool narrow = (int64_t)rows * g.groups < LG_SAMPLE_WIDE;
    a.slices = (int)(narrow ? few : many).x;
    if (narrow) hipLaunchKernelGGL((lg_k_sample_sums<VEC, 256>), few, dim3(256), 0, st, a, work);
    else hipLaunchKernelGGL((lg_k_sample_sums<VEC, 1024>), many, dim3(1024), 0, st, a, work);
    hipLaunchKernelGGL((lg_k_sample_finish<VEC, false, LG_SAMPLE_CAND / LG_SAMPLE_WG>), dim3(rows), dim3(LG_SAMPLE_WG), 0, st, a, work);
}

extern "C" int lg_hip_sample(const float *d_logits, int64_t stride, int rows, int n_vocab, const struct lg_hip_sampling *d_params, const float *d_u,
                             int32_t *d_tok, float *d_prob, int32_t *d_kept, void *d_work, size_t work_bytes, void *stream) {
    if (rows < 0 || rows > 65535) return lg_fail(-2, "sample: %d rows (0..65535)", rows);
    if (n_vocab < 1 || n_vocab > LG_SAMPLE_VOCAB) return lg_fail(-2, "sample: a vocabulary of %d (1..%d)", n_vocab, LG_SAMPLE_VOCAB);
    if (stride < n_vocab) return lg_fail(-2, "sample: rows of %d logits, %lld apart", n_vocab, (long long)stride);
    if (rows == 0) return 0;
    if (!d_logits || !d_params || !d_u || !d_tok) return lg_fail(-1, "sample: null argument");
    if (((uintptr_t)d_logits | (uintptr_t)d_params) & 3) return lg_fail(-2, "sample: arguments that are not aligned to 4 bytes");
    const size_t need = lg_hip_sample_workspace(rows, n_vocab);
    if (need && (!d_work || work_bytes < need || ((uintptr_t)d_work & 255)))
        return lg_fail(-2, "sample: %zu bytes of working memory (aligned to 256), given %zu", need, d_work ? work_bytes : 0);
    const SampleArgs a{ d_logits, (long long)stride, (const SampleRow *)d_params, d_u, d_tok, d_prob, d_kept, n_vocab, 0 };
    // loads of 16 bytes where every row is aligned to that (top-p of 33 rows of 262144: 66.4 us, of rows that are not 75.2)
    if (aligned16(d_logits) && stride % 4 == 0) launch_sample<true>(a, rows, need ? (char *)d_work : nullptr, (hipStream_t)stream);
    else launch_sample<false>(a, rows, need ? (char *)d_work : nullptr, (hipStream_t)stream);
    LG_TRY(hipGetLastError());
    return 0;
}

// ---- trees ------------------------------------------------------------------------------------------------------
static int check_trees(const char *who, int n_seq, int max_tree, int n_rows) {
    if (n_seq < 0 || n_seq > LG_PA_SEQS) return lg_fail(-2, "%s: %d sequences (0..%d)", who, n_seq, LG_PA_SEQS);
    if (max_tree < 1 || max_tree > LG_TREE_ROWS) return lg_fail(-2, "%s: trees of up to %d rows (1..%d)", who, max_tree, LG_TREE_ROWS);
    if (n_rows < 0) return lg_fail(-2, "%s: %d rows", who, n_rows);
    return 0;
}
static dim3 waves_for(int n_seq) { return dim3((unsigned)((n_seq + LG_TREE_WG / 64 - 1) / (LG_TREE_WG / 64))); }

static int launch_tree_plan(const char *who, int n_seq, int max_tree, int n_rows, const int32_t *d_start, const int32_t *d_parent, const int32_t *d_len, int32_t *d_grown, uint64_t *d_mask,
                            int32_t *d_pos, int32_t *d_seq, int32_t *d_status, void *stream) {
    if (!d_start || !d_len || !d_status || (n_rows && (!d_parent || !d_mask || !d_pos || !d_seq))) return lg_fail(-1, "%s: null argument", who);
    if ((uintptr_t)d_mask & 7) return lg_fail(-2, "%s: sets that are not aligned to 8 bytes", who);
    hipLaunchKernelGGL(lg_k_tree_plan, waves_for(n_seq), dim3(LG_TREE_WG), 0, (hipStream_t)stream, d_start, d_parent, d_len, d_grown, (lg_u64 *)d_mask, d_pos, d_seq, d_status, n_seq, n_rows,
                       max_tree);
    LG_TRY(hipGetLastError());
    return 0;
}
extern "C" int lg_hip_tree_plan(int n_seq, int max_tree, int n_rows, const int32_t *d_start, const int32_t *d_parent, const int32_t *d_len, uint64_t *d_mask, int32_t *d_pos,
                                int32_t *d_seq, int32_t *d_status, void *stream) {
    const int rc = check_trees("tree_plan", n_seq, max_tree, n_rows);
    if (rc || n_seq == 0) return rc;
    return launch_tree_plan("tree_plan", n_seq, max_tree, n_rows, d_start, d_parent, d_len, nullptr, d_mask, d_pos, d_seq, d_status, stream);
}
extern "C" int lg_hip_tree_plan_from(int n_seq, int max_tree, int n_rows, const int32_t *d_start, const int32_t *d_parent, const int32_t *d_len, int32_t *d_len_grown, uint64_t *d_mask,
                                     int32_t *d_pos, int32_t *d_seq, int32_t *d_status, void *stream) {
    const int rc = check_trees("tree_plan_from", n_seq, max_tree, n_rows);
    if (rc || n_seq == 0) return rc;
    if (!d_len_grown) return lg_fail(-1, "tree_plan_from: null argument");
    if (d_len_grown == d_len) return lg_fail(-2, "tree_plan_from: lengths before and behind the plan in one place");
    return launch_tree_plan("tree_plan_from", n_seq, max_tree, n_rows, d_start, d_parent, d_len, d_len_grown, d_mask, d_pos, d_seq, d_status, stream);
}

extern "C" int lg_hip_tree_accept(int n_seq, int max_tree, int n_rows, const int32_t *d_start, const int32_t *d_parent, const int32_t *d_token, const int32_t *d_next, const int32_t *d_len,
                                  int32_t *d_path, int32_t *d_count, int32_t *d_len_out, int32_t *d_last, void *stream) {
    const int rc = check_trees("tree_accept", n_seq, max_tree, n_rows);
    if (rc) return rc;
    if (n_seq == 0) return 0;
    if (!d_start || !d_len || !d_path || !d_count || !d_len_out || !d_last || (n_rows && (!d_parent || !d_token || !d_next))) return lg_fail(-1, "tree_accept: null argument");
    hipLaunchKernelGGL(lg_k_tree_accept, waves_for(n_seq), dim3(LG_TREE_WG), 0, (hipStream_t)stream, d_start, d_parent, d_token, d_next, d_len, d_path, d_count, d_len_out, d_last, n_seq, n_rows,
                       max_tree);
    LG_TRY(hipGetLastError());
    return 0;
}

// How many pairs a workgroup takes, 16 RT by each of WR wavefronts, goes by how much there is to read: tiles of all sequences and key heads, as often as groups of so many pairs read them.
// Few pairs make short workgroups, and many of them; where the chip is full their reads of the same keys again cost more.  Us, trees of 8 and 16 rows, 4 query heads to a key head:
//
//   heads  keys of sequences     tiles, read by 16   16 pairs  32       heads  keys of sequences     tiles, read by 64   32 pairs  64
//   256    windows of 512, 32    4608                20.3      25.2     256    windows of 512, 64    2304                27.0      33.3
//          windows of 512, 40    5760                36.9      25.4            windows of 512, 96    3456                46.5      36
//          4096, 4               4096                23.3      24.7            windows of 512, 128   4608                48.4      36.2
//          4096, 8               8192                36.0      32.0            4096, 8               2048                33.0      33.7
//          100, 1 (trees of 5)   8                   9.7       12.9            4096, 20              5120                47.3      45.7
//   128    all                   2048                14.8      15.8            4096, 32              8192                75.9      63.5
//          all                   4096                20.3      18.3     128    windows               4608                31.8      24.8
//          windows               4608                12.5      15.9     512    windows               2304                62.6      55.9
//          windows               9216                18.5      17.3
//   64     all                   8192                19.3      20.5     (64 pairs: lg_k_tree_wide, which reads keys once for all four wavefronts but
//          all                   16384               28.1      21.5     spends 10 us beside its tiles.  Trees of up to 32 pairs in its workgroups:
//   512    all                   4096                38.4      42.8     100003 tokens 166 for 147, 64 sequences in windows of 512 31.1 for 25.5)
//          windows               4352                32.9      54.8
struct TreeForm { int rt, wr; bool wide; };
static TreeForm tree_form(int pairs, int hd, int64_t tiles) {
    if (pairs <= 16 || tiles * ((pairs + 15) / 16) <= (hd == 64 ? 9216 : 4608)) return { 1, 1, false };
    if (pairs <= 32 || (hd < 512 && tiles * ((pairs + 63) / 64) <= 2560)) return hd == 512 ? TreeForm{ 1, 2, false } : TreeForm{ 2, 1, false };
    return { 1, LG_PA_WAVES, true };
}
// Trees of up to so many tiles are left whole, as alone_of says for one row.  A workgroup of 64 pairs spends 10 us beside its tiles, of 1.5 us each, and the joining launch takes 8.
// Whole and in splits, us, heads of 256, by units (sequences x key heads x groups) and keys:
//   2 units    512 31.6 and 19.3                      128 units  144 17.6 and 29.4, 272 24.6 and 30.3, 528 35.7 and 34.9 (all lengths up to it: 36.7 and 33.2)
//   16 units   512 33.9 and 23.2                      256 units  272 26.7 and 47.7, 528 39.6 and 55.6                512 units  528 65.1 and 114.8
static int tree_alone_of(int hd, int64_t units, bool wide) {
    if (!wide) return alone_of(hd, units);
    return units < 64 ? 8 : units < 160 ? 16 : units < 512 ? 24 : 32;
}
struct TreeCut { AttnCut c; int64_t items; TreeForm form; int rows, groups, slots, longest; };
// As cut_of, for workgroups of several pairs: a split of a tree takes as many as its pairs need, and those are what the chip's room is counted in.  items: workgroups of a key head, at most
static TreeCut tree_cut_of(int n_seq, int max_tree, int n_head, int n_head_kv, int hd, int max_len, int window) {
    const int pairs = max_tree * (n_head / n_head_kv);
    // (a tree's rows see a window from the first committed position that its row 0 sees to its last row)
    const int64_t reach = window > 0 ? (int64_t)window + max_tree + LG_PA_TILE : max_len, span = std::min<int64_t>(reach, max_len), tiles = (span + LG_PA_TILE - 1) / LG_PA_TILE;
    const TreeForm form = tree_form(pairs, hd, tiles * n_seq * n_head_kv);
    const int rows = 16 * form.rt * form.wr, groups = (pairs + rows - 1) / rows, slots = 256 * (form.wide ? lg_wide_per_simd(hd) : lg_tree_per_simd(hd, form.rt));
    const int longest = form.wide ? LG_PA_CHUNK / LG_PA_TILE : LG_TREE_TILES;
    const int64_t all = (int64_t)n_seq * groups, units = all * n_head_kv;
    const int alone = tree_alone_of(hd, units, form.wide), min_tiles = tiles <= alone ? alone : 4;
    const int64_t least = std::max<int64_t>(1, (tiles + min_tiles - 1) / min_tiles), one = std::max<int64_t>(1, slots / n_head_kv * longest);
    const int64_t rounds = std::max<int64_t>({ 1, (units + slots / 2 - 1) / (slots / 2), (all * tiles + one - 1) / one });
    const int64_t full = std::max<int64_t>(rounds * slots / n_head_kv, all * tiles / longest);
    return { { std::min<int64_t>(n_seq * least, full + n_seq), all * tiles, least > 1, min_tiles }, std::min<int64_t>(all * least, full + all), form, rows, groups, slots, longest };
}
static size_t tree_cut_bytes(int n_seq, const TreeCut &t) { return up256(((size_t)n_seq + 1 + (n_seq > LG_PA_LANES ? n_seq + 2 + t.items : 0)) * 4); }
extern "C" size_t lg_hip_paged_tree_attention_workspace(int n_seq, int max_tree, int n_head, int n_head_kv, int hd, int max_len, int window) {
    if (!attn_shape(n_seq, n_head, n_head_kv, hd, max_len) || max_tree < 1 || max_tree > LG_TREE_ROWS || window < 0) return 0;
    const TreeCut t = tree_cut_of(n_seq, max_tree, n_head, n_head_kv, hd, max_len, window);
    if (!t.c.join) return 0;
    const size_t slots = (size_t)t.c.splits * max_tree * n_head;
    return tree_cut_bytes(n_seq, t) + 2 * up256(slots * 4) + slots * hd * 4;
}

extern "C" int lg_hip_paged_tree_attention_pairs(int n_seq, int max_tree, int n_head, int n_head_kv, int hd, int max_len, int window) {
    if (!attn_shape(n_seq, n_head, n_head_kv, hd, max_len) || max_tree < 1 || max_tree > LG_TREE_ROWS || window < 0) return 0;
    return tree_cut_of(n_seq, max_tree, n_head, n_head_kv, hd, max_len, window).rows;
}
// (lg_tree_number turns 64 workgroups in a row: launches are of whole sixty-fours)
static int64_t tree_groups(const TreeCut &t, int n_head_kv) { return (t.items * n_head_kv + 63) / 64 * 64; }

#define LG_TREE_FEW 1024
template <int HD>
static void launch_tree(const TreeAttn &a, const TreeCut &t, hipStream_t st) {
    const dim3 grid((unsigned)tree_groups(t, a.nkv)), wg(LG_PA_WAVES * 64);
    if (t.form.wide) {
        hipLaunchKernelGGL(lg_k_tree_wide<HD>, grid, wg, 0, st, a);
    } else if (t.form.rt * t.form.wr == 1) hipLaunchKernelGGL((lg_k_tree_attn<HD, 1, 1>), grid, wg, 0, st, a);
    else if constexpr (HD == 512) hipLaunchKernelGGL((lg_k_tree_attn<HD, 1, 2>), grid, wg, 0, st, a);
    else hipLaunchKernelGGL((lg_k_tree_attn<HD, 2, 1>), grid, wg, 0, st, a);
    if (!t.c.join) return;
    // a wavefront to a row's head, or eight where those are few (24 sequences with trees of 64: 8.2 and 30 us; one of 100003 keys with 16 rows: 29 and 7.3)
    if ((int64_t)a.H * a.max_tree * a.n_seq > LG_TREE_FEW) hipLaunchKernelGGL((lg_k_page_merge<HD, 1, TreeAttn>), dim3(a.H * a.max_tree, a.n_seq), dim3(64), 0, st, a);
    else hipLaunchKernelGGL((lg_k_page_merge<HD, 8, TreeAttn>), dim3(a.H * a.max_tree, a.n_seq), dim3(512), 0, st, a);
}

extern "C" int lg_hip_paged_tree_attention(const struct lg_hip_pages *p, const float *d_q, int64_t q_stride, int n_rows, int n_seq, int max_tree, int n_head, const int32_t *d_table, int max_blocks,
                                           const int32_t *d_len, const int32_t *d_start, const uint64_t *d_mask, const int32_t *d_pos, int max_len, int window, float scale, float *d_out,
                                           int64_t out_stride, void *d_work, size_t work_bytes, void *stream) {
    PageGeo g;
    int rc = check_pages("paged_tree_attention", p, &g);
    if (rc || (rc = check_trees("paged_tree_attention", n_seq, max_tree, n_rows))) return rc;
    const int hd = p->head_dim;
    if (!attn_shape(n_seq, n_head, p->n_head_kv, hd, max_len))
        return lg_fail(-2, "paged_tree_attention: %d query heads on %d key heads (at most 8 each), lengths up to %d", n_head, p->n_head_kv, max_len);
    if (p->row_stride > 1 << 27) return lg_fail(-2, "paged_tree_attention: rows %lld values apart (at most 2^27)", (long long)p->row_stride);
    if (max_blocks < 1 || (int64_t)max_blocks * p->page_size > INT32_MAX) return lg_fail(-2, "paged_tree_attention: %d blocks of %d positions", max_blocks, p->page_size);
    if (window < 0) return lg_fail(-2, "paged_tree_attention: a window of %d", window);
    if (n_seq == 0 || n_rows == 0) return 0;
    if (!d_q || !d_table || !d_len || !d_start || !d_mask || !d_pos || !d_out) return lg_fail(-1, "paged_tree_attention: null argument");
    const int64_t qd = (int64_t)n_head * hd;
    if (q_stride < qd || q_stride % 4 || !aligned16(d_q)) return lg_fail(-2, "paged_tree_attention: query rows of %lld values, %lld apart (aligned to 16 bytes)", (long long)qd, (long long)q_stride);
    if (out_stride < qd || ((uintptr_t)d_out & 3)) return lg_fail(-2, "paged_tree_attention: output rows of %lld values, %lld apart", (long long)qd, (long long)out_stride);
    if ((uintptr_t)d_mask & 7) return lg_fail(-2, "paged_tree_attention: sets that are not aligned to 8 bytes");
    const TreeCut t = tree_cut_of(n_seq, max_tree, n_head, p->n_head_kv, hd, max_len, window);
    const AttnCut &c = t.c;
    // (sums over the sequences are 32 bits on the device, and so are a launch's threads; the joining launch has 512 to a row's head)
    if (c.tiles > INT32_MAX || tree_groups(t, p->n_head_kv) > LG_MOST_GROUPS || (c.join && (int64_t)n_head * max_tree * n_seq > LG_MOST_GROUPS / 2))
        return lg_fail(-2, "paged_tree_attention: %d sequences of up to %d rows of %d heads in %lld splits in one call", n_seq, max_tree, n_head, (long long)c.splits);
    const size_t need = lg_hip_paged_tree_attention_workspace(n_seq, max_tree, n_head, p->n_head_kv, hd, max_len, window);
    if (need && (!d_work || work_bytes < need || ((uintptr_t)d_work & 255)))
        return lg_fail(-2, "paged_tree_attention: %zu bytes of working memory (aligned to 256), given %zu", need, d_work ? work_bytes : 0);
    const size_t part = up256((size_t)c.splits * max_tree * n_head * 4);
    char *const w = need ? (char *)d_work + tree_cut_bytes(n_seq, t) : nullptr;
    const TreeAttn a{ { g, d_q, (long long)q_stride, d_table, d_len, d_out, (long long)out_stride, (float *)w, need ? (float *)(w + part) : nullptr, need ? (float *)(w + 2 * part) : nullptr, scale,
                        need ? (int32_t *)d_work : nullptr, n_head, p->n_head_kv, n_seq, max_blocks, max_len, window, t.slots, c.least },
                      d_start, d_pos, (const lg_u64 *)d_mask, n_rows, max_tree, t.groups, t.rows, (int)t.items, t.longest };
    hipStream_t st = (hipStream_t)stream;
    if (c.join && n_seq > LG_PA_LANES) hipLaunchKernelGGL(lg_k_tree_cut, dim3(1), dim3(LG_PC_WG), 0, st, a);
    switch (hd) {
        case 64:  launch_tree<64>(a, t, st); break;
        case 128: launch_tree<128>(a, t, st); break;
        case 256: launch_tree<256>(a, t, st); break;
        default:  launch_tree<512>(a, t, st); break;
    }
    LG_TRY(hipGetLastError());
    return 0;
}

// ---- shared pages -----------------------------------------------------------------------------------------------
// A workgroup of four wavefronts where the table has a few entries: its barriers are shorter.  Eight forks of 16 pages and their end: 23.0 us, with 1024 threads 24.7; 15 of 250 pages 87 and 42
#define LG_FORK_FEW 16
static size_t fork_page_bytes(int n_pages) { return up256((size_t)n_pages * sizeof(ForkPage)); }
static bool fork_shape(int n_seq, int n_pages, int max_blocks) {
    // (entries of the table are counted in 31 bits)
    return n_seq >= 0 && n_seq <= LG_PLAN_SEQS && n_pages >= 1 && max_blocks >= 1 && (int64_t)n_seq * max_blocks <= 1 << 30;
}
extern "C" size_t lg_hip_paged_fork_workspace(int n_seq, int n_pages, int max_blocks) {
    if (!fork_shape(n_seq, n_pages, max_blocks)) return 0;
    return fork_page_bytes(n_pages) + up256((size_t)n_seq * max_blocks * 4);
}
extern "C" int lg_hip_paged_fork(int n_seq, int page_size, int n_pages, int max_blocks, const int32_t *d_src, const int32_t *d_len_old, const int32_t *d_len_new, int32_t *d_table,
                                 int32_t *d_shares, int32_t *d_free, int32_t *d_n_free, int32_t *d_from, int32_t *d_to, int32_t *d_rows, int32_t *d_status, void *d_work, size_t work_bytes,
                                 void *stream) {
    const int shift = shift_of(page_size);
    if (n_seq < 0 || n_seq > LG_PLAN_SEQS) return lg_fail(-2, "paged_fork: %d sequences (0..%d)", n_seq, LG_PLAN_SEQS);
    if (shift < 0) return lg_fail(-2, "paged_fork: pages of %d positions (a power of two of 16..256)", page_size);
    if (n_pages < 1 || (int64_t)n_pages * page_size > INT32_MAX || max_blocks < 1 || (int64_t)max_blocks * page_size > INT32_MAX || !fork_shape(n_seq, n_pages, max_blocks))
        return lg_fail(-2, "paged_fork: %d pages and %d blocks of %d positions for %d sequences (positions and entries are 31 bits)", n_pages, max_blocks, page_size, n_seq);
    if (!d_shares || !d_free || !d_n_free || !d_status || (n_seq && (!d_src || !d_len_old || !d_len_new || !d_table || !d_from || !d_to || !d_rows)))
        return lg_fail(-1, "paged_fork: null argument");
    const size_t need = lg_hip_paged_fork_workspace(n_seq, n_pages, max_blocks);
    if (!d_work || work_bytes < need || ((uintptr_t)d_work & 255)) return lg_fail(-2, "paged_fork: %zu bytes of working memory (aligned to 256), given %zu", need, d_work ? work_bytes : 0);
    const ForkArgs a{ d_src, d_len_old, d_len_new, d_table, d_shares, d_free, d_n_free, d_from, d_to, d_rows, d_status, (ForkPage *)d_work, (int32_t *)((char *)d_work + fork_page_bytes(n_pages)),
                      n_seq, shift, n_pages, max_blocks };
    if (n_seq <= LG_FORK_FEW && (int64_t)n_seq * max_blocks <= 1024) hipLaunchKernelGGL((lg_k_page_fork<256, LG_FORK_FEW>), dim3(1), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((lg_k_page_fork<1024, LG_PLAN_SEQS>), dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
    LG_TRY(hipGetLastError());
    return 0;
}

// The layers of a cache: one table serves them, so pages are alike in size and number; heads and strides are each layer's own
static int check_layers(const char *who, const struct lg_hip_pages *p, int n_layers) {
    if (n_layers < 0) return lg_fail(-2, "%s: %d layers", who, n_layers);
    if (n_layers && !p) return lg_fail(-1, "%s: null argument", who);
    for (int i = 0; i < n_layers; ++i) {
        PageGeo g;
        const int rc = check_pages(who, p + i, &g);
        if (rc) return rc;
        if (p[i].page_size != p[0].page_size || p[i].n_pages != p[0].n_pages)
            return lg_fail(-2, "%s: layer %d has %d pages of %d positions, layer 0 %d of %d", who, i, p[i].n_pages, p[i].page_size, p[0].n_pages, p[0].page_size);
    }
    return 0;
}
// LG_LAYERS at a time: launch(layers, how many, most units of one)
template <typename Launch>
static void each_layers(const struct lg_hip_pages *p, int n_layers, Launch launch) {
    for (int from = 0; from < n_layers; from += LG_LAYERS) {
        PageLayers ls = {};
        const int n = std::min(LG_LAYERS, n_layers - from);
        int most = 0;
        for (int i = 0; i < n; ++i) {
            const struct lg_hip_pages &x = p[from + i];
            ls.l[i] = PageLayer{ x.k, x.v, x.row_stride, x.page_stride, x.n_head_kv * x.head_dim / 8 };
            most = std::max(most, ls.l[i].units);
        }
        launch(ls, n, most);
    }
}
extern "C" int lg_hip_paged_compact(const struct lg_hip_pages *layers, int n_layers, int n_seq, int max_tree, const int32_t *d_table, int max_blocks, const int32_t *d_len, const int32_t *d_start,
                                    const int32_t *d_path, const int32_t *d_count, void *stream) {
    int rc = check_layers("paged_compact", layers, n_layers);
    if (rc || (rc = check_trees("paged_compact", n_seq, max_tree, 0))) return rc;
    if (n_layers == 0) return 0;
    if (max_blocks < 1 || (int64_t)max_blocks * layers->page_size > INT32_MAX) return lg_fail(-2, "paged_compact: %d blocks of %d positions", max_blocks, layers->page_size);
    if (n_seq == 0) return 0;
    if (!d_table || !d_len || !d_start || !d_path || !d_count) return lg_fail(-1, "paged_compact: null argument");
    each_layers(layers, n_layers, [&](const PageLayers &ls, int n, int most) {
        hipLaunchKernelGGL(lg_k_page_compact, dim3((unsigned)(2 * most + LG_MOVE_PLACES - 1) / LG_MOVE_PLACES, (unsigned)n, (unsigned)n_seq), dim3(256), 0, (hipStream_t)stream, ls, d_table, d_len, d_start,
                           d_path, d_count, max_tree, max_blocks, shift_of(layers->page_size), layers->n_pages);
    });
    LG_TRY(hipGetLastError());
    return 0;
}
extern "C" int lg_hip_paged_copy(const struct lg_hip_pages *layers, int n_layers, int n, const int32_t *d_from, const int32_t *d_to, const int32_t *d_rows, void *stream) {
    const int rc = check_layers("paged_copy", layers, n_layers);
    if (rc) return rc;
    if (n < 0 || n > 65535) return lg_fail(-2, "paged_copy: %d pages (0..65535)", n);
    if (n == 0 || n_layers == 0) return 0;
    if (!d_from || !d_to || !d_rows) return lg_fail(-1, "paged_copy: null argument");
    each_layers(layers, n_layers, [&](const PageLayers &ls, int k, int most) {
        // several workgroups to a page where there are few pages, up to 4096 in all.  Forks and copy, one workgroup to a page, this, and one to every 4 loads of a thread: two pages of 256
        // positions of one layer 33.7, 16.3 and 16.3 us, of 48 layers 47.6, 42.7 and 47.6, nine of 48 261, 240 and 235, 244 pages of 32 positions of 48 layers 394, 394 and 408
        const int64_t pages = (int64_t)n * k * 2, whole = ((int64_t)layers->page_size * most + 1023) / 1024;
        const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(whole, 4096 / pages));
        hipLaunchKernelGGL(lg_k_page_copy, dim3((unsigned)(2 * parts), (unsigned)k, (unsigned)n), dim3(256), 0, (hipStream_t)stream, ls, d_from, d_to, d_rows, shift_of(layers->page_size),
                           layers->n_pages, parts);
    });
    LG_TRY(hipGetLastError());
    return 0;
}

// ---- rules ------------------------------------------------------------------------------------------------------
template <bool VEC>
static void launch_rules(const RulesArgs &a, hipStream_t st) {
    const unsigned lds = LG_RULES_SLICE * 4 * (a.bias_start ? 2 : a.penalty ? 1 : 0);
    hipLaunchKernelGGL(lg_k_rules<VEC>, dim3((unsigned)((a.n_vocab + LG_RULES_SLICE - 1) / LG_RULES_SLICE), (unsigned)a.rows), dim3(LG_RULES_WG), lds, st, a);
}
extern "C" int lg_hip_adjust_logits(const struct lg_hip_logit_rules *r, const float *d_logits, int64_t stride, int rows, int n_vocab, float *d_out, int64_t out_stride, void *stream) {
    if (!r) return lg_fail(-1, "adjust_logits: null argument");
    if (rows < 0 || rows > 65535) return lg_fail(-2, "adjust_logits: %d rows (0..65535)", rows);
    if (n_vocab < 1 || n_vocab > LG_RULES_VOCAB) return lg_fail(-2, "adjust_logits: a vocabulary of %d (1..%d)", n_vocab, LG_RULES_VOCAB);
    if (stride < n_vocab || out_stride < n_vocab) return lg_fail(-2, "adjust_logits: rows of %d logits, %lld and %lld apart", n_vocab, (long long)stride, (long long)out_stride);
    if (r->n_seq < 0 || r->n_bias < 0 || r->n_allow < 0) return lg_fail(-2, "adjust_logits: %d sequences, %d biases, %d grammars", r->n_seq, r->n_bias, r->n_allow);
    if (r->n_bias > 1 << 30) return lg_fail(-2, "adjust_logits: %d biases (at most 2^30: a workgroup counts past the last one by its threads)", r->n_bias);
    if (r->hist && (r->hist_stride < 1 || r->hist_stride > 1 << 30)) return lg_fail(-2, "adjust_logits: texts %lld tokens apart", (long long)r->hist_stride);
    if (r->n_allow && r->allow_stride < (n_vocab + 31) / 32) return lg_fail(-2, "adjust_logits: sets of %d tokens, %lld words apart", n_vocab, (long long)r->allow_stride);
    if (rows == 0) return 0;
    if (!d_logits || !d_out || (r->hist && (!r->hist_len || !r->penalty)) || (r->tree_mask && (!r->tree_start || !r->tree_tok || !r->penalty)) ||
        (r->n_bias && (!r->bias_start || !r->bias_tok || !r->bias)) || (r->n_allow && !r->allow))
        return lg_fail(-1, "adjust_logits: null argument");
    if ((((uintptr_t)d_logits | (uintptr_t)d_out | (uintptr_t)r->hist) & 3) || ((uintptr_t)r->tree_mask & 7)) return lg_fail(-2, "adjust_logits: arguments that are not aligned");
    if (d_out == d_logits && stride != out_stride) return lg_fail(-2, "adjust_logits: rows in place, %lld and %lld apart", (long long)stride, (long long)out_stride);
    const RulesArgs a{ d_logits, (long long)stride, d_out, (long long)out_stride, r->seq, (const RulesPenalty *)r->penalty, r->hist, r->hist_len, (long long)r->hist_stride,
                       (const lg_u64 *)r->tree_mask, r->tree_start, r->tree_tok, r->n_bias ? r->bias_start : nullptr, r->bias_tok, r->bias, r->allow, r->allow_row, (long long)r->allow_stride,
                       rows, n_vocab, r->n_seq, r->n_bias, r->n_allow };
    if (aligned16(d_logits) && aligned16(d_out) && stride % 4 == 0 && out_stride % 4 == 0) launch_rules<true>(a, (hipStream_t)stream);
    else launch_rules<false>(a, (hipStream_t)stream);
    LG_TRY(hipGetLastError());
    return 0;
}
