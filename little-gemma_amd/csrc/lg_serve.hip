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

static_assert(LG_PLAN_BAD_LEN == LG_HIP_PLAN_BAD_LENGTH && LG_PLAN_NO_PAGES == LG_HIP_PLAN_NO_PAGES && LG_PLAN_NO_SLOTS == LG_HIP_PLAN_NO_SLOTS &&
              LG_PLAN_BAD_STACK == LG_HIP_PLAN_BAD_STACK && LG_PLAN_BAD_PAGE == LG_HIP_PLAN_BAD_PAGE, "status bits of a plan");
static_assert(sizeof(SampleRow) == sizeof(struct lg_hip_sampling), "parameters of a row");

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
    if (a.n_seq > LG_PA_LANES) hipLaunchKernelGGL((lg_k_page_merge<HD, 1>), dim3(a.H, a.n_seq), dim3(64), 0, st, a);
    else hipLaunchKernelGGL((lg_k_page_merge<HD, 8>), dim3(a.H, a.n_seq), dim3(512), 0, st, a);
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
