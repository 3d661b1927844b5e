// lg_tree.h — trees of drafted tokens over a cache in pages: ancestors and positions of their rows, the accepted path, and attention of all rows of a tree.
//
// The n rows of a sequence's tree stand behind its committed positions: row k's K and V at position committed + k, committed = len - n.  Row 0 is the token chosen
// last, every other row hangs on an earlier one, its parent.  Row r of the tree is row start[i] + r of the step.
#pragma once

#include "lg_pages.h"

#define LG_TREE_TILES 127            // of a split at most, where its page ids lie in LDS: an id for each thread
#define LG_TREE_ROWS 64             // rows of a tree: a set of them is 64 bits, a lane each

enum { LG_TREE_BAD_ROWS = 1, LG_TREE_BAD_PARENT = 2, LG_TREE_BAD_LEN = 4 };            // LG_HIP_TREE_* of lg_hip.h

// A tree's rows: [row0, row0 + n), n = -1 where they are not rows of this step
struct TreeRows { int row0, n; };
__device__ __forceinline__ TreeRows lg_tree_rows(const int32_t *start, int seq, int n_rows, int max_tree) {
    const int row0 = start[seq];
    const long long n = (long long)start[seq + 1] - row0;
    return { row0, row0 < 0 || n < 0 || n > max_tree || row0 + n > n_rows ? -1 : (int)n };
}

// ---- plan and accept -------------------------------------------------------------------------------------------------
// A wavefront to a tree, a lane to a row.  Both are chains of a few hundred clocks behind two round trips to memory: one tree of 8 rows 1.4 us each, 256 of 64 rows (a few hundred KB) 2.6.
#define LG_TREE_WG 256
// anc(j) = anc(parent j) + {j}: every lane takes over what the row it points at has reached, then points where that one points; the reach doubles, so six steps do for 64 rows.
// With `grown`, len holds the lengths ahead of the plan that made `start`, and grown gets those behind it: by the rows that the plan has given, which are none where it was refused
__global__ __launch_bounds__(LG_TREE_WG) void lg_k_tree_plan(const int32_t *start, const int32_t *parent, const int32_t *len, int32_t *grown, lg_u64 *mask, int32_t *pos, int32_t *seq_of,
                                                            int32_t *status, int n_seq, int n_rows, int max_tree) {
    const int seq = (int)(blockIdx.x * (LG_TREE_WG / 64) + (threadIdx.x >> 6)), j = threadIdx.x & 63;
    if (seq >= n_seq) return;
    const TreeRows w = lg_tree_rows(start, seq, n_rows, max_tree);
    int total = len[seq];
    if (grown) {
        const long long rows = (long long)start[seq + 1] - start[seq], sum = total + rows;
        if (rows > 0 && sum <= INT32_MAX) total = (int)sum;
        if (j == 0) grown[seq] = total;
    }
    if (w.n < 0) { if (j == 0) status[seq] = LG_TREE_BAD_ROWS; return; }
    const bool live = j < w.n;
    int up = live ? parent[w.row0 + j] : 0;
    const bool wrong = live && j && (up < 0 || up >= j);
    int st = __any(wrong) ? LG_TREE_BAD_PARENT : 0;
    if (total < w.n) st |= LG_TREE_BAD_LEN;
    if (!live || j == 0 || st) up = j;
    lg_u64 set = 1ull << j;
    for (int reach = 1; reach < w.n; reach <<= 1) {
        set |= (lg_u64)(uint32_t)__shfl((int)(set >> 32), up) << 32 | (uint32_t)__shfl((int)set, up);
        up = __shfl(up, up);
    }
    if (live) {
        mask[w.row0 + j] = st ? 0 : set;
        pos[w.row0 + j] = st ? -1 : total - w.n + __popcll(set) - 1;
        seq_of[w.row0 + j] = seq;
    }
    if (j == 0) status[seq] = st;
}
// From row 0 on to the first row behind the current one that hangs on it and carries the token picked after it, as long as there is one.  Trees that lg_k_tree_plan refuses have been given no sets: what was
// picked behind their rows comes of no attention, so none of it is accepted, and the sequence stays at its committed length (at the length it has, where that is below the rows)
__global__ __launch_bounds__(LG_TREE_WG) void lg_k_tree_accept(const int32_t *start, const int32_t *parent, const int32_t *token, const int32_t *next, const int32_t *len,
                                                              int32_t *path, int32_t *count, int32_t *len_out, int32_t *last, int n_seq, int n_rows, int max_tree) {
    const int seq = (int)(blockIdx.x * (LG_TREE_WG / 64) + (threadIdx.x >> 6)), j = threadIdx.x & 63;
    if (seq >= n_seq) return;
    const TreeRows w = lg_tree_rows(start, seq, n_rows, max_tree);
    const int total = len[seq];
    const bool live = j < w.n;
    const int up = live ? parent[w.row0 + j] : -1, tok = live ? token[w.row0 + j] : -1, picked = live ? next[w.row0 + j] : -1;
    const bool orphan = __any(live && j && (up < 0 || up >= j)), fits = w.n > 0 && total >= w.n;
    int cur = 0, n = 0, mine = -1, want = -1;
    if (fits) {
        for (;;) {                                            // (rows only rise: at most 64 rounds)
            if (j == n) mine = cur;
            ++n;
            if (orphan) break;
            want = __builtin_amdgcn_readlane(picked, cur);
            const lg_u64 goes_on = __ballot(live && j > cur && up == cur && tok == want && want >= 0);
            if (!goes_on) break;
            cur = (int)__builtin_ctzll(goes_on);
        }
    }
    if (j < max_tree) path[(long long)seq * max_tree + j] = mine;
    if (j == 0) {
        count[seq] = n;
        len_out[seq] = fits ? total - w.n + (orphan ? 0 : n) : total;
        last[seq] = want;
    }
}

// ---- attend ----------------------------------------------------------------------------------------------------------
// o[j, h] = sum_t softmax_t(scale q[j, h].k[t]) v[t] over the committed positions t of a row's window and the rows of its tree that its set names.
//
// A workgroup takes a stretch of keys of one key head and up to ROWS = 16 RT WR of the n G (row, query head) pairs that share them; its four wavefronts take tiles of 32 keys in
// turn, as lg_k_page_attn does, and for the same reason no key or value passes through LDS: a lane's 16 bytes of a key row are the operand of the scores as they lie in memory, and the 8 x 8 values
// that a lane loads are turned in registers, here once for all pairs.
// Queries and probabilities are f32 and keep their precision as two binary16 parts (22 bits together) whose products go into one sum: two instructions for each 16 pairs, where the one-row
// kernel puts the second part into rows that it has anyway.  Queries lie in LDS as operands; maxima, sums and outputs are in f32.
// A tile that all pairs see whole (every tile but those at a window's border and of the tree) has no mask.  In the others a value that is infinite or NaN must not reach rows that
// do not see it through 0 * inf: it is taken out of the product and marked by a product of its own.
// Bound by memory where there is much to read (one tree of 16 rows over 100003 tokens, 8 key heads of 256: 820 MB in 139 to 145 us, 5.7 TB/s), by the chain lengths -> ids, queries -> keys -> products ->
// joining in LDS where there is little (a chain of 5 over 100 tokens 6 us, heads of 256 9.7): 64 trees of 16 in windows of 512, 65 MB, take 26 us, a workgroup to each compute unit.  Of a workgroup's 23 us, by clock stamps,
// 1.6 go by until starts and lengths are there, 3.8 until pages, sets and queries are and the first keys are on their way, 5.6 until the first tile is done (its keys, then its values, arrive), 9.3 with the three or four other tiles
// of a wavefront, 2.9 with the joining of the four and the stores.
struct TreeAttn : PageAttn {        // len: with the tree's rows
    const int32_t *start, *pos;
    const lg_u64 *mask;
    int n_rows, max_tree, groups, rows, items;  // groups of `rows` pairs, at most; workgroups of a key head, at most
    int longest;                    // tiles of a split at most
};
// The keys that rows of a tree see: [lo, len)
struct TreeSeq { int row0, n, done, lo, len; };
__device__ __forceinline__ TreeSeq lg_tree_seq(const TreeAttn &a, int seq) {
    const TreeRows w = lg_tree_rows(a.start, seq, a.n_rows, a.max_tree);
    const long long room = (long long)a.max_blocks << a.g.shift;
    const int len = a.len[seq];
    if (w.n <= 0 || len < w.n || len > a.max_len || len > room) return { w.row0, w.n < 0 ? 0 : w.n, 0, 0, 0 };
    const int done = len - w.n;
    return { w.row0, w.n, done, a.window > 0 && done >= a.window ? done + 1 - a.window : 0, len };
}
__device__ __forceinline__ void lg_pa_range(const TreeAttn &a, int seq, int &lo, int &len) {
    const TreeSeq s = lg_tree_seq(a, seq);
    lo = s.lo; len = s.len;
}
// How a call is cut: as lg_pa_cut does it, with a workgroup for each group of a sequence's pairs in each of its splits.  Workgroups are numbered sequence by sequence, split by split.
__device__ __forceinline__ uint32_t lg_tree_groups(const TreeAttn &a, int seq) {
    const int n = lg_tree_rows(a.start, seq, a.n_rows, a.max_tree).n * (a.H / a.nkv);
    return n > a.rows ? (uint32_t)(n + a.rows - 1) / (uint32_t)a.rows : 1u;
}
// `total` tiles, each as often as groups read it, of `some` groups.  (A split's page ids have a fixed place, so it has a.longest tiles at most: with fewer rounds than are asked for here all splits would be of
// that size and the last round of workgroups hardly filled)
template <typename Count>
__device__ __forceinline__ uint32_t lg_tree_tiles(const TreeAttn &a, uint32_t total, uint32_t some, Count count) {
    const uint32_t one = (uint32_t)a.slots / a.nkv * a.longest, most = one ? one : 1;
    return lg_pa_split_tiles(a, total, some, count, (total + most - 1) / most, a.longest);
}
struct TreePart { int tiles, seq, index, first, n, group; };       // as PageCut; the group of pairs
__device__ __forceinline__ TreePart lg_tree_part(const TreeAttn &a, int item) {
    if (!a.pm) { const int seq = item / a.groups; return { a.least, seq < a.n_seq ? seq : -1, 0, seq, 1, item % a.groups }; }
    if (a.n_seq > LG_PA_LANES) {
        const int32_t *const items = a.cut + a.n_seq + 2;
        if (item >= items[a.n_seq]) return { 0, -1, 0, 0, 0, 0 };
        const int seq = items[a.n_seq + 1 + item], first = a.cut[seq], n = a.cut[seq + 1] - first, k = item - items[seq], groups = (items[seq + 1] - items[seq]) / n;
        return { a.cut[a.n_seq + 1], seq, k / groups, first, n, k % groups };
    }
    // a lane for each, in every wavefront: no barrier
    const int i = threadIdx.x & 63;
    const uint32_t mine = i < a.n_seq ? lg_pa_tiles(a, i) : 0, by = i < a.n_seq ? lg_tree_groups(a, i) : 0;
    const uint32_t tiles = lg_tree_tiles(a, lg_wave_total(mine * by), lg_wave_total(mine ? by : 0), [&](uint32_t t) { return lg_wave_total(by * ((mine + t - 1) / t)); });
    const uint32_t n = i < a.n_seq ? lg_pa_splits(mine, tiles) : 0, first = lg_wave_run(n) - n, run = lg_wave_run(n * by) - n * by;
    const lg_u64 it = __ballot((uint32_t)item - run < n * by);
    if (!it) return { (int)tiles, -1, 0, 0, 0, 0 };
    const int lane = (int)__builtin_ctzll(it), k = item - (int)lg_lane(run, lane), groups = (int)lg_lane(by, lane);
    return { (int)tiles, lane, k / groups, (int)lg_lane(first, lane), (int)lg_lane(n, lane), k % groups };
}
// The cut of more sequences than a wavefront has lanes, worked out once: splits before each sequence and their tiles, workgroups before each sequence and their sequences
__global__ __launch_bounds__(LG_PC_WG) void lg_k_tree_cut(TreeAttn a) {
    __shared__ uint32_t part[LG_PC_WG / 64];
    __shared__ int32_t before[LG_PA_SEQS + 1];
    constexpr int PER = LG_PA_SEQS / LG_PC_WG;
    const int per = (a.n_seq + LG_PC_WG - 1) / LG_PC_WG, i0 = threadIdx.x * per;
    uint32_t x[PER], by[PER], mine = 0, some = 0, all;
    #pragma unroll
    for (int k = 0; k < PER; ++k) {
        const bool is = k < per && i0 + k < a.n_seq;
        x[k] = is ? lg_pa_tiles(a, i0 + k) : 0;
        by[k] = is ? lg_tree_groups(a, i0 + k) : 0;
        mine += x[k] * by[k]; some += x[k] ? by[k] : 0;
    }
    const uint32_t total = lg_block_sum<LG_PC_WG>(mine, part);
    some = lg_block_sum<LG_PC_WG>(some, part);
    const uint32_t tiles = lg_tree_tiles(a, total, some, [&](uint32_t t) {
        uint32_t n = 0;
        #pragma unroll
        for (int k = 0; k < PER; ++k) n += by[k] * ((x[k] + t - 1) / t);
        return lg_block_sum<LG_PC_WG>(n, part);
    });
    uint32_t n = 0, m = 0;
    #pragma unroll
    for (int k = 0; k < PER; ++k) if (by[k]) { const uint32_t s = lg_pa_splits(x[k], tiles); n += s; m += s * by[k]; }
    uint32_t run = lg_block_run<LG_PC_WG>(n, part, &all) - n;
    if (threadIdx.x == 0) { a.cut[a.n_seq] = (int32_t)all; a.cut[a.n_seq + 1] = (int32_t)tiles; }
    uint32_t item = lg_block_run<LG_PC_WG>(m, part, &all) - m;
    int32_t *const items = a.cut + a.n_seq + 2;
    #pragma unroll
    for (int k = 0; k < PER; ++k)
        if (by[k]) {
            a.cut[i0 + k] = (int32_t)run; items[i0 + k] = before[i0 + k] = (int32_t)item;
            const uint32_t s = lg_pa_splits(x[k], tiles);
            run += s; item += s * by[k];
        }
    if (threadIdx.x == 0) items[a.n_seq] = before[a.n_seq] = (int32_t)all;
    __syncthreads();
    for (int s = threadIdx.x; s < (int)all; s += LG_PC_WG) items[a.n_seq + 1 + s] = lg_owner(before, a.n_seq, s);
}
// Workgroups are dealt over 8 XCDs in turn; eight in a row of the numbers above go to one, so that the groups of a split, which read the same keys, find them in its L2
__device__ __forceinline__ int lg_tree_number(int block) { const int y = block >> 3; return ((y >> 3) * 8 + (block & 7)) * 8 + (y & 7); }
__device__ __forceinline__ MergeRow lg_merge_row(const TreeAttn &a) {
    const int seq = blockIdx.y, node = blockIdx.x / a.H, head = blockIdx.x % a.H;
    const TreeRows w = lg_tree_rows(a.start, seq, a.n_rows, a.max_tree);
    return { seq, node < w.n ? (long long)w.row0 + node : -1, (long long)a.max_tree * a.H, blockIdx.x, head };
}

// Probabilities are 2^(x - m), m the largest score of a while ago, rounded up to a whole number, less SHIFT (both and factors between two of them are exact): it is taken anew, and the sums so far scaled,
// only when a score passes it by SLACK more, which few tiles of a long row do.  So they stay below 2^15 in binary16, and what their two parts leave of a small one is at most 2^-32 of the largest.
// Where f32 does not hold the difference, from 2^27 on, where scores lie 16 and more apart, nothing is taken off (rounded, it was 16 for half of them, and the largest probability 2^16)
#define LG_TREE_SLACK 7.0f
#define LG_TREE_SHIFT 8.0f
__device__ __forceinline__ float lg_tree_base(float top) {
    const float c = ceilf(top), m = c - LG_TREE_SHIFT;
    return c - m > LG_TREE_SHIFT ? c : m;           // (infinities stay: their difference is NaN)
}
__device__ __forceinline__ bool lg_tree_passes(float top, float m) { return top - m > LG_TREE_SHIFT + LG_TREE_SLACK; }         // (both -inf: no)
// 1 in each half of a pair of binary16 values that is infinite or NaN (all bits of the exponent: one more carries into the sign's place)
__device__ __forceinline__ uint32_t lg_not_finite(uint32_t u) { return ((u & 0x7C007C00u) + 0x04000400u) >> 15 & 0x00010001u; }
// The largest `whole` of the wavefront's pairs; rows of the tree in front of a pair's window are taken out of its set (which the usual windows, wider than a tree is deep, do not ask for)
template <class Trim>
__device__ __forceinline__ void lg_tree_trim(const TreeAttn &a, const TreeSeq &w, const int32_t *s_pos, int &whole, Trim trim) {
    // (rows of 16 lanes by turning them: 0x128, 0x124, 0x122, 0x121 row_ror 8, 4, 2, 1)
    auto top = [&](int y) { if (y > whole) whole = y; };
    top(__builtin_amdgcn_mov_dpp(whole, 0x128, 0xF, 0xF, true)); top(__builtin_amdgcn_mov_dpp(whole, 0x124, 0xF, 0xF, true));
    top(__builtin_amdgcn_mov_dpp(whole, 0x122, 0xF, 0xF, true)); top(__builtin_amdgcn_mov_dpp(whole, 0x121, 0xF, 0xF, true));
    whole = __builtin_amdgcn_readfirstlane(whole);
    if (a.window <= 0) return;
    const int lane = threadIdx.x & 63;
    // (lg_wave_max is of numbers from 0 up: positions below 0 count as behind every window)
    const uint32_t before = lane < w.n ? s_pos[lane] < 0 ? 0x80000000u : 0x7FFFFFFFu - (uint32_t)s_pos[lane] : 0u;
    const uint32_t most = lg_wave_max(before);
    if (most < 0x80000000u && (int)(0x7FFFFFFFu - most) >= whole) return;
    #pragma unroll 1
    for (int k = 0; k < w.n; ++k) trim(s_pos[k], 1ull << k);
}
// Four keys in a row from position t on: which of them are committed, which there are at all, and where they are in the tree
struct LgQuad { uint32_t old, there; int t, k; };
__device__ __forceinline__ uint32_t lg_below(int x) { return (1u << (x < 0 ? 0 : x > 4 ? 4 : x)) - 1; }
__device__ __forceinline__ LgQuad lg_tree_quad(int t, int done, int end) { return { lg_below(done - t), lg_below(end - t), t, t - done }; }
// Those that a pair sees: of the committed ones the ones from lo on, of the tree's the ones of its set
__device__ __forceinline__ uint32_t lg_tree_sees(const LgQuad &x, int lo, lg_u64 set) {
    const int ahead = lo < x.t ? 0 : lo > x.t + 4 ? 4 : lo - x.t;
    const uint32_t tree = x.k <= -4 || x.k > 63 ? 0u : x.k < 0 ? (uint32_t)set << (-x.k & 3) : (uint32_t)(set >> (x.k & 63));
    return ((x.old & ~lg_below(ahead)) | (tree & ~x.old)) & x.there & 15u;
}
// Scores of eight keys (base-2 exponents) -> their probabilities as two binary16 parts, and their sum
typedef _Float16 lg_h2 __attribute__((ext_vector_type(2)));
typedef float lg_f2 __attribute__((ext_vector_type(2)));
template <int HALVES, class Part>
__device__ __forceinline__ void lg_tree_parts(const lg_f4 (&x)[HALVES], float m, float &l, Part &hi, Part &lo) {
    const float under = m == -INFINITY ? 0.0f : m;
    #pragma unroll
    for (int j = 0; j < 4 * HALVES; j += 2) {
        lg_f2 p, left;
        #pragma unroll
        for (int k = 0; k < 2; ++k) { p[k] = __builtin_amdgcn_exp2f(x[j >> 2][(j + k) & 3] - under); l += p[k]; }
        const lg_h2 h = __builtin_convertvector(p, lg_h2);
        #pragma unroll
        for (int k = 0; k < 2; ++k) left[k] = __builtin_fmaf((float)h[k], -1.0f, p[k]);
        const lg_h2 u = __builtin_convertvector(left, lg_h2);
        #pragma unroll
        for (int k = 0; k < 2; ++k) { hi[j + k] = h[k]; lo[j + k] = u[k]; }
    }
}
// The largest of the four rows of 16 lanes, lane by lane: rows are exchanged between two registers, without LDS
__device__ __forceinline__ float lg_max_of_rows(float x) {
    const auto u = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1]));
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
// How the four wavefronts of a workgroup share its work: WR of them take 16 RT pairs each, the others different keys
constexpr int lg_tree_per_simd(int hd, int rt) { return hd * rt <= 128 ? 3 : hd * rt < 256 ? 2 : 1; }
template <int HD, int RT, int WR>
__global__ __launch_bounds__(LG_PA_WAVES * 64, lg_tree_per_simd(HD, RT)) void lg_k_tree_attn(TreeAttn a) {
    constexpr int KS = HD / 32;                     // score steps
    constexpr int DL = HD >= 128 ? 8 : HD / 16;     // dimensions of a value load
    constexpr int CH = HD / (16 * DL);              // value loads of a key row
    constexpr int NT = HD / 16;                     // output tiles
    constexpr int HALVES = HD > 256 ? 1 : 2, TILE = 16 * HALVES, ROWS = 16 * RT * WR, WK = LG_PA_WAVES / WR;
    __shared__ float s_m[WK][ROWS], s_l[WK][ROWS], s_top[LG_PA_WAVES][ROWS];
    __shared__ long long s_to[ROWS];
    __shared__ __align__(16) union { lg_h8 q[RT * WR][KS][2][64]; float o[LG_PA_WAVES][16][HD]; } s;
    __shared__ int32_t s_ids[LG_TREE_TILES * 2 + 1], s_pos[LG_TREE_ROWS];
    const int number = lg_tree_number(blockIdx.x), kvh = number / a.items, G = a.H / a.nkv;
    if (kvh >= a.nkv) return;
    const TreePart cut = lg_tree_part(a, number % a.items);
    const int seq = __builtin_amdgcn_readfirstlane(cut.seq);
    if (seq < 0) return;
    const TreeSeq w = lg_tree_seq(a, seq);
    const int group = __builtin_amdgcn_readfirstlane(cut.group), at = __builtin_amdgcn_readfirstlane(cut.first + cut.index), n_pairs = w.n * G, p0 = group * ROWS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4, wr = wave % WR, wk = wave / WR;
    const int chunk = __builtin_amdgcn_readfirstlane(cut.tiles) * LG_PA_TILE, n_split = __builtin_amdgcn_readfirstlane(cut.n);
    auto tell = [&]() {                             // the joining launch
        if (a.pm && a.n_seq <= LG_PA_LANES && kvh == 0 && cut.index == 0 && group == 0 && threadIdx.x == 0) {
            a.cut[seq] = cut.first;
            if (seq == a.n_seq - 1) a.cut[a.n_seq] = cut.first + cut.n;
        }
    };
    if (p0 >= n_pairs) { tell(); return; }
    constexpr int STEP = WK * TILE;
    const int32_t *table = a.table + (long long)seq * a.max_blocks;
    const int first = (w.lo & ~(LG_PA_TILE - 1)) + __builtin_amdgcn_readfirstlane(cut.index) * chunk, end = w.len < first + chunk ? w.len : first + chunk;

    // queries: a wavefront takes every fourth 32 dimensions of all pairs
    constexpr int QS = (KS + LG_PA_WAVES - 1) / LG_PA_WAVES;
    const int qw = KS < LG_PA_WAVES ? wave % KS : wave;
    float4 qv[RT * WR][QS][2];
    #pragma unroll
    for (int rt = 0; rt < RT * WR; ++rt) {
        const int p = p0 + rt * 16 + c, q = p < n_pairs ? p : p0;
        const float *src = a.q + (w.row0 + q / G) * a.q_stride + (long long)(kvh * G + q % G) * HD + g * 8;
        #pragma unroll
        for (int i = 0; i < QS; ++i)
            #pragma unroll
            for (int j = 0; j < 2; ++j) qv[rt][i][j] = *(const float4 *)(src + (i * LG_PA_WAVES + qw) * 32 + j * 4);
    }
    // of pair c of the wavefront's own: the first position that it sees, and its set
    int lo_row[RT], whole = w.lo;
    lg_u64 set[RT];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int p = p0 + (wr * RT + rt) * 16 + c, row = w.row0 + (p < n_pairs ? p : p0) / G;
        const int pos = a.pos[row];
        set[rt] = pos < w.done ? 0 : a.mask[row] & (w.n < 64 ? (1ull << w.n) - 1 : ~0ull);
        lo_row[rt] = pos < w.done ? INT32_MAX : a.window > 0 ? pos - a.window + 1 : INT32_MIN;
        if (p < n_pairs && lo_row[rt] > whole) whole = lo_row[rt];
    }
    const int b0 = first >> a.g.shift;
    const bool has_id = (int)threadIdx.x <= ((end - 1) >> a.g.shift) - b0;
    const int my_id = has_id && b0 + (int)threadIdx.x < a.max_blocks ? table[b0 + threadIdx.x] : -1;
    const int my_pos = (int)threadIdx.x < w.n ? a.pos[w.row0 + threadIdx.x] : 0;
    auto tile_at = [&](int t) {
        PageIds p;
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = ((t + 16 * h < end ? t + 16 * h : t) >> a.g.shift) - b0;             // (a half behind the end is masked)
            p.id[h] = __builtin_amdgcn_readfirstlane(s_ids[i]);
        }
        return lg_pa_tile(a, p, t, kvh * HD);
    };
    lg_h8 kf[HALVES][KS];
    int t0 = p0 + wr * RT * 16 < n_pairs ? first + wk * TILE : end;      // (no pairs: nothing to do)
    PageTile now = lg_pa_tile(a, lg_pa_ids(a, table, t0 < end ? t0 : first), t0 < end ? t0 : first, kvh * HD);
    auto load_keys = [&](const PageTile &p) {
        #pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const uint16_t *kp = a.g.k + p.row[h] + c * a.g.row_stride + g * 8;
            #pragma unroll
            for (int i = 0; i < KS; ++i) kf[h][i] = *(const lg_h8 *)(kp + i * 32);
        }
    };
    float qs[RT];                                   // factor of the raw scores: base-2 exponents
    auto queries = [&]() {
        if ((int)threadIdx.x < w.n) s_pos[threadIdx.x] = my_pos;
        if (has_id) s_ids[threadIdx.x] = my_id;
        float top[RT * WR];
        #pragma unroll
        for (int rt = 0; rt < RT * WR; ++rt) {
            top[rt] = 0;
            #pragma unroll
            for (int i = 0; i < QS; ++i)
                #pragma unroll
                for (int j = 0; j < 2; ++j)
                    top[rt] = fmaxf(top[rt], fmaxf(fmaxf(fabsf(qv[rt][i][j].x), fabsf(qv[rt][i][j].y)), fmaxf(fabsf(qv[rt][i][j].z), fabsf(qv[rt][i][j].w))));
            top[rt] = fmaxf(top[rt], __shfl_xor(top[rt], 16));
            top[rt] = fmaxf(top[rt], __shfl_xor(top[rt], 32));
            if (lane < 16) s_top[wave][rt * 16 + lane] = top[rt];
        }
        lg_barrier_lds();
        auto power = [&](int row) {                 // top * 2^-e in [2^14, 2^15)
            float x = 0;
            #pragma unroll
            for (int v = 0; v < LG_PA_WAVES; ++v) x = fmaxf(x, s_top[v][row]);
            const int e = (int)(__float_as_uint(x) >> 23) - 127 - 14;
            return e < -100 ? -100 : e;             // (zero and tiny rows; 2^-e stays a float)
        };
        #pragma unroll
        for (int rt = 0; rt < RT * WR; ++rt) {
            const float up = __uint_as_float((unsigned)(127 - power(rt * 16 + c)) << 23);
            #pragma unroll
            for (int i = 0; i < QS; ++i) {
                const int step = i * LG_PA_WAVES + wave;
                if (step >= KS) continue;
                const float v[8] = { qv[rt][i][0].x, qv[rt][i][0].y, qv[rt][i][0].z, qv[rt][i][0].w, qv[rt][i][1].x, qv[rt][i][1].y, qv[rt][i][1].z, qv[rt][i][1].w };
                lg_h8 hi, lo;
                #pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float z = v[j] * up;
                    hi[j] = (_Float16)z;
                    lo[j] = (_Float16)(z - (float)hi[j]);
                }
                s.q[rt][step][0][lane] = hi;
                s.q[rt][step][1][lane] = lo;
            }
        }
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) qs[rt] = a.scale * 1.44269504088896341f * __uint_as_float((unsigned)(127 + power((wr * RT + rt) * 16 + c)) << 23);
        lg_barrier_lds();
    };
    // (on either side of the branch: behind it they would have to wait for everything in flight)
    if (t0 < end) {
        __builtin_amdgcn_sched_barrier(0);
        load_keys(now);
        __builtin_amdgcn_sched_barrier(0);
        queries();
    } else {
        queries();
        asm volatile("");                           // (so that the two sides stay apart)
    }
    // tiles in [whole, w.done) need no mask; rows of the tree in front of a window are taken out of the sets
    lg_tree_trim(a, w, s_pos, whole, [&](int pos, lg_u64 row) {
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) if (pos < lo_row[rt]) set[rt] &= ~row;
    });

    typedef uint32_t values[CH][4 * HALVES][DL / 2];
    auto load_values = [&](const PageTile &p, values &v) {
        #pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            #pragma unroll
            for (int j = 0; j < 4 * HALVES; ++j) {
                const uint16_t *vp = a.g.v + p.row[j >> 2] + (4 * g + (j & 3)) * a.g.row_stride + ch * 128 + c * DL;
                if constexpr (DL == 8) { const uint4 u = *(const uint4 *)vp; v[ch][j][0] = u.x; v[ch][j][1] = u.y; v[ch][j][2] = u.z; v[ch][j][3] = u.w; }
                else { const uint2 u = *(const uint2 *)vp; v[ch][j][0] = u.x; v[ch][j][1] = u.y; }
            }
    };
    lg_f4 acc[RT][NT];
    float m[RT], l[RT];                             // of pair c; l of this lane's keys alone
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY; l[rt] = 0;
        #pragma unroll
        for (int i = 0; i < NT; ++i) acc[rt][i] = (lg_f4){ 0, 0, 0, 0 };
    }
    typedef _Float16 part __attribute__((ext_vector_type(4 * HALVES)));
    auto product = [&](const part &x, const part &y, const lg_f4 &z) {
        if constexpr (HALVES == 2) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, z, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x16f16(x, y, z, 0, 0, 0);
    };

    auto turned = [&](const values &v, int ch, int i) {          // dimension ch * 128 + c * DL + i of the lane's keys
        union { uint32_t u[2 * HALVES]; part h; } b;
        #pragma unroll
        for (int k = 0; k < 2 * HALVES; ++k) b.u[k] = __builtin_amdgcn_perm(v[ch][2 * k + 1][i >> 1], v[ch][2 * k][i >> 1], i & 1 ? 0x07060302 : 0x05040100);
        return b.h;
    };
    auto plain = [&](int t, const PageTile &p) { return t >= whole && t + TILE <= w.done && t + TILE <= end && p.ok[0] && p.ok[HALVES - 1]; };
    // which of the lane's keys pair c sees: four bits for four keys in a row from the committed positions [lo_row, done) and from the set, none behind the end or in a page that is not there
    auto seen_in = [&](int t0, const PageTile &p, uint32_t (&sees)[RT]) {
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) sees[rt] = 0;
        #pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const LgQuad x = lg_tree_quad(t0 + 16 * h + 4 * g, w.done, p.ok[h] ? end : 0);
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) sees[rt] |= lg_tree_sees(x, lo_row[rt], set[rt]) << (4 * h);
        }
    };
    // One tile: its values are requested before its scores are made, the next tile's keys before its values are used (behind the last tile its own once more: a branch around the
    // loads would have them waited for with this tile's)
    // Outputs of forms that have a SIMD to themselves stay in the accumulation registers: where a product's sum is also read by an ordinary instruction the compiler keeps it in the others, and moves all of
    // them there and back for each tile
    constexpr bool ALONE = lg_tree_per_simd(HD, RT) == 1;
    auto stay = [&]() {
        if constexpr (ALONE)
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                #pragma unroll
                for (int i = 0; i < NT; ++i) asm volatile("" : "+a"(acc[rt][i]));
    };
    auto out_of = [&](float x) {
        if constexpr (!ALONE) return x;
        float y;
        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(y) : "a"(x));
        return y;
    };
    uint32_t odd = 0;
    const int t_first = t0;
    stay();
    for (; t0 < end; t0 += STEP) {
        const bool masked = !plain(t0, now);
        const PageTile here = now;
        now = tile_at(t0 + STEP < end ? t0 + STEP : t0);
        // queries from LDS a few steps ahead of their products
        constexpr int AT = RT == 1 && KS > 1 ? 2 : 1, GROUPS = KS / AT;
        lg_h8 q[2][AT][2][RT];
        auto ask = [&](int i) {
            #pragma unroll
            for (int k = 0; k < AT; ++k)
                #pragma unroll
                for (int x = 0; x < 2; ++x)
                    #pragma unroll
                    for (int rt = 0; rt < RT; ++rt) q[i & 1][k][x][rt] = s.q[wr * RT + rt][i * AT + k][x][lane];
        };
        ask(0);
        values v;
        load_values(here, v);
        __builtin_amdgcn_sched_barrier(0);
        lg_f4 sc[RT][HALVES];
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            #pragma unroll
            for (int h = 0; h < HALVES; ++h) sc[rt][h] = (lg_f4){ 0, 0, 0, 0 };
        #pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            if (i + 1 < GROUPS) ask(i + 1);
            __builtin_amdgcn_sched_barrier(0);
            #pragma unroll
            for (int k = 0; k < AT; ++k)
                #pragma unroll
                for (int x = 0; x < 2; ++x)
                    #pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        #pragma unroll
                        for (int h = 0; h < HALVES; ++h) sc[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[h][i * AT + k], q[i & 1][k][x][rt], sc[rt][h], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_keys(now);
        __builtin_amdgcn_sched_barrier(0);
        uint32_t sees[RT];
        if (masked) seen_in(t0, here, sees);
        else
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) sees[rt] = 255;
        float top[RT];
        bool higher = false;
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            top[rt] = -INFINITY;
            #pragma unroll
            for (int h = 0; h < HALVES; ++h)
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = sc[rt][h][r] * qs[rt];
                    if (!(sees[rt] >> (4 * h + r) & 1)) x = -INFINITY;
                    sc[rt][h][r] = x;
                    top[rt] = fmaxf(top[rt], x);
                }
            top[rt] = fmaxf(top[rt], __shfl_xor(top[rt], 16));
            top[rt] = fmaxf(top[rt], __shfl_xor(top[rt], 32));
            higher |= lg_tree_passes(top[rt], m[rt]);
        }
        if (__any(higher)) {
            if constexpr (ALONE) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");           // (products write accumulation registers up to 16 cycles after they are issued; out_of reads them where the compiler does not see it)
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float mn = fmaxf(m[rt], lg_tree_base(top[rt]));
                const float f = m[rt] == mn ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);       // (both -inf: nothing seen yet)
                l[rt] *= f; m[rt] = mn;
                float fr[4];
                #pragma unroll
                for (int r = 0; r < 4; ++r) fr[r] = __shfl(f, 4 * g + r);
                #pragma unroll
                for (int i = 0; i < NT; ++i) {
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) acc[rt][i][r] = fr[r] * out_of(acc[rt][i][r]);
                }
            }
            stay();
        }
        part hi[RT], lo[RT];
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) lg_tree_parts(sc[rt], m[rt], l[rt], hi[rt], lo[rt]);
        if (masked) {
            // keys that no pair of the group can see may hold anything: zeros in their place.  So are values that are not finite, until all else is done
            #pragma unroll
            for (int j = 0; j < 4 * HALVES; ++j) {
                const int t = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
                const uint32_t there = here.ok[j >> 2] && t >= w.lo && t < end ? ~0u : 0u;
                #pragma unroll
                for (int ch = 0; ch < CH; ++ch)
                    #pragma unroll
                    for (int i = 0; i < DL / 2; ++i) {
                        const uint32_t u = v[ch][j][i] & there, x = lg_not_finite(u);
                        odd |= x;
                        v[ch][j][i] = u & ~(x * 0xFFFFu);
                    }
            }
        }
        #pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            #pragma unroll
            for (int i = 0; i < DL; ++i) {
                const part b = turned(v, ch, i);
                #pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    acc[rt][ch * DL + i] = product(hi[rt], b, acc[rt][ch * DL + i]);
                    acc[rt][ch * DL + i] = product(lo[rt], b, acc[rt][ch * DL + i]);
                }
            }
        stay();
    }
    // values that are not finite, of tiles that not all pairs see whole: NaN for the pairs that see them, found by a product of their own
    if (__any(odd != 0))
        #pragma unroll 1
        for (t0 = t_first; t0 < end; t0 += STEP) {
            const PageTile here = tile_at(t0);
            if (plain(t0, here)) continue;
            values v;
            load_values(here, v);
            uint32_t sees[RT];
            seen_in(t0, here, sees);
            part seen[RT];
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                #pragma unroll
                for (int j = 0; j < 4 * HALVES; ++j) seen[rt][j] = sees[rt] >> j & 1 ? (_Float16)1.0f : (_Float16)0.0f;
            #pragma unroll
            for (int ch = 0; ch < CH; ++ch)
                #pragma unroll
                for (int i = 0; i < DL; ++i) {
                    union { part h; uint32_t u[2 * HALVES]; } b;
                    b.h = turned(v, ch, i);
                    #pragma unroll
                    for (int k = 0; k < 2 * HALVES; ++k) b.u[k] = lg_not_finite(b.u[k]) * 0x3C00u;       // 1 where it is not
                    #pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const lg_f4 mark = product(seen[rt], b.h, (lg_f4){ 0, 0, 0, 0 });
                        #pragma unroll
                        for (int r = 0; r < 4; ++r) if (mark[r] != 0.0f) acc[rt][ch * DL + i][r] = NAN;
                    }
                }
        }
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16);
        l[rt] += __shfl_xor(l[rt], 32);
        if (lane < 16) { s_m[wk][(wr * RT + rt) * 16 + lane] = m[rt]; s_l[wk][(wr * RT + rt) * 16 + lane] = l[rt]; }
    }
    // (behind the loads: lengths and page ids come through the scalar cache as long as nothing has been stored)
    tell();
    // the parts of wavefronts with different keys: their factors and where a pair's output goes, once for each pair; then 16 pairs of every WR at a time
    __syncthreads();
    if ((int)threadIdx.x < ROWS) {
        const int pair = threadIdx.x, p = p0 + pair, node = p / G, head = kvh * G + p - node * G;
        float M = -INFINITY, L = 0;
        #pragma unroll
        for (int u = 0; u < WK; ++u) M = fmaxf(M, s_m[u][pair]);
        #pragma unroll
        for (int u = 0; u < WK; ++u) {
            const float lv = s_l[u][pair], f = lv == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s_m[u][pair] - M);       // (0: no key; a score of NaN leaves its mark in the sum)
            L += f * lv;
            s_m[u][pair] = f;
        }
        const long long place = ((long long)at * a.max_tree + node) * a.H + head;
        s_l[0][pair] = n_split > 1 ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;
        s_to[pair] = p >= n_pairs ? -1 : n_split == 1 ? (w.row0 + node) * a.out_stride + (long long)head * HD : place * HD;
        if (n_split > 1 && p < n_pairs) { a.pm[place] = M; a.pl[place] = L; }
    }
    float *const to = n_split == 1 ? a.out : a.pacc;
    const bool wide = n_split > 1 || (((uintptr_t)a.out | (uintptr_t)a.out_stride * 4) & 15) == 0;
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt) __syncthreads();                    // (the sums' readers of the 16 before)
        #pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            #pragma unroll
            for (int r = 0; r < 4; ++r)
                #pragma unroll
                for (int i = 0; i < DL; i += 4)
                    *(float4 *)&s.o[wave][4 * g + r][ch * 128 + c * DL + i] = make_float4(acc[rt][ch * DL + i][r], acc[rt][ch * DL + i + 1][r], acc[rt][ch * DL + i + 2][r], acc[rt][ch * DL + i + 3][r]);
        __syncthreads();
        constexpr int SUMS = WR * 16 * (HD / 4), EACH = (SUMS + LG_PA_WAVES * 64 - 1) / (LG_PA_WAVES * 64);
        #pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int id = threadIdx.x + k * LG_PA_WAVES * 64, x = id / (HD / 4), d = id % (HD / 4) * 4, r = x / 16, pair = (r * RT + rt) * 16 + x % 16;
            static_assert(SUMS % (LG_PA_WAVES * 64) == 0, "one for each thread in every round");
            lg_f4 o = { 0, 0, 0, 0 };
            #pragma unroll
            for (int u = 0; u < WK; ++u) o += s_m[u][pair] * *(const lg_f4 *)&s.o[u * WR + r][x % 16][d];
            o *= s_l[0][pair];
            const long long base = s_to[pair];
            if (base < 0) continue;
            float *const z = to + base + d;
            if (wide) *(lg_f4 *)z = o;
            else
                #pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = o[i];
        }
    }
}

// The same for more than 32 pairs, where there is much to read: their wavefronts share keys and values through LDS.  From memory to registers each of them would ask for the same rows again, and rows of keys as operands are asked for
// in 16 pieces of 64 bytes, for which the memory pipeline takes four times as long as for whole rows; here a tile of 32 keys and values goes to LDS once, by loads that pass no
// register, while the tile before is worked on.  Queries stay in registers: a wavefront takes 16 pairs, and all keys, so that nothing is joined in the end.
// Measured: 24 trees of up to 64 rows over up to 8192 tokens, heads of 256 (159 MB of keys and values, 57 GFLOP issued) 87.5 us in a row of calls, and 7.6 the joining launch behind it (121 in lg_k_tree_attn's groups of 32 pairs;
// 95 and more by itself under a profiler).  Without the loads of later tiles it would take 79, and those alone 41; its matrix units are busy a quarter of the time, its compute units three quarters, since splits are of 31 tiles where 26
// would be even.  64 trees of 16 over 4096 tokens 129 us, 537 MB, of which loads alone take 116: a workgroup's loads drain at each tile's barrier.
// Tried: values read once a workgroup, by wavefronts that take a quarter of the dimensions for all pairs and get the probabilities through LDS (heads of 256 131 -> 123 us and 99 -> 97, but heads of 64 28 -> 32, 128 38 -> 41,
// 512 137 -> 236); 32 pairs to a wavefront (spills); loads of the next tile between score steps, four chains of scores, priorities around products (nothing).
// A row's 16-byte pieces lie in LDS in an order of the row's own (piece j ^ swap), so that reads of a column of 16 rows touch all banks.
constexpr int lg_wide_per_simd(int hd) { return hd <= 256 ? 2 : 1; }
// 16 bytes of each lane, from a common place and its own distance behind it, to LDS, one after another from byte `to` on
__device__ __forceinline__ void lg_to_lds(const void *from, uint32_t behind, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(to), "v"(behind), "s"(from) : "m0", "memory");
}
template <int HD>
__global__ __launch_bounds__(LG_PA_WAVES * 64, lg_wide_per_simd(HD)) void lg_k_tree_wide(TreeAttn a) {
    constexpr int KS = HD / 32;                     // score steps
    constexpr int NT = HD / 16;                     // output tiles
    constexpr int TILE = LG_PA_TILE, ROWS = 16 * LG_PA_WAVES;
    constexpr int PIECES = HD / 8, AT_ONCE = 64 / PIECES, LOADS = TILE / AT_ONCE / LG_PA_WAVES;      // 16-byte pieces of a row; rows of a load; loads of a wavefront for a tile's keys, and for its values
    constexpr int TURN = 64 + 4;                    // floats between rows of the outputs' turn: no two of a column in a bank
    __shared__ __align__(16) union { uint16_t kv[2][2][TILE * HD]; float turn[LG_PA_WAVES][16][TURN]; } s;
    __shared__ int32_t s_pos[LG_TREE_ROWS];
    const int number = lg_tree_number(blockIdx.x), kvh = number / a.items, G = a.H / a.nkv;
    if (kvh >= a.nkv) return;
    const TreePart cut = lg_tree_part(a, number % a.items);
    const int seq = __builtin_amdgcn_readfirstlane(cut.seq);
    if (seq < 0) return;
    const TreeSeq w = lg_tree_seq(a, seq);
    const int group = __builtin_amdgcn_readfirstlane(cut.group), at = __builtin_amdgcn_readfirstlane(cut.first + cut.index), n_pairs = w.n * G, p0 = group * ROWS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int chunk = __builtin_amdgcn_readfirstlane(cut.tiles) * LG_PA_TILE, n_split = __builtin_amdgcn_readfirstlane(cut.n);
    auto tell = [&]() {                             // the joining launch
        if (a.pm && a.n_seq <= LG_PA_LANES && kvh == 0 && cut.index == 0 && group == 0 && threadIdx.x == 0) {
            a.cut[seq] = cut.first;
            if (seq == a.n_seq - 1) a.cut[a.n_seq] = cut.first + cut.n;
        }
    };
    if (p0 >= n_pairs) { tell(); return; }
    const int32_t *table = a.table + (long long)seq * a.max_blocks;
    const int first = (w.lo & ~(LG_PA_TILE - 1)) + __builtin_amdgcn_readfirstlane(cut.index) * chunk, end = w.len < first + chunk ? w.len : first + chunk;
    const int b0 = first >> a.g.shift;
    // page ids of the stretch, a lane each
    static_assert(LG_PA_CHUNK / 16 + 1 <= 192, "in three registers");
    auto id_of = [&](int i) { return i <= ((end - 1) >> a.g.shift) - b0 && b0 + i < a.max_blocks ? table[b0 + i] : -1; };
    const int ids0 = id_of(lane), ids1 = id_of(64 + lane), ids2 = id_of(128 + lane);
    const int n_ids = ((end - 1) >> a.g.shift) - b0 + 1;
    auto is_page = [&](int id) { return id >= 0 && id < a.g.n_pages; };
    const bool all_there = __ballot((lane < n_ids && !is_page(ids0)) || (64 + lane < n_ids && !is_page(ids1)) || (128 + lane < n_ids && !is_page(ids2))) == 0;
    auto id_at = [&](int t) {
        const int i = (t >> a.g.shift) - b0;
        int x = __builtin_amdgcn_readlane(ids0, i & 63);
        if (n_ids > 64) { const int y = __builtin_amdgcn_readlane(ids1, i & 63), z = __builtin_amdgcn_readlane(ids2, i & 63); x = i < 64 ? x : i < 128 ? y : z; }
        return x;
    };
    // a tile, for this wavefront: which half tiles are there, and where the half that it fetches from begins
    constexpr int OWN = TILE / LG_PA_WAVES;         // its rows
    const int half = wave * OWN / 16;
    struct Tile { long long row; bool ok[2]; };
    auto tile_at = [&](int t) {
        Tile p;
        const int mine = t + 16 * half, id = id_at(mine < end ? mine : t);      // (a half behind the end is masked)
        p.row = (is_page(id) ? id : 0) * a.g.page_stride + (mine & ((1 << a.g.shift) - 1)) * a.g.row_stride;
        p.ok[0] = p.ok[1] = true;
        if (!all_there) { p.ok[0] = is_page(id_at(t)); p.ok[1] = is_page(id_at(t + 16 < end ? t + 16 : t)); }
        return p;
    };

    auto swap = [](int row) { return HD == 64 ? row >> 1 & 7 : row & 15; };
    // of its loads: the lane's row and piece, in bytes behind the half tile's first row (rows are at most 2^27 values apart: 32 bits)
    uint32_t behind[LOADS];
    #pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int row = (wave * OWN + i * AT_ONCE + lane / PIECES) & 15;
        behind[i] = (uint32_t)row * (uint32_t)(a.g.row_stride * 2) + (uint32_t)((lane % PIECES) ^ swap(row)) * 16;
    }
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t *)&s.kv[0][0][0] + (uint32_t)(wave * OWN * HD * 2);
    const uint16_t *const keys_of = a.g.k + kvh * HD, *const values_of = a.g.v + kvh * HD;
    auto fetch = [&](const Tile &p, int buffer) {
        const uint32_t to = lds + (uint32_t)(buffer * 2 * TILE * HD * 2);
        #pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            lg_to_lds(keys_of + p.row, behind[i], to + i * AT_ONCE * HD * 2);
            lg_to_lds(values_of + p.row, behind[i], to + i * AT_ONCE * HD * 2 + TILE * HD * 2);
        }
    };
    Tile now;
    if (first < end) { now = tile_at(first); fetch(now, 0); }
    if ((int)threadIdx.x < w.n) s_pos[threadIdx.x] = a.pos[w.row0 + threadIdx.x];

    // queries of the wavefront's pairs, as operands
    lg_h8 q[KS][2];
    float qs;                                       // factor of the raw scores: base-2 exponents
    int lo_row, whole = w.lo;                       // of pair c: the first position that it sees, and its set
    lg_u64 set;
    const int pair = p0 + wave * 16 + c, x = pair < n_pairs ? pair : p0, row = w.row0 + x / G;
    const float *src = a.q + row * a.q_stride + (long long)(kvh * G + x % G) * HD + g * 8;
    float4 v[KS][2];
    #pragma unroll
    for (int i = 0; i < KS; ++i)
        #pragma unroll
        for (int j = 0; j < 2; ++j) v[i][j] = *(const float4 *)(src + i * 32 + j * 4);
    const int pos = a.pos[row];
    set = pos < w.done ? 0 : a.mask[row] & (w.n < 64 ? (1ull << w.n) - 1 : ~0ull);
    lo_row = pos < w.done ? INT32_MAX : a.window > 0 ? pos - a.window + 1 : INT32_MIN;
    if (pair < n_pairs && lo_row > whole) whole = lo_row;
    float top = 0;
    #pragma unroll
    for (int i = 0; i < KS; ++i)
        #pragma unroll
        for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(fmaxf(fabsf(v[i][j].x), fabsf(v[i][j].y)), fmaxf(fabsf(v[i][j].z), fabsf(v[i][j].w))));
    top = lg_max_of_rows(top);
    int e = (int)(__float_as_uint(top) >> 23) - 127 - 14;         // top * 2^-e in [2^14, 2^15)
    if (e < -100) e = -100;                                       // (zero and tiny rows; 2^-e stays a float)
    const float up = __uint_as_float((unsigned)(127 - e) << 23);
    #pragma unroll
    for (int i = 0; i < KS; ++i) {
        const float y[8] = { v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w, v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w };
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float z = y[j] * up;
            q[i][0][j] = (_Float16)z;
            q[i][1][j] = (_Float16)(z - (float)q[i][0][j]);
        }
    }
    qs = a.scale * 1.44269504088896341f * __uint_as_float((unsigned)(127 + e) << 23);
    lg_barrier_lds();                               // (positions)
    // tiles in [whole, w.done) need no mask; rows of the tree in front of a window are taken out of the sets
    lg_tree_trim(a, w, s_pos, whole, [&](int pos, lg_u64 row) { if (pos < lo_row) set &= ~row; });

    const bool busy = p0 + wave * 16 < n_pairs;     // (a wavefront without pairs only fetches)
    lg_f4 acc[NT];
    float m, l;                                     // of pair c; l of this lane's keys alone
    auto clear = [&]() {
        m = -INFINITY; l = 0;
        #pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = (lg_f4){ 0, 0, 0, 0 };
    };
    auto plain = [&](int t, const Tile &p) { return t >= whole && t + TILE <= w.done && t + TILE <= end && p.ok[0] && p.ok[1]; };
    auto seen_in = [&](int t0, const Tile &p) {
        uint32_t sees = 0;
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const LgQuad x = lg_tree_quad(t0 + 16 * h + 4 * g, w.done, p.ok[h] ? end : 0);
            sees |= lg_tree_sees(x, lo_row, set) << (4 * h);
        }
        return sees;
    };
    // where a lane reads, in values: its piece of a key row differs from that of the step before by a piece's place, of those 4 (2) steps before by a whole number of rounds
    constexpr int KEY_AT = KS < 4 ? KS : 4;
    int at_key[KEY_AT];
    #pragma unroll
    for (int i = 0; i < KEY_AT; ++i) at_key[i] = c * HD + ((4 * i + g) ^ swap(c)) * 8;
    // Values of 16 dimensions: sixteen lanes give the places of four values each of four keys' rows, and get four keys of one dimension each (ds_read_b64_tr_b16).  A round of places takes VAL_AT tiles
    constexpr int VAL_AT = HD == 64 ? 4 : 8;
    int at_val[VAL_AT];
    #pragma unroll
    for (int i = 0; i < VAL_AT; ++i) { const int row = 4 * g + (c >> 2); at_val[i] = row * HD + ((2 * i + (c >> 1 & 1)) ^ swap(row)) * 8 + (c & 1) * 4; }
    typedef short lg_s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) lg_s4 lds_s4;
    union operand { lg_s4 s[2]; uint32_t u[4]; lg_h8 h; };
    // A value that is infinite or NaN reaches rows that do not see it as 0 * inf: found in the end, by sums that are not finite, and then all is done again with such values taken out of the products and marked by
    // products of their own
    auto run = [&](auto safe) {
    constexpr bool SAFE = decltype(safe)::value;
    clear();
    int buffer = 0;
    for (int t0 = first; t0 < end; t0 += TILE, buffer ^= 1) {
        // this tile has arrived, and every wavefront has done with the one before
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const Tile here = now;
        if (t0 + TILE < end) { now = tile_at(t0 + TILE); fetch(now, buffer ^ 1); }
        if (!busy) continue;
        const uint16_t *const keys = s.kv[buffer][0], *const vals = s.kv[buffer][1];
        lg_f4 sc[2] = {};
        constexpr int DEEP = KS < 3 ? 2 : 3;     // key operands on their way
        lg_h8 kf[DEEP][2];
        auto ask = [&](int i) {
            #pragma unroll
            for (int h = 0; h < 2; ++h) kf[i % DEEP][h] = *(const lg_h8 *)(keys + at_key[i % KEY_AT] + (i / KEY_AT) * KEY_AT * 32 + h * 16 * HD);
        };
        #pragma unroll
        for (int i = 0; i < DEEP - 1; ++i) ask(i);
        #pragma unroll
        for (int i = 0; i < KS; ++i) {
            if (i + DEEP - 1 < KS) ask(i + DEEP - 1);
            __builtin_amdgcn_sched_barrier(0);
            #pragma unroll
            for (int x = 0; x < 2; ++x)
                #pragma unroll
                for (int h = 0; h < 2; ++h) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i % DEEP][h], q[i][x], sc[h], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        constexpr int FAR = NT / 4 < 3 ? NT / 4 : 3;          // groups of values on their way
        operand b[FAR][4];
        auto ask_values = [&](int n) {              // four tiles of 16 dimensions
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                #pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int tile = 4 * n + i;
                    b[n % FAR][i].s[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(vals + at_val[tile % VAL_AT] + tile / VAL_AT * VAL_AT * 16 + h * 16 * HD));
                }
        };
        #pragma unroll
        for (int n = 0; n < FAR - 1 || n < 1; ++n) ask_values(n);
        __builtin_amdgcn_sched_barrier(0);
        const bool masked = !plain(t0, here);
        #pragma unroll
        for (int h = 0; h < 2; ++h) sc[h] *= qs;
        uint32_t sees;
        if (masked) {
            sees = seen_in(t0, here);
            #pragma unroll
            for (int j = 0; j < 8; ++j) if (!(sees >> j & 1)) sc[j >> 2][j & 3] = -INFINITY;
        }
        float top = -INFINITY;
        #pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, sc[j >> 2][j & 3]);
        top = lg_max_of_rows(top);
        if (__any(lg_tree_passes(top, m))) {
            const float mn = fmaxf(m, lg_tree_base(top));
            const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);       // (both -inf: nothing seen yet)
            l *= f; m = mn;
            float fr[4];
            #pragma unroll
            for (int r = 0; r < 4; ++r) fr[r] = __shfl(f, 4 * g + r);
            #pragma unroll
            for (int i = 0; i < NT; ++i)
                #pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][r] *= fr[r];
        }
        lg_h8 hi, lo;
        lg_tree_parts(sc, m, l, hi, lo);
        // keys that are not there may hold anything: zeros in their place
        const bool partly = t0 < w.lo || t0 + TILE > end || !here.ok[0] || !here.ok[1];
        uint32_t there[4];
        if (partly)
            #pragma unroll
            for (int k = 0; k < 4; ++k) {           // keys 4 g + 2 (k % 2) and the next of half k / 2
                const int t = t0 + 16 * (k >> 1) + 4 * g + 2 * (k & 1);
                there[k] = !here.ok[k >> 1] ? 0u : (t >= w.lo && t < end ? 0xFFFFu : 0u) | (t + 1 >= w.lo && t + 1 < end ? 0xFFFF0000u : 0u);
            }
        #pragma unroll
        for (int n = 0; n < NT / 4; ++n) {          // (four sums in turn: a product waits for the one before it into the same sum)
            if (FAR > 1 && n + FAR - 1 < NT / 4) ask_values(n + FAR - 1);
            __builtin_amdgcn_sched_barrier(0);
            operand (&v)[4] = b[n % FAR];
            if (partly)
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) v[i].u[k] &= there[k];
            if (SAFE && masked)
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    operand odd;
                    #pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = lg_not_finite(v[i].u[k]);
                        v[i].u[k] &= ~(x * 0xFFFFu);
                        odd.u[k] = x * 0x3C00u;                   // 1 where it is not finite
                    }
                    lg_h8 seen;
                    #pragma unroll
                    for (int j = 0; j < 8; ++j) seen[j] = sees >> j & 1 ? (_Float16)1.0f : (_Float16)0.0f;
                    const lg_f4 mark = __builtin_amdgcn_mfma_f32_16x16x32_f16(seen, odd.h, (lg_f4){ 0, 0, 0, 0 }, 0, 0, 0);
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) if (mark[r] != 0.0f) acc[4 * n + i][r] = NAN;
                }
            #pragma unroll
            for (int x = 0; x < 2; ++x)
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[4 * n + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x ? lo : hi, v[i].h, acc[4 * n + i], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    };
    run(std::false_type{});
    float finite = 0;                               // or NaN
    #pragma unroll
    for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int r = 0; r < 4; ++r) finite = __builtin_fmaf(acc[n][r], 0.0f, finite);
    if (__syncthreads_or(finite != 0.0f)) {
        now = tile_at(first);
        fetch(now, 0);
        run(std::true_type{});
    }
    tell();
    __syncthreads();                                // (the last tile's readers)
    if (!busy) return;
    float total = l;
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
    // outputs turned in LDS, each wavefront by itself, for stores of 16 bytes: 16 pairs of 64 dimensions at a time
    float (&turn)[16][TURN] = s.turn[wave];
    const bool aligned = n_split > 1 || (((uintptr_t)a.out | (uintptr_t)a.out_stride * 4) & 15) == 0;
    float *to[4], by[4];                            // of pairs 4 k + g
    #pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int p = p0 + wave * 16 + 4 * k + g, node = p / G, head = kvh * G + p - node * G;
        const float L = __shfl(total, 4 * k + g);
        to[k] = p >= n_pairs ? nullptr : (n_split == 1 ? a.out + (w.row0 + node) * a.out_stride + (long long)head * HD : a.pacc + (((long long)at * a.max_tree + node) * a.H + head) * HD) + c * 4;
        by[k] = n_split > 1 ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L;
    }
    #pragma unroll
    for (int n = 0; n < NT; n += 4) {
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            #pragma unroll
            for (int r = 0; r < 4; ++r) turn[4 * g + r][i * 16 + c] = acc[n + i][r];
        lg_f4 y[4];
        #pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = *(const lg_f4 *)&turn[4 * k + g][c * 4] * by[k];
        #pragma unroll
        for (int k = 0; k < 4; ++k)
            if (to[k]) {
                if (aligned) *(lg_f4 *)(to[k] + n * 16) = y[k];
                else
                    #pragma unroll
                    for (int i = 0; i < 4; ++i) to[k][n * 16 + i] = y[k][i];
            }
    }
    const int p = p0 + wave * 16 + lane;
    if (n_split > 1 && lane < 16 && p < n_pairs) {
        const long long place = ((long long)at * a.max_tree + p / G) * a.H + kvh * G + p % G;
        a.pm[place] = m; a.pl[place] = total;
    }
}
