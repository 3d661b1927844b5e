// lg_tree.h — trees of drafted tokens over a cache in pages: ancestors and positions of their rows, the accepted path, and attention of all rows of a tree.
//
// The n rows of a sequence's tree stand behind its committed positions: row k's K and V at position committed + k, committed = len - n.  Row 0 is the token chosen
// last, every other row hangs on an earlier one, its parent.  Row r of the tree is row start[i] + r of the step.
#pragma once

#include "lg_pages.h"

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
// A wavefront to a tree, a lane to a row.  Both are chains of a few hundred clocks behind two round trips to memory.
#define LG_TREE_WG 256
// anc(j) = anc(parent j) + {j}: every lane takes over what the row it points at has reached, then points where that one points; the reach doubles, so six steps do for 64 rows.
__global__ __launch_bounds__(LG_TREE_WG) void lg_k_tree_plan(const int32_t *start, const int32_t *parent, const int32_t *len, lg_u64 *mask, int32_t *pos, int32_t *seq_of,
                                                            int32_t *status, int n_seq, int n_rows, int max_tree) {
    const int seq = (int)(blockIdx.x * (LG_TREE_WG / 64) + (threadIdx.x >> 6)), j = threadIdx.x & 63;
    if (seq >= n_seq) return;
    const TreeRows w = lg_tree_rows(start, seq, n_rows, max_tree);
    const int total = len[seq];
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
// From row 0 on to the first row behind the current one that hangs on it and carries the token picked after it, as long as there is one
__global__ __launch_bounds__(LG_TREE_WG) void lg_k_tree_accept(const int32_t *start, const int32_t *parent, const int32_t *token, const int32_t *next, const int32_t *len,
                                                              int32_t *path, int32_t *count, int32_t *len_out, int32_t *last, int n_seq, int n_rows, int max_tree) {
    const int seq = (int)(blockIdx.x * (LG_TREE_WG / 64) + (threadIdx.x >> 6)), j = threadIdx.x & 63;
    if (seq >= n_seq) return;
    const TreeRows w = lg_tree_rows(start, seq, n_rows, max_tree);
    const int total = len[seq];
    const bool live = j < w.n;
    const int up = live ? parent[w.row0 + j] : -1, tok = live ? token[w.row0 + j] : -1, picked = live ? next[w.row0 + j] : -1;
    int cur = 0, n = 0, mine = -1, want = -1;
    if (w.n > 0) {
        for (;;) {                                            // (rows only rise: at most 64 rounds)
            if (j == n) mine = cur;
            ++n;
            want = __builtin_amdgcn_readlane(picked, cur);
            const lg_u64 fits = __ballot(live && j > cur && up == cur && tok == want && want >= 0);
            if (!fits) break;
            cur = (int)__builtin_ctzll(fits);
        }
    }
    if (j < max_tree) path[(long long)seq * max_tree + j] = mine;
    if (j == 0) {
        count[seq] = n;
        len_out[seq] = w.n > 0 ? total - w.n + n : total;
        last[seq] = want;
    }
}

// ---- attend ----------------------------------------------------------------------------------------------------------
// o[j, h] = sum_t softmax_t(scale q[j, h].k[t]) v[t] over the committed positions t of a row's window and the rows of its tree that its set names.
//
// A workgroup takes a stretch of keys of one key head and up to ROWS = 16 RT of the n G (row, query head) pairs that share them; its four wavefronts take tiles of 32 keys in
// turn, as lg_k_page_attn does, and for the same reason no key or value passes through LDS: a lane's 16 bytes of a key row are the operand of the scores as they lie in memory, and the 8 x 8 values
// that a lane loads are turned in registers, here once for all pairs.
// Queries and probabilities are f32 and keep their precision as two binary16 parts (22 bits together) whose products go into one sum: two instructions for each 16 pairs, where the one-row
// kernel puts the second part into rows that it has anyway.  Queries lie in LDS as operands; maxima, sums and outputs are in f32.
// A tile that all pairs see whole (every tile but those at a window's border and of the tree) has no mask.  In the others a value that is infinite or NaN must not reach rows that
// do not see it through 0 * inf: it is taken out of the product and marked by a product of its own.
struct TreeAttn : PageAttn {        // len: with the tree's rows
    const int32_t *start, *pos;
    const lg_u64 *mask;
    int n_rows, max_tree, groups, units;        // groups of ROWS pairs; stretches of keys: splits x key heads
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
__device__ __forceinline__ MergeRow lg_merge_row(const TreeAttn &a) {
    const int seq = blockIdx.y, node = blockIdx.x / a.H, head = blockIdx.x % a.H;
    const TreeRows w = lg_tree_rows(a.start, seq, a.n_rows, a.max_tree);
    return { seq, node < w.n ? (long long)w.row0 + node : -1, (long long)a.max_tree * a.H, blockIdx.x, head };
}

// Probabilities are 2^(x - m + SHIFT).  m is the largest score of a while ago, rounded up to a whole number (m - SHIFT and factors between two of them are exact): it is taken anew, and the sums so far scaled,
// only when a score passes it by SLACK, which few tiles of a long row do.  So they stay below 2^15 in binary16, and what their two parts leave of a small one is at most 2^-32 of the largest
#define LG_TREE_SLACK 7.0f
#define LG_TREE_SHIFT 8.0f
// 1 in each half of a pair of binary16 values that is infinite or NaN (all bits of the exponent: one more carries into the sign's place)
__device__ __forceinline__ uint32_t lg_not_finite(uint32_t u) { return ((u & 0x7C007C00u) + 0x04000400u) >> 15 & 0x00010001u; }
// How the four wavefronts of a workgroup share its work: WR of them take 16 RT pairs each, the others different keys
constexpr int lg_tree_per_simd(int hd, int rt) { return hd * rt <= 128 ? 3 : hd * rt <= 256 ? 2 : 1; }
template <int HD, int RT, int WR>
__global__ __launch_bounds__(LG_PA_WAVES * 64, lg_tree_per_simd(HD, RT)) void lg_k_tree_attn(TreeAttn a) {
    constexpr int KS = HD / 32;                     // score steps
    constexpr int DL = HD >= 128 ? 8 : HD / 16;     // dimensions of a value load
    constexpr int CH = HD / (16 * DL);              // value loads of a key row
    constexpr int NT = HD / 16;                     // output tiles
    constexpr int HALVES = HD > 256 ? 1 : 2, TILE = 16 * HALVES, ROWS = 16 * RT * WR, WK = LG_PA_WAVES / WR;
    __shared__ float s_m[WK][ROWS], s_l[WK][ROWS], s_top[LG_PA_WAVES][ROWS];
    __shared__ __align__(16) union { lg_h8 q[RT * WR][KS][2][64]; float o[LG_PA_WAVES][16][HD]; } s;
    __shared__ int32_t s_ids[LG_PA_CHUNK / 16 + 1], s_pos[LG_TREE_ROWS];
    // The groups of one stretch of keys run on one XCD at a time (workgroups are dealt over 8 of them in turn): what the first asks for is in its L2 for the others
    const int line = blockIdx.x >> 3, unit = line / a.groups * 8 + (blockIdx.x & 7), group = line % a.groups;
    if (unit >= a.units) return;
    const int kvh = unit % a.nkv, G = a.H / a.nkv, at = unit / a.nkv;
    const PageCut cut = lg_pa_cut(a, at);
    const int seq = __builtin_amdgcn_readfirstlane(cut.seq);
    if (seq < 0) return;
    const TreeSeq w = lg_tree_seq(a, seq);
    const int n_pairs = w.n * G, p0 = group * ROWS;
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
    if ((int)threadIdx.x < w.n) s_pos[threadIdx.x] = a.pos[w.row0 + threadIdx.x];
    if (has_id) s_ids[threadIdx.x] = my_id;
    auto tile_at = [&](int t) {
        PageIds p;
        #pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = ((t + 16 * h < end ? t + 16 * h : t) >> a.g.shift) - b0;             // (a half behind the end is masked)
            p.id[h] = __builtin_amdgcn_readfirstlane(s_ids[i]);
        }
        return lg_pa_tile(a, p, t, kvh * HD);
    };
    float qs[RT];                                   // factor of the raw scores: base-2 exponents
    {
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
    }
    // tiles in [whole, w.done) need no mask; rows of the tree in front of a window are taken out of the sets
    #pragma unroll
    for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(whole, o); if (x > whole) whole = x; }
    whole = __builtin_amdgcn_readfirstlane(whole);
    if (whole > w.done)
        #pragma unroll 1
        for (int k = 0; k < w.n; ++k) {
            const int pos = s_pos[k];
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) if (pos < lo_row[rt]) set[rt] &= ~(1ull << k);
        }

    lg_h8 kf[HALVES][KS];
    PageTile now;
    auto load_keys = [&](const PageTile &p) {
        #pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const uint16_t *kp = a.g.k + p.row[h] + c * a.g.row_stride + g * 8;
            #pragma unroll
            for (int i = 0; i < KS; ++i) kf[h][i] = *(const lg_h8 *)(kp + i * 32);
        }
    };
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
    int t0 = p0 + wr * RT * 16 < n_pairs ? first + wk * TILE : end;      // (no pairs: nothing to do)
    if (t0 < end) { now = tile_at(t0); load_keys(now); }
    lg_f4 acc[RT][NT];
    float m[RT], l[RT];                             // of pair c; l of this lane's keys alone
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY; l[rt] = 0;
        #pragma unroll
        for (int i = 0; i < NT; ++i) acc[rt][i] = (lg_f4){ 0, 0, 0, 0 };
    }
    typedef _Float16 lg_h2 __attribute__((ext_vector_type(2)));
    typedef float lg_f2 __attribute__((ext_vector_type(2)));
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
        auto below = [](int x) { return (1u << (x < 0 ? 0 : x > 4 ? 4 : x)) - 1; };
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) sees[rt] = 0;
        #pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const int t = t0 + 16 * h + 4 * g, k = t - w.done;
            const uint32_t there = p.ok[h] ? below(end - t) : 0u, old = below(-k);
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int ahead = lo_row[rt] < t ? 0 : lo_row[rt] > t + 4 ? 4 : lo_row[rt] - t;
                const uint32_t tree = k <= -4 || k > 63 ? 0u : k < 0 ? (uint32_t)set[rt] << (-k & 3) : (uint32_t)(set[rt] >> (k & 63));
                sees[rt] |= (((old & ~below(ahead)) | (tree & ~old)) & there & 15u) << (4 * h);
            }
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
            higher |= top[rt] > m[rt] + LG_TREE_SLACK;
        }
        if (__any(higher)) {
            if constexpr (ALONE) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");           // (products write accumulation registers up to 16 cycles after they are issued; out_of reads them where the compiler does not see it)
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float mn = fmaxf(m[rt], ceilf(top[rt]));
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
        for (int rt = 0; rt < RT; ++rt) {
            const float under = (m[rt] == -INFINITY ? 0.0f : m[rt]) - LG_TREE_SHIFT;
            #pragma unroll
            for (int j = 0; j < 4 * HALVES; j += 2) {
                lg_f2 p, left;
                #pragma unroll
                for (int k = 0; k < 2; ++k) { p[k] = __builtin_amdgcn_exp2f(sc[rt][j >> 2][j + k & 3] - under); l[rt] += p[k]; }
                const lg_h2 h = __builtin_convertvector(p, lg_h2);
                #pragma unroll
                for (int k = 0; k < 2; ++k) left[k] = __builtin_fmaf((float)h[k], -1.0f, p[k]);
                const lg_h2 u = __builtin_convertvector(left, lg_h2);
                #pragma unroll
                for (int k = 0; k < 2; ++k) { hi[rt][j + k] = h[k]; lo[rt][j + k] = u[k]; }
            }
        }
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
    // the parts of wavefronts with different keys, 16 pairs of every WR at a time
    const bool wide = (((uintptr_t)a.out | (uintptr_t)a.out_stride * 4) & 15) == 0;
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        __syncthreads();                            // (the queries' last reader; the sums' of the 16 before)
        #pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            #pragma unroll
            for (int r = 0; r < 4; ++r)
                #pragma unroll
                for (int i = 0; i < DL; i += 4)
                    *(float4 *)&s.o[wave][4 * g + r][ch * 128 + c * DL + i] = make_float4(acc[rt][ch * DL + i][r], acc[rt][ch * DL + i + 1][r], acc[rt][ch * DL + i + 2][r], acc[rt][ch * DL + i + 3][r]);
        __syncthreads();
        #pragma unroll 4
        for (int id = threadIdx.x; id < WR * 16 * (HD / 4); id += LG_PA_WAVES * 64) {
            const int x = id / (HD / 4), d = id % (HD / 4) * 4, r = x / 16, pair = (r * RT + rt) * 16 + x % 16, p = p0 + pair;
            float M = -INFINITY, L = 0;
            float4 o = make_float4(0, 0, 0, 0);
            #pragma unroll
            for (int u = 0; u < WK; ++u) M = fmaxf(M, s_m[u][pair]);
            #pragma unroll
            for (int u = 0; u < WK; ++u) {
                const float lv = s_l[u][pair], f = lv == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s_m[u][pair] - M);       // (0: no key; a score of NaN leaves its mark in the sum)
                const float4 y = *(const float4 *)&s.o[u * WR + r][x % 16][d];
                L += f * lv;
                o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w;
            }
            if (p >= n_pairs) continue;
            const int node = p / G, head = kvh * G + p % G;
            if (n_split == 1) {
                float *const to = a.out + (w.row0 + node) * a.out_stride + (long long)head * HD + d;
                const float4 y = L == 0.0f ? make_float4(0, 0, 0, 0) : make_float4(o.x / L, o.y / L, o.z / L, o.w / L);
                if (wide) *(float4 *)to = y;
                else { to[0] = y.x; to[1] = y.y; to[2] = y.z; to[3] = y.w; }
            } else {
                const long long place = ((long long)at * a.max_tree + node) * a.H + head;
                *(float4 *)(a.pacc + place * HD + d) = o;
                if (d == 0) { a.pm[place] = M; a.pl[place] = L; }
            }
        }
    }
}
