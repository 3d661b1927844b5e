// lg_pages.h — a KV cache in pages that many sequences share: its bookkeeping, the rows of new tokens, and attention of one new token per sequence.
//
// Position t of sequence i is row t % P of page table[i][t / P] (P = page_size, a power of two of 16..256).  Free pages lie on a stack.
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>
#include <type_traits>

#include "lg_block.h"

#define LG_PLAN_SEQS 4096           // sequences of a plan: their running sums lie in LDS

// ---- plan ------------------------------------------------------------------------------------------------------------
enum { LG_PLAN_BAD_LEN = 1, LG_PLAN_NO_PAGES = 2, LG_PLAN_NO_SLOTS = 4, LG_PLAN_BAD_STACK = 8, LG_PLAN_BAD_PAGE = 16 };   // LG_HIP_PLAN_* of lg_hip.h

struct PlanArgs {
    const int32_t *len_old, *len_new;   // [n_seq]
    int32_t *table;                     // [n_seq][max_blocks]
    int32_t *stack, *n_free;            // [n_pages], its height
    int32_t *start;                     // [n_seq + 1]
    int32_t *slots;                     // [n_slots]
    int32_t *status;
    int n_seq, shift, n_pages, max_blocks, n_slots;
};

// The sequence that entry e belongs to: sums[i] <= e < sums[i + 1]
__device__ __forceinline__ int lg_owner(const int32_t *sums, int n, int e, int lo = 0) {        // it is one of lo .. n
    int hi = n;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (sums[mid + 1] <= e) lo = mid + 1; else hi = mid; }
    return lo;
}

// Lengths before and after a step -> pages and slots.  With nb(l) = ceil(l / P), sequence i returns max(0, nb(old) - nb(new)) pages and takes
// max(0, nb(new) - nb(old)); all returned pages go on the stack first, the first one topmost, then the needed ones are taken from its top in
// order, so that the plan with the lengths exchanged undoes this one exactly: needed page e is returned page e as long as there are those.  All or
// nothing: whatever *status reports leaves table and stack alone.
// One workgroup, of NT threads: the step is a few thousand words (64 sequences, one new token each: 2 KB), its time a chain of memory round trips.  Where
// every thread has one page and one token at most the chain is lengths, pages, stores: 64 sequences 3.6 us.  Otherwise pages are taken NT at a time, each by a
// search for its sequence and a round trip or two: 333 prompts, together 10000 pages, 9.8 us.  Slots of many tokens are left to lg_k_plan_slots (`slots` null).
template <int NT>
__global__ __launch_bounds__(NT) void lg_k_plan(PlanArgs a) {
    __shared__ int32_t tok[LG_PLAN_SEQS + 1], need[LG_PLAN_SEQS + 1], freed[LG_PLAN_SEQS + 1], olds[LG_PLAN_SEQS], news[LG_PLAN_SEQS];
    __shared__ lg_u64 part[3 * NT / 64];
    __shared__ int32_t taken[NT + 1];
    __shared__ int bad, bad_page;                             // (a word of its own: wavefronts may find pages while others still read the first)
    const int t = threadIdx.x, P = 1 << a.shift, n = a.n_seq, n_slots = a.slots ? a.n_slots : 0;
    const long long most = (long long)a.max_blocks << a.shift;
    const int per = (n + NT - 1) / NT, i0 = t * per;
    const int nf = *a.n_free;
    if (t == 0) { bad = 0; bad_page = 0; }
    auto blocks = [&](int len) { return (int)(((long long)len + P - 1) >> a.shift); };
    auto parts = [&](int i, lg_u64 (&v)[3]) {
        const int lo = olds[i], ln = news[i], d = blocks(ln) - blocks(lo);
        v[0] = ln > lo ? ln - lo : 0; v[1] = d > 0 ? d : 0; v[2] = d < 0 ? -d : 0;
    };
    // running sums: sequences i0 .. i0 + per - 1 are this thread's
    lg_u64 run[3] = { 0, 0, 0 }, all[3], v[3];
    bool wrong = false;
    for (int i = i0; i < i0 + per && i < n; ++i) {
        int lo = a.len_old[i], ln = a.len_new[i];
        if (lo < 0 || ln < 0 || lo > most || ln > most) { wrong = true; lo = ln = 0; }
        olds[i] = lo; news[i] = ln;
        parts(i, v);
        #pragma unroll
        for (int k = 0; k < 3; ++k) run[k] += v[k];
    }
    lg_block_run3<NT>(run, all, part);
    if (wrong) atomicOr(&bad, LG_PLAN_BAD_LEN);
    for (int i = i0; i < i0 + per && i < n; ++i) {            // (used only where the totals fit, below)
        tok[i] = (int32_t)run[0]; need[i] = (int32_t)run[1]; freed[i] = (int32_t)run[2];
        parts(i, v);
        #pragma unroll
        for (int k = 0; k < 3; ++k) run[k] += v[k];
    }
    if (t == 0) {
        tok[n] = (int32_t)all[0]; need[n] = (int32_t)all[1]; freed[n] = (int32_t)all[2];
        if (nf < 0 || nf > a.n_pages || all[2] + nf > (lg_u64)a.n_pages) atomicOr(&bad, LG_PLAN_BAD_STACK);
        else if (all[1] > nf + all[2]) atomicOr(&bad, LG_PLAN_NO_PAGES);
        if (all[0] > (lg_u64)a.n_slots) atomicOr(&bad, LG_PLAN_NO_SLOTS);
    }
    __syncthreads();
    int st = bad;
    const int nt = (int)all[0], nn = (int)all[1], ng = (int)all[2], top = nf + ng;
    auto place = [&](int i, int block) { return a.table + (size_t)i * a.max_blocks + block; };
    auto stands = [&](int i, int e) { return place(i, blocks(news[i]) + e - freed[i]); };     // the e-th returned page, of sequence i
    auto goes = [&](int i, int e) { return place(i, blocks(olds[i]) + e - need[i]); };        // where the e-th needed one goes
    auto outside = [&](int id) { return id < 0 || id >= a.n_pages; };
    auto half_full = [&](int i) { return news[i] > olds[i] && (olds[i] & (P - 1)); };         // its last page is written into
    if (!st && ng <= NT && nn <= NT && n_slots <= NT) {
        // everything is read, then everything is written
        int32_t *from = nullptr, page = 0, slot = -1, later = -1;
        if (t < ng) { from = stands(lg_owner(freed, n, t), t); page = *from; }
        else if (t < nn) page = a.stack[top - 1 - t];
        int here = 0, pos = 0;
        bool ids = false;
        if (!n_slots) for (int i = t; i < n; i += NT) if (half_full(i)) ids |= outside(*place(i, olds[i] >> a.shift));      // (no slots here)
        if (n_slots && t < nt) {
            const int i = lg_owner(tok, n, t);
            pos = olds[i] + t - tok[i];
            const int block = pos >> a.shift, nb = blocks(olds[i]);
            if (block < nb) here = *place(i, block); else later = need[i] + block - nb;
        }
        if (ids || outside(page) || outside(here)) atomicOr(&bad_page, LG_PLAN_BAD_PAGE);
        taken[t] = page;
        __syncthreads();
        st = bad_page;
        if (!st) {
            if (from) { *from = -1; a.stack[top - 1 - t] = page; }
            if (t < nn) *goes(lg_owner(need, n, t), t) = page;
            if (n_slots && t < nt) slot = (later < 0 ? here : taken[later]) * P + (pos & (P - 1));
        }
        if (t < n_slots) a.slots[t] = slot;
    } else {
        // of many entries the sequences of NT first, between which the others' are: a step of a search or two each instead of nine (333 prompts 12.0 -> 9.8 us; of up to 4 NT entries it saves nothing)
        int gap = -1;
        auto sample = [&](const int32_t *sums, int total) {
            gap = -1;
            if (total <= 4 * NT) return;
            for (gap = 0; (total - 1) >> gap >= NT; ) ++gap;
            __syncthreads();
            taken[t] = t <= (total - 1) >> gap ? lg_owner(sums, n, t << gap) : n;
            if (t == 0) taken[NT] = n;
            __syncthreads();
        };
        auto owner = [&](const int32_t *sums, int e) { return gap < 0 ? lg_owner(sums, n, e) : lg_owner(sums, taken[(e >> gap) + 1], e, taken[e >> gap]); };
        if (!st) {
            bool ids = false;
            sample(freed, ng);
            for (int e = t; e < ng; e += NT) ids |= outside(*stands(owner(freed, e), e));
            for (int e = ng + t; e < nn; e += NT) ids |= outside(a.stack[top - 1 - e]);
            for (int i = t; i < n; i += NT) if (half_full(i)) ids |= outside(*place(i, olds[i] >> a.shift));
            if (ids) atomicOr(&bad_page, LG_PLAN_BAD_PAGE);
            __syncthreads();
            st = bad_page;
        }
        if (!st) {
            for (int e = t; e < ng; e += NT) { int32_t *const p = stands(owner(freed, e), e); a.stack[top - 1 - e] = *p; *p = -1; }
            __syncthreads();
            sample(need, nn);
            for (int e = t; e < nn; e += NT) *goes(owner(need, e), e) = a.stack[top - 1 - e];
            __syncthreads();
        }
        for (int s = t; s < n_slots; s += NT) {
            int slot = -1;
            if (!st && s < nt) {
                const int i = lg_owner(tok, n, s), pos = olds[i] + s - tok[i];
                slot = *place(i, pos >> a.shift) * P + (pos & (P - 1));
            }
            a.slots[s] = slot;
        }
    }
    for (int i = t; i <= n; i += NT) a.start[i] = st ? 0 : tok[i];
    if (t == 0) { *a.status = st; if (!st) *a.n_free = top - nn; }
}
// Slots of many tokens, behind the plan (start of what it refused is 0: no token).  Four in a row to a thread: one search each, then along the sequences.  37000 slots 4 us.
__global__ __launch_bounds__(256) void lg_k_plan_slots(PlanArgs a) {
    __shared__ int32_t tok[LG_PLAN_SEQS + 1];
    const int n = a.n_seq, P = 1 << a.shift;
    for (int i = threadIdx.x; i <= n; i += 256) tok[i] = a.start[i];
    __syncthreads();
    const int s0 = (int)(blockIdx.x * 256 + threadIdx.x) * 4, nt = tok[n];
    if (s0 >= a.n_slots) return;
    int out[4] = { -1, -1, -1, -1 };
    int i = s0 < nt ? lg_owner(tok, n, s0) : 0;
    #pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int s = s0 + k;
        if (s >= nt) continue;
        while (tok[i + 1] <= s) ++i;
        const int pos = a.len_old[i] + s - tok[i];
        out[k] = a.table[(size_t)i * a.max_blocks + (pos >> a.shift)] * P + (pos & (P - 1));
    }
    #pragma unroll
    for (int k = 0; k < 4; ++k) if (s0 + k < a.n_slots) a.slots[s0 + k] = out[k];
}

// ---- write -----------------------------------------------------------------------------------------------------------
struct PageGeo {
    uint16_t *k, *v;
    long long row_stride, page_stride;  // values
    int n_pages, shift;                 // page_size = 1 << shift
};
// New K and V rows, f32 -> binary16 (nearest even: the rounding that the cache's type asks for), into their slots.  Bound by memory: 6 bytes a value.  A thread takes 8
// values: two 16-byte loads and one 16-byte store.  20011 tokens of 2 x 2048 values 86 us, 5.5 TB/s; 64 tokens of 2 x 512 2.5 us.
__global__ __launch_bounds__(256) void lg_k_page_write(PageGeo g, const float *k, const float *v, long long stride, const int32_t *slots, int n_tok, int units) {
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int tok = (int)(id / (2 * units)), u = (int)(id % (2 * units));
    if (tok >= n_tok) return;
    const int slot = slots[tok], page = slot >> g.shift;
    if (slot < 0 || page >= g.n_pages) return;
    const bool second = u >= units;
    const int c = (second ? u - units : u) * 8;
    const float4 *src = (const float4 *)((second ? v : k) + (long long)tok * stride + c);
    const float4 x = src[0], y = src[1];
    union { _Float16 h[8]; uint4 q; } o;
    o.h[0] = (_Float16)x.x; o.h[1] = (_Float16)x.y; o.h[2] = (_Float16)x.z; o.h[3] = (_Float16)x.w;
    o.h[4] = (_Float16)y.x; o.h[5] = (_Float16)y.y; o.h[6] = (_Float16)y.z; o.h[7] = (_Float16)y.w;
    *(uint4 *)((second ? g.v : g.k) + page * g.page_stride + (slot & ((1 << g.shift) - 1)) * g.row_stride + c) = o.q;
}

// ---- attend ----------------------------------------------------------------------------------------------------------
// One new token per sequence: o[h] = sum_t softmax_t(scale q[h].k[t, h / G]) v[t, h / G] over the keys t of [max(0, len - window), len).
//
// A wavefront takes tiles of 32 keys (aligned to position 0, so a page holds whole half tiles of 16) of one key head, whose G <= 8 query heads share
// what it reads.  All products run on v_mfma_f32_16x16x32_f16.  Queries and probabilities are f32 and keep their precision: each is split into a
// binary16 value and the binary16 of what that leaves (22 bits together), which are rows 0..7 and 8..15 of the 16 that an instruction multiplies
// anyway, so that the second half costs nothing; the two results are added in f32.  Both are scaled by a power of two first (queries so that the largest
// of a head lies in [2^14, 2^15), probabilities by 2^14), away from binary16's subnormals.
//   scores, transposed: S^T = K Q^T.  A lane's 16 bytes of a key row are the operand as they lie in memory.  Lane l gets query row l % 16 and the keys
//   4 (l / 16) .. + 3 of either half tile.
//   values: O = P V needs 8 keys of one dimension per lane.  The order of keys inside a product is free, so it is the one in which the lane has
//   its scores already, and no probability crosses lanes; a lane loads 16 bytes (8 dimensions) of each of its 8 key rows and turns the 8 x 8
//   values in registers (v_perm_b32).
// K and V never pass through LDS.  Maximum and sum run in f32; the sum is of the unsplit probabilities.
// Bound by memory: a flop for every byte of K and V and query head of a group, where the matrix cores have hundreds.  What remains beside the bytes is the chain at either end
// (lengths, page ids, first keys; sums of the wavefronts: 3 to 6 us together).  24 sequences of up to 16384 keys, 8 key heads of 256: 503 us, 6.4 TB/s; one of 100003 keys:
// 134 us, 6.1 TB/s; 61 ragged ones of up to 8192, 2 key heads: 66 us, 5.2 TB/s (what the splits leave uneven); 64 windows of 512: 16 us, 3.3 TB/s (128 of 256 compute
// units, each at what it can draw); one of 100 keys: 3.9 us.
#define LG_PA_WAVES 4
#define LG_PA_TILE  32
#define LG_PA_LANES 64
#define LG_PA_SEQS  4096            // sequences of a call
#define LG_PA_CHUNK 2048            // keys of a split at most: their page ids lie in LDS
// A barrier for what went through LDS: loads from memory stay on their way, which the barrier of __syncthreads waits for as well
__device__ __forceinline__ void lg_barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
typedef _Float16 lg_h8 __attribute__((ext_vector_type(8)));
typedef float lg_f4 __attribute__((ext_vector_type(4)));

struct PageAttn {
    PageGeo g;
    const float *q; long long q_stride;
    const int32_t *table, *len;
    float *out; long long out_stride;
    float *pm, *pl, *pacc;              // [splits of all][H], [..][hd]: partials of sequences of more than one split
    float scale;
    int32_t *cut;                       // [n_seq + 1] splits before each sequence, for the joining launch; of more than LG_PA_LANES sequences from lg_k_page_cut, and then: tiles of a split; the splits' sequences
    int H, nkv, n_seq, max_blocks, max_len, window, slots, least;       // slots: workgroups that the chip holds at a time; least: tiles of a split, or all of a sequence's where there are no partials
};
// The keys a sequence sees: [lo, len)
__device__ __forceinline__ void lg_pa_range(const PageAttn &a, int seq, int &lo, int &len) {
    const long long room = (long long)a.max_blocks << a.g.shift;
    len = a.len[seq];
    if (len > a.max_len) len = a.max_len;
    if (len > room) len = (int)room;
    if (len < 0) len = 0;
    lo = a.window > 0 && len > a.window ? len - a.window : 0;
}
__device__ __forceinline__ int lg_pa_tiles(const PageAttn &a, int seq) {
    int lo, len;
    lg_pa_range(a, seq, lo, len);
    return (len + LG_PA_TILE - 1) / LG_PA_TILE - lo / LG_PA_TILE;
}
// How the call is cut, from the lengths: by every workgroup for up to LG_PA_LANES sequences, by lg_k_page_cut for more.  A compute unit draws a fixed share of what memory gives (it keeps about 32 KB
// of misses on their way), so the call takes as long as the unit with the most keys: splits of one size, chosen so that their number is what the
// chip holds at a time, not splits of a fixed size that the lengths fill unevenly.
// A sequence without keys has one split too: it writes the zeros.
struct PageCut { int tiles; int seq, index, first, n; };       // tiles of a split; of split number `at`: its sequence, its place there, the number of the sequence's first, how many it has
// `total` tiles of `some` sequences that have any: the smallest of a few sizes whose splits are at most a whole number of rounds of a.slots workgroups, as few as leave half of
// them to splits that are full.  Were every sequence's last split a full one, `some` more than total / size would be needed; ragged ones need half as many, and the size
// for that is tried first (61 sequences of 4..8192 keys, heads of 256: 74.3 -> 72.1 us).  count(t): the splits of size t
template <typename Count>
__device__ __forceinline__ uint32_t lg_pa_split_tiles(const PageAttn &a, uint32_t total, uint32_t some, Count count) {
    const uint32_t units = some * a.nkv, half = (uint32_t)a.slots / 2, rounds = units > half ? (units + half - 1) / half : 1, room = rounds * a.slots / a.nkv;
    auto size = [&](uint32_t spare) {
        const uint32_t full = room > spare ? room - spare : 1, tiles = (total + full - 1) / full;
        return tiles < (uint32_t)a.least ? a.least : tiles > LG_PA_CHUNK / LG_PA_TILE ? LG_PA_CHUNK / LG_PA_TILE : tiles;
    };
    const uint32_t most = size(some);
    if (some < 2 || most == (uint32_t)a.least) return most;
    #pragma unroll 1
    for (uint32_t eighths = 4; eighths < 8; ++eighths) {
        const uint32_t tiles = size((some * eighths + 7) / 8);
        if (tiles == most) break;
        if (count(tiles) <= room) return tiles;
    }
    return most;
}
__device__ __forceinline__ uint32_t lg_pa_splits(uint32_t of, uint32_t tiles) { const uint32_t x = (of + tiles - 1) / tiles; return x ? x : 1u; }
__device__ __forceinline__ PageCut lg_pa_cut(const PageAttn &a, int at) {
    if (!a.pm) return { a.least, at, 0, at, 1 };
    if (a.n_seq > LG_PA_LANES) {
        const int seq = a.cut[2 + a.n_seq + at];
        if (at >= a.cut[a.n_seq]) return { 0, -1, 0, 0, 0 };
        const int first = a.cut[seq];
        return { a.cut[1 + a.n_seq], seq, at - first, first, a.cut[seq + 1] - first };
    }
    // a lane for each, in every wavefront: no barrier
    const int i = threadIdx.x & 63;
    const uint32_t mine = i < a.n_seq ? lg_pa_tiles(a, i) : 0, some = (uint32_t)__popcll(__ballot(mine != 0));
    const uint32_t tiles = lg_pa_split_tiles(a, lg_wave_total(mine), some, [&](uint32_t t) { return lg_wave_total((mine + t - 1) / t); });
    const uint32_t n = i < a.n_seq ? lg_pa_splits(mine, tiles) : 0, run = lg_wave_run(n) - n;
    const lg_u64 it = __ballot((uint32_t)at - run < n);
    if (!it) return { (int)tiles, -1, 0, 0, 0 };
    const int lane = (int)__builtin_ctzll(it), first = (int)lg_lane(run, lane);
    return { (int)tiles, lane, at - first, first, (int)lg_lane(n, lane) };
}
// The cut of more sequences than a wavefront has lanes, worked out once: in every workgroup it takes several barriers and passes over the
// lengths.  400 sequences of all lengths up to 1024, heads of 128: 66.8 -> 48.0 us, with the joining launch's workgroups of one wavefront
#define LG_PC_WG    1024
__global__ __launch_bounds__(LG_PC_WG) void lg_k_page_cut(PageAttn a) {
    __shared__ uint32_t part[LG_PC_WG / 64];
    __shared__ int32_t before[LG_PA_SEQS + 1];
    constexpr int PER = LG_PA_SEQS / LG_PC_WG;
    const int per = (a.n_seq + LG_PC_WG - 1) / LG_PC_WG, i0 = threadIdx.x * per;
    uint32_t x[PER], mine = 0, some = 0, all;
    #pragma unroll
    for (int k = 0; k < PER; ++k) {
        x[k] = k < per && i0 + k < a.n_seq ? lg_pa_tiles(a, i0 + k) : 0;
        mine += x[k]; some += x[k] != 0;
    }
    const uint32_t total = lg_block_sum<LG_PC_WG>(mine, part);
    some = lg_block_sum<LG_PC_WG>(some, part);
    const uint32_t tiles = lg_pa_split_tiles(a, total, some, [&](uint32_t t) {
        uint32_t n = 0;
        #pragma unroll
        for (int k = 0; k < PER; ++k) n += (x[k] + t - 1) / t;
        return lg_block_sum<LG_PC_WG>(n, part);
    });
    uint32_t n = 0;
    #pragma unroll
    for (int k = 0; k < PER; ++k) n += k < per && i0 + k < a.n_seq ? lg_pa_splits(x[k], tiles) : 0;
    uint32_t run = lg_block_run<LG_PC_WG>(n, part, &all) - n;
    #pragma unroll
    for (int k = 0; k < PER; ++k)
        if (k < per && i0 + k < a.n_seq) { before[i0 + k] = (int32_t)run; a.cut[i0 + k] = (int32_t)run; run += lg_pa_splits(x[k], tiles); }
    if (threadIdx.x == 0) { before[a.n_seq] = (int32_t)all; a.cut[a.n_seq] = (int32_t)all; a.cut[a.n_seq + 1] = (int32_t)tiles; }
    __syncthreads();
    for (int s = threadIdx.x; s < (int)all; s += LG_PC_WG) a.cut[2 + a.n_seq + s] = lg_owner(before, a.n_seq, s);
}
// The pages of a tile's two halves, and where their rows lie: page 0's first value where there is no such page
struct PageTile { long long row[2]; bool ok[2]; };
struct PageIds { int id[2]; };
__device__ __forceinline__ PageIds lg_pa_ids(const PageAttn &a, const int32_t *table, int t0) {
    PageIds p;
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int b = (t0 + 16 * h) >> a.g.shift, id = table[b < a.max_blocks ? b : a.max_blocks - 1];
        p.id[h] = b < a.max_blocks ? id : -1;
    }
    return p;
}
__device__ __forceinline__ PageTile lg_pa_tile(const PageAttn &a, const PageIds &ids, int t0, int head) {
    PageTile p;
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        p.ok[h] = ids.id[h] >= 0 && ids.id[h] < a.g.n_pages;
        p.row[h] = (p.ok[h] ? ids.id[h] : 0) * a.g.page_stride + ((t0 + 16 * h) & ((1 << a.g.shift) - 1)) * a.g.row_stride + head;
    }
    return p;
}

// Two wavefronts on a SIMD at heads of up to 256: registers for both have to be asked for
constexpr int lg_pa_per_simd(int hd) { return hd == 512 ? 1 : hd == 256 ? 2 : hd == 128 ? 3 : 4; }
template <int HD>
__global__ __launch_bounds__(LG_PA_WAVES * 64, lg_pa_per_simd(HD)) void lg_k_page_attn(PageAttn a) {
    constexpr int KS = HD / 32;                     // score steps
    constexpr int DL = HD >= 128 ? 8 : HD / 16;     // dimensions of a value load
    constexpr int CH = HD / (16 * DL);              // value loads of a key row
    constexpr int NT = HD / 16;                     // output tiles
    constexpr int HALVES = HD > 256 ? 1 : 2, TILE = 16 * HALVES;       // keys of a step: rows of 512 leave registers for a half tile (a whole one spills: one key of 512, 15.4 -> 12.4 us)
    __shared__ float s_m[LG_PA_WAVES][8], s_l[LG_PA_WAVES][8];
    __shared__ __align__(16) union { lg_h8 q[KS][64]; float o[LG_PA_WAVES][8][HD]; } s;
    __shared__ int32_t s_ids[LG_PA_CHUNK / 16 + 1];
    const int kvh = blockIdx.x % a.nkv, G = a.H / a.nkv;
    const PageCut cut = lg_pa_cut(a, blockIdx.x / a.nkv);
    const int seq = __builtin_amdgcn_readfirstlane(cut.seq);
    if (seq < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    constexpr int STEP = LG_PA_WAVES * TILE;
    const int32_t *table = a.table + (long long)seq * a.max_blocks;
    // queries are asked for first: what is asked for later arrives later, and behind the keys they would hold the first scores up
    // A wavefront takes every fourth step's (all of them in every wavefront: one key, heads of 512 12.0 -> 9.4 us, of 256 7.1 -> 6.3)
    constexpr int QS = (KS + LG_PA_WAVES - 1) / LG_PA_WAVES;
    float4 qv[QS][2];
    const float *qrow = a.q + seq * a.q_stride + (long long)(kvh * G + ((c & 7) < G ? c & 7 : 0)) * HD + g * 8;
    #pragma unroll
    for (int i = 0; i < QS; ++i)
        #pragma unroll
        for (int j = 0; j < 2; ++j) qv[i][j] = *(const float4 *)(qrow + (KS < LG_PA_WAVES ? wave % KS : i * LG_PA_WAVES + wave) * 32 + j * 4);
    int lo, len;
    lg_pa_range(a, seq, lo, len);
    const int chunk = __builtin_amdgcn_readfirstlane(cut.tiles) * LG_PA_TILE, n_split = __builtin_amdgcn_readfirstlane(cut.n);
    const int first = (lo & ~(LG_PA_TILE - 1)) + __builtin_amdgcn_readfirstlane(cut.index) * chunk, end = len < first + chunk ? len : first + chunk;
    int t0 = first + wave * TILE;
    const PageIds ids = lg_pa_ids(a, table, t0);
    // the later tiles' ids through LDS: a load of them inside the loop would be waited for together with the keys that are on their way
    const int b0 = first >> a.g.shift;
    static_assert(LG_PA_CHUNK / 16 + 1 <= LG_PA_WAVES * 64, "an id for each thread");
    const bool has_id = (int)threadIdx.x <= ((end - 1) >> a.g.shift) - b0;
    const int my_id = has_id && b0 + (int)threadIdx.x < a.max_blocks ? table[b0 + threadIdx.x] : -1;
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
    PageTile now = lg_pa_tile(a, ids, t0, kvh * HD);
    auto load_keys = [&](const PageTile &p) {
        #pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            const uint16_t *kp = a.g.k + p.row[h] + c * a.g.row_stride + g * 8;
            #pragma unroll
            for (int i = 0; i < KS; ++i) kf[h][i] = *(const lg_h8 *)(kp + i * 32);
        }
    };
    // queries: operand B of the scores, column c = query head c % 8, high part for c < 8
    float qs;                                       // factor of the raw scores: base-2 exponents
    auto queries = [&]() {
        if (has_id) s_ids[threadIdx.x] = my_id;
        float top = 0;
        #pragma unroll
        for (int i = 0; i < QS; ++i)
            #pragma unroll
            for (int j = 0; j < 2; ++j) top = fmaxf(top, fmaxf(fmaxf(fabsf(qv[i][j].x), fabsf(qv[i][j].y)), fmaxf(fabsf(qv[i][j].z), fabsf(qv[i][j].w))));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (lane < 8) s_m[wave][lane] = top;
        lg_barrier_lds();
        #pragma unroll
        for (int v = 0; v < LG_PA_WAVES; ++v) top = fmaxf(top, s_m[v][c & 7]);
        int e = (int)(__float_as_uint(top) >> 23) - 127 - 14;       // top * 2^-e in [2^14, 2^15)
        if (e < -100) e = -100;                                     // (zero and tiny rows; 2^-e stays a float)
        const float up = __uint_as_float((unsigned)(127 - e) << 23);
        #pragma unroll
        for (int i = 0; i < QS; ++i) {
            const int step = i * LG_PA_WAVES + wave;
            if (step >= KS) continue;
            const float v[8] = { qv[i][0].x, qv[i][0].y, qv[i][0].z, qv[i][0].w, qv[i][1].x, qv[i][1].y, qv[i][1].z, qv[i][1].w };
            lg_h8 part;
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float z = v[j] * up;
                const _Float16 hi = (_Float16)z;
                part[j] = c < 8 ? hi : (_Float16)(z - (float)hi);
            }
            s.q[step][lane] = part;
        }
        qs = a.scale * 1.44269504088896341f * __uint_as_float((unsigned)(127 + e) << 23);
        lg_barrier_lds();
    };
    // A wavefront without a tile asks for no keys (84 short sequences of heads of 256: 12.0 -> 9.7 us).  The queries are prepared on either side of that branch: behind it
    // they would have to wait for everything in flight
    if (t0 < end) {
        __builtin_amdgcn_sched_barrier(0);
        load_keys(now);
        __builtin_amdgcn_sched_barrier(0);
        queries();
    } else {
        queries();
        asm volatile("");                           // (so that the two sides stay apart)
    }
    lg_f4 acc[NT];
    #pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = (lg_f4){ 0, 0, 0, 0 };
    float m = -INFINITY, l = 0;                     // of query row c; l of this lane's keys alone

    // One tile: its values are requested before its scores are made, the next tile's keys before its values are used
    auto work = [&](auto more) {                    // more: a tile follows (a branch around its loads would have them waited for with this tile's)
        constexpr bool MORE = decltype(more)::value;
        const PageTile here = now;
        if constexpr (MORE) now = tile_at(t0 + STEP);
        uint32_t w[CH][4 * HALVES][DL / 2];
        #pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            #pragma unroll
            for (int j = 0; j < 4 * HALVES; ++j) {
                const uint16_t *vp = a.g.v + here.row[j >> 2] + (4 * g + (j & 3)) * a.g.row_stride + ch * 128 + c * DL;
                if constexpr (DL == 8) { const uint4 u = *(const uint4 *)vp; w[ch][j][0] = u.x; w[ch][j][1] = u.y; w[ch][j][2] = u.z; w[ch][j][3] = u.w; }
                else { const uint2 u = *(const uint2 *)vp; w[ch][j][0] = u.x; w[ch][j][1] = u.y; }
            }
        __builtin_amdgcn_sched_barrier(0);
        lg_f4 sc[HALVES];
        #pragma unroll
        for (int h = 0; h < HALVES; ++h) sc[h] = (lg_f4){ 0, 0, 0, 0 };
        #pragma unroll
        for (int i = 0; i < KS; ++i) {
            const lg_h8 q = s.q[i][lane];
            #pragma unroll
            for (int h = 0; h < HALVES; ++h) sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[h][i], q, sc[h], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MORE) load_keys(now);
        __builtin_amdgcn_sched_barrier(0);
        // base-2 exponents; rows c and c + 8 hold the two parts of a query's score
        float x[HALVES][4], top = -INFINITY;
        #pragma unroll
        for (int h = 0; h < HALVES; ++h)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float both = sc[h][r] + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(sc[h][r]), 0x128, 0xF, 0xF, true));   // row_ror:8
                const int t = t0 + 16 * h + 4 * g + r;
                x[h][r] = here.ok[h] && t >= lo && t < end ? both * qs : -INFINITY;
                top = fmaxf(top, x[h][r]);
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        if (__any(top > m)) {
            const float mn = fmaxf(m, top);
            const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mn);   // (both -inf: nothing seen yet)
            l *= f; m = mn;
            float fr[4];
            #pragma unroll
            for (int r = 0; r < 4; ++r) fr[r] = __shfl(f, (4 * g + r) & 7);
            #pragma unroll
            for (int i = 0; i < NT; ++i)
                #pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][r] *= fr[r];
        }
        typedef _Float16 part __attribute__((ext_vector_type(4 * HALVES)));
        part pf;
        #pragma unroll
        for (int h = 0; h < HALVES; ++h)
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = x[h][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x[h][r] - m + 14.0f);
                l += p;
                const _Float16 hi = (_Float16)p;
                pf[4 * h + r] = c < 8 ? hi : (_Float16)(p - (float)hi);
            }
        // a masked key's values may be anything (0 * inf is not 0): zeros in their place
        if (!(t0 >= lo && t0 + TILE <= end && here.ok[0] && here.ok[HALVES - 1])) {
            #pragma unroll
            for (int j = 0; j < 4 * HALVES; ++j) {
                const int t = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
                if (!(here.ok[j >> 2] && t >= lo && t < end)) {
                    #pragma unroll
                    for (int ch = 0; ch < CH; ++ch)
                        #pragma unroll
                        for (int i = 0; i < DL / 2; ++i) w[ch][j][i] = 0;
                }
            }
        }
        #pragma unroll
        for (int ch = 0; ch < CH; ++ch)
            #pragma unroll
            for (int i = 0; i < DL; ++i) {
                union { uint32_t u[2 * HALVES]; part h; } b;
                #pragma unroll
                for (int k2 = 0; k2 < 2 * HALVES; ++k2) b.u[k2] = __builtin_amdgcn_perm(w[ch][2 * k2 + 1][i >> 1], w[ch][2 * k2][i >> 1], i & 1 ? 0x07060302 : 0x05040100);
                lg_f4 &to = acc[ch * DL + i];
                if constexpr (HALVES == 2) to = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, b.h, to, 0, 0, 0);
                else to = __builtin_amdgcn_mfma_f32_16x16x16f16(pf, b.h, to, 0, 0, 0);
            }
    };
    for (; t0 + STEP < end; t0 += STEP) work(std::true_type{});
    if (t0 < end) work(std::false_type{});
    // the wavefronts' parts: sums over the quarters of a tile, then the four together
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 8) { s_m[wave][lane] = m; s_l[wave][lane] = l; }
    __syncthreads();                                // (the queries' last reader)
    // the two parts of a probability: rows 4 g + r of the lower and the upper half of the lanes.  One exchange joins two registers' halves
    #pragma unroll
    for (int ch = 0; ch < CH; ++ch)
        #pragma unroll
        for (int r = 0; r < 4; r += 2) {
            float o[DL];
            #pragma unroll
            for (int i = 0; i < DL; ++i) {
                const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[ch * DL + i][r]), __float_as_uint(acc[ch * DL + i][r + 1]), false, false);
                o[i] = __uint_as_float(u[0]) + __uint_as_float(u[1]);
            }
            #pragma unroll
            for (int i = 0; i < DL; i += 4) *(float4 *)&s.o[wave][4 * (g & 1) + r + (g >> 1)][ch * 128 + c * DL + i] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
    __syncthreads();
    // (behind the loads: lengths and page ids come through the scalar cache as long as nothing has been stored)
    if (a.pm && a.n_seq <= LG_PA_LANES && kvh == 0 && cut.index == 0 && threadIdx.x == 0) {
        a.cut[seq] = cut.first;
        if (seq == a.n_seq - 1) a.cut[a.n_seq] = cut.first + cut.n;
    }
    // all eight heads' sums, so that nothing waits for a branch; those there are are stored (rows may start anywhere: four values at a time where they are aligned for that)
    constexpr int OUT = 8 * HD / 4, ROUNDS = (OUT + LG_PA_WAVES * 64 - 1) / (LG_PA_WAVES * 64);
    const bool wide = (((uintptr_t)a.out | (uintptr_t)a.out_stride * 4) & 15) == 0;
    #pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const int id = threadIdx.x + k * (LG_PA_WAVES * 64), h = id / (HD / 4) & 7, d = id % (HD / 4) * 4;
        float M = -INFINITY, L = 0;
        float4 o = make_float4(0, 0, 0, 0);
        #pragma unroll
        for (int v = 0; v < LG_PA_WAVES; ++v) M = fmaxf(M, s_m[v][h]);
        #pragma unroll
        for (int v = 0; v < LG_PA_WAVES; ++v) {
            const float lv = s_l[v][h], f = lv == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s_m[v][h] - M);       // (0: no key; a score of NaN leaves its mark in the sum)
            const float4 x = *(const float4 *)&s.o[v][h][d];
            L += f * lv;
            o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
        }
        if (id >= G * (HD / 4)) continue;
        const int head = kvh * G + h;
        if (n_split == 1) {
            float *const p = a.out + seq * a.out_stride + (long long)head * HD + d;
            const float4 x = L == 0.0f ? make_float4(0, 0, 0, 0) : make_float4(o.x / L, o.y / L, o.z / L, o.w / L);
            if (wide) *(float4 *)p = x;
            else { p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w; }
        } else {
            const long long at = (long long)(blockIdx.x / a.nkv) * a.H + head;
            *(float4 *)(a.pacc + at * HD + d) = o;
            if (d == 0) { a.pm[at] = M; a.pl[at] = L; }
        }
    }
}

// The splits of a sequence, joined: a workgroup per (sequence, head).  A split's factor is computed once, by one thread; then the wavefronts take splits in
// turn, a lane HD / 64 dimensions, and their sums are added in order.  A chain of maxima, factors and sums: 5 us for 8 or 16 heads of 256, 65 splits of one sequence or 317 of 61; 8 to 9 where one sequence has 250 to 510 of them.
template <int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void lg_k_page_merge(PageAttn a) {
    constexpr int NT = WAVES * 64, D = HD / 64;
    __shared__ float s_f[NT], s_w[WAVES], s_o[WAVES][HD];
    const int head = blockIdx.x, seq = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int from = a.cut[seq], n = a.cut[seq + 1] - from;
    if (n < 2) return;                                       // (its one split has written the output)
    // what the first NT splits need is asked for at once: a wavefront's first eight sums with the maxima
    typedef float vec __attribute__((ext_vector_type(D)));
    constexpr int FIRST = HD == 512 ? 4 : 8;
    auto place = [&](int k) { return (long long)(from + k) * a.H + head; };
    auto sums = [&](int k) { return *(const vec *)(a.pacc + place(k) * HD + lane * D); };
    vec ahead[FIRST];
    const float m0 = t < n ? a.pm[place(t)] : -INFINITY, l0 = t < n ? a.pl[place(t)] : 0.0f;
    #pragma unroll
    for (int j = 0; j < FIRST; ++j) { const int k = wave + j * WAVES; ahead[j] = sums(k < n ? k : n - 1); }
    float M = m0;
    for (int i = t + NT; i < n; i += NT) M = fmaxf(M, a.pm[place(i)]);
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    if (lane == 0) s_w[wave] = M;
    __syncthreads();
    #pragma unroll
    for (int v = 0; v < WAVES; ++v) M = fmaxf(M, s_w[v]);
    float L = 0;
    vec o = 0;
    for (int base = 0; base < n; base += NT) {
        const int i = base + t;
        const float mi = base ? i < n ? a.pm[place(i)] : 0.0f : m0, ls = base ? i < n ? a.pl[place(i)] : 0.0f : l0;
        const float f = ls == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mi - M);                 // (0: no key, its pages are left out)
        L += ls == 0.0f ? 0.0f : f * ls;
        __syncthreads();
        s_f[t] = f;
        __syncthreads();
        const int m = n - base < NT ? n - base : NT;
        int k = wave;
        if (!base)
            #pragma unroll
            for (int j = 0; j < FIRST; ++j, k += WAVES) if (k < m) o += s_f[k] * ahead[j];
        #pragma unroll 4
        for (; k < m; k += WAVES) o += s_f[k] * sums(base + k);
    }
    for (int x = 1; x < 64; x <<= 1) L += __shfl_xor(L, x);
    __syncthreads();
    if (lane == 0) s_w[wave] = L;
    #pragma unroll
    for (int d = 0; d < D; ++d) s_o[wave][lane * D + d] = o[d];
    __syncthreads();
    L = 0;
    #pragma unroll
    for (int v = 0; v < WAVES; ++v) L += s_w[v];
    for (int d = t; d < HD; d += NT) {
        float x = 0;
        #pragma unroll
        for (int v = 0; v < WAVES; ++v) x += s_o[v][d];
        a.out[seq * a.out_stride + (long long)head * HD + d] = L == 0.0f ? 0.0f : x / L;
    }
}
