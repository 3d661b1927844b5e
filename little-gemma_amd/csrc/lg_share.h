// lg_share.h — pages of a cache that sequences share: forks and ends of them, and rows moved and copied in every layer.
#pragma once

#include "lg_pages.h"

// ---- fork ------------------------------------------------------------------------------------------------------------
enum { LG_FORK_BAD_LEN = 1, LG_FORK_NO_PAGES = 2, LG_FORK_BAD_SOURCE = 4, LG_FORK_BAD_STACK = 8, LG_FORK_BAD_PAGE = 16, LG_FORK_BAD_SHARES = 32 };   // LG_HIP_FORK_* of lg_hip.h

struct ForkPage { int32_t holders, first, parts, keeper; };      // of a page that the call touches: rows that hold it afterwards, its first release, rows that end in it, the one of them that keeps it
struct ForkArgs {
    const int32_t *src, *len_old, *len_new;     // [n_seq]
    int32_t *table;                             // [n_seq][max_blocks]
    int32_t *shares, *stack, *n_free;           // [n_pages], [n_pages], height
    int32_t *from, *to, *rows;                  // [n_seq]
    int32_t *status;
    ForkPage *page;                             // [n_pages] working memory: what is used is set first
    int32_t *stage;                             // [n_seq * max_blocks] the pages that come to a row
    int n_seq, shift, n_pages, max_blocks;
};

// Row i afterwards holds the first len_new[i] positions of what row src[i] held.  Only rows that change count: a row that takes another's pages releases all of its own and takes nb(len_new) of
// that one's, any other releases those behind nb(len_new).  A page's holders afterwards are those before and what comes and goes, in whole numbers, so the order of the additions does not matter; pages with none go on the
// stack, each at its first release (sequence by sequence, block by block), the first one topmost.  Of the rows that end inside a page one may keep it if no row holds it whole: the first that had it, or
// else the first; each of the others takes a page off the stack, in order, and is told what to copy.
// All or nothing: everything is read and counted in working memory, then everything is written.
// One workgroup, of NT threads: a few words for every page that moves, its time a chain of round trips to memory (lengths, ids, shares; counts; places; stores).  A thread keeps its first release, arrival and
// row in registers, so that a call of up to NT of each asks for them once: eight forks of 16 pages 9.7 -> 7.1 us.  61 conversations with three forks each 11.8 us; 63 forks of
// 250 pages of one page list 70, eight of 1563 pages 80: atomics for each page of each fork, on the same pages one after another, from one workgroup.
template <int NT, int SEQS>
__global__ __launch_bounds__(NT) void lg_k_page_fork(ForkArgs a) {
    __shared__ int32_t gone[SEQS + 1], come[SEQS + 1], fresh[SEQS];      // releases and arrivals before each row; which of the new pages it takes, -1 none
    __shared__ int32_t s_src[SEQS], s_old[SEQS], s_new[SEQS];
    __shared__ lg_u64 part[3 * NT / 64];
    __shared__ int32_t bad, wrong_page;
    const int t = threadIdx.x, P = 1 << a.shift, n = a.n_seq;
    const long long most = (long long)a.max_blocks << a.shift;
    const int per = (n + NT - 1) / NT, i0 = t * per < n ? t * per : n, i1 = i0 + per < n ? i0 + per : n;
    const int nf = *a.n_free;
    if (t == 0) { bad = nf < 0 || nf > a.n_pages ? LG_FORK_BAD_STACK : 0; wrong_page = 0; }
    for (int i = t; i < n; i += NT) { s_src[i] = a.src[i]; s_old[i] = a.len_old[i]; s_new[i] = a.len_new[i]; }
    __syncthreads();
    auto blocks = [&](int len) { return (int)(((long long)len + P - 1) >> a.shift); };
    auto place = [&](int i, int block) { return a.table + (size_t)i * a.max_blocks + block; };
    auto outside = [&](int id) { return id < 0 || id >= a.n_pages; };
    auto now = [&](const int32_t &x) { return __hip_atomic_load(&x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    lg_u64 run[3] = { 0, 0, 0 }, all[3];
    int st = 0;
    for (int i = i0; i < i1; ++i) {
        const int s = s_src[i], lo = s_old[i], ln = s_new[i];
        if (s < -1 || s >= n) st |= LG_FORK_BAD_SOURCE;
        else if (ln > (s >= 0 ? s_old[s] : 0)) st |= LG_FORK_BAD_LEN;
        if (lo < 0 || lo > most || ln < 0) st |= LG_FORK_BAD_LEN;
        if (st) break;
        gone[i] = (int)run[0]; come[i] = (int)run[1];
        run[0] += s != i ? blocks(lo) : blocks(lo) - blocks(ln);
        run[1] += s != i ? blocks(ln) : 0;
    }
    if (st) atomicOr(&bad, st);
    lg_block_run3<NT>(run, all, part);                        // (run: exclusive now; its barriers also show `bad`)
    st = bad;
    const int n_gone = st ? 0 : (int)all[0], n_come = st ? 0 : (int)all[1];
    if (!st) for (int i = i0; i < i1; ++i) { gone[i] += (int)run[0]; come[i] += (int)run[1]; }
    if (t == 0) { gone[n] = n_gone; come[n] = n_come; }
    __syncthreads();
    auto leaves = [&](int i, int e) { const int b = e - gone[i]; return s_src[i] != i ? b : blocks(s_new[i]) + b; };            // the block of release e
    auto ends = [&](int i) { return s_src[i] >= 0 && (s_new[i] & (P - 1)); };
    auto ends_in = [&](int i) { return place(s_src[i], s_new[i] >> a.shift); };
    auto key = [&](int i) { return (s_src[i] != i ? LG_PLAN_SEQS : 0) + i; };
    // the thread's first of each
    const bool has_g = t < n_gone, has_c = t < n_come, has_r = !st && i0 < i1 && ends(i0);
    const int gi = has_g ? lg_owner(gone, n, t) : 0, ci = has_c ? lg_owner(come, n, t) : 0;
    const int g_id = has_g ? *place(gi, leaves(gi, t)) : -1, c_id = has_c ? *place(s_src[ci], t - come[ci]) : -1, r_id = has_r ? *ends_in(i0) : -1;
    auto gone_of = [&](int e) { return e == t ? gi : lg_owner(gone, n, e); };
    auto come_of = [&](int e) { return e == t ? ci : lg_owner(come, n, e); };
    auto gone_id = [&](int e, int i) { return e == t ? g_id : *place(i, leaves(i, e)); };
    auto come_id = [&](int e) { return e == t ? c_id : a.stage[e]; };
    auto end_id = [&](int i) { return i == i0 ? r_id : ends(i) ? *ends_in(i) : -1; };
    // every page that the call touches: its holders before
    auto touch = [&](int id, int shares) {
        if (outside(id)) atomicOr(&wrong_page, LG_FORK_BAD_PAGE);
        else if (shares < 0 || shares >= LG_PLAN_SEQS) atomicOr(&wrong_page, LG_FORK_BAD_SHARES);
        else a.page[id] = ForkPage{ shares + 1, INT32_MAX, 0, INT32_MAX };
    };
    auto shares_of = [&](int id) { return outside(id) ? 0 : a.shares[id]; };
    if (!st) {
        const int sg = shares_of(g_id), sc = shares_of(c_id), sr = shares_of(r_id);
        if (has_g) touch(g_id, sg);
        if (has_c) touch(c_id, sc);
        if (has_r) touch(r_id, sr);
        for (int e = t + NT; e < n_gone; e += NT) { const int i = lg_owner(gone, n, e), id = *place(i, leaves(i, e)); touch(id, shares_of(id)); }
        for (int e = t + NT; e < n_come; e += NT) { const int i = lg_owner(come, n, e), id = *place(s_src[i], e - come[i]); a.stage[e] = id; touch(id, shares_of(id)); }
        for (int i = i0 + 1; i < i1; ++i) if (ends(i)) { const int id = *ends_in(i); touch(id, shares_of(id)); }
        __syncthreads();
        st = wrong_page;
    }
    int F = 0, N = 0, top = nf;
    if (!st) {
        for (int e = t; e < n_gone; e += NT) {
            const int id = gone_id(e, gone_of(e));
            atomicAdd(&a.page[id].holders, -1);
            atomicMin(&a.page[id].first, e);
        }
        for (int e = t; e < n_come; e += NT) atomicAdd(&a.page[come_id(e)].holders, 1);
        for (int i = i0; i < i1; ++i) {
            const int id = end_id(i);
            if (id >= 0) { atomicAdd(&a.page[id].parts, 1); atomicMin(&a.page[id].keeper, key(i)); }
        }
        __syncthreads();
        // releases in a row to a thread, as their places on the stack follow each other
        const int each = (n_gone + NT - 1) / NT, e0 = t * each < n_gone ? t * each : n_gone, e1 = e0 + each < n_gone ? e0 + each : n_gone;
        auto releases = [&](auto &&f) {
            for (int e = e0, i = e0 < e1 ? gone_of(e0) : 0; e < e1; ++e) {
                while (gone[i + 1] <= e) ++i;
                const int id = gone_id(e, i), h = now(a.page[id].holders), first = now(a.page[id].first);
                if (h < 0) atomicOr(&wrong_page, LG_FORK_BAD_SHARES);
                if (h == 0 && first == e) f(id);
            }
        };
        run[0] = run[1] = run[2] = 0;
        releases([&](int) { ++run[0]; });
        for (int i = i0; i < i1; ++i) {
            const int id = end_id(i);
            bool copies = false;
            if (id >= 0) {
                const int h = now(a.page[id].holders), p = now(a.page[id].parts), k = now(a.page[id].keeper);
                if (p > h) atomicOr(&wrong_page, LG_FORK_BAD_SHARES);
                copies = p != h || k != key(i);
            }
            fresh[i] = copies ? (int)run[1] : -1;
            run[1] += copies;
        }
        lg_block_run3<NT>(run, all, part);
        F = (int)all[0]; N = (int)all[1]; top = nf + F;
        for (int i = i0; i < i1; ++i) if (fresh[i] >= 0) fresh[i] += (int)run[1];
        if (t == 0) {
            if (top > a.n_pages) atomicOr(&wrong_page, LG_FORK_BAD_STACK);
            else if (N > top) atomicOr(&wrong_page, LG_FORK_NO_PAGES);
        }
        if (top <= a.n_pages && N <= top) for (int k = F + t; k < N; k += NT) if (outside(a.stack[top - 1 - k])) atomicOr(&wrong_page, LG_FORK_BAD_PAGE);
        __syncthreads();
        st = wrong_page;
        if (!st) {
            // counts and the stack first, while the table is as it was
            auto count = [&](int id) {
                const int h = now(a.page[id].holders), p = now(a.page[id].parts), left = h - (p && p == h ? p - 1 : p);
                a.shares[id] = left > 0 ? left - 1 : 0;
            };
            int at = top - 1 - (int)run[0];
            releases([&](int id) { a.stack[at--] = id; });
            for (int e = t; e < n_gone; e += NT) count(gone_id(e, gone_of(e)));
            for (int e = t; e < n_come; e += NT) count(come_id(e));
            for (int i = i0; i < i1; ++i) {
                const int id = end_id(i);
                if (id >= 0) count(id);
                a.from[i] = fresh[i] >= 0 ? id : -1;
                a.rows[i] = fresh[i] >= 0 ? s_new[i] & (P - 1) : 0;
            }
            __syncthreads();
            for (int e = t; e < n_gone; e += NT) { const int i = gone_of(e), b = leaves(i, e); if (b >= blocks(s_new[i])) *place(i, b) = -1; }
            for (int e = t; e < n_come; e += NT) {
                const int i = come_of(e), b = e - come[i];
                if (!(fresh[i] >= 0 && b == s_new[i] >> a.shift)) *place(i, b) = come_id(e);
            }
            for (int i = i0; i < i1; ++i) {
                const int id = fresh[i] >= 0 ? now(a.stack[top - 1 - fresh[i]]) : -1;
                a.to[i] = id;
                if (id >= 0) { *place(i, s_new[i] >> a.shift) = id; a.shares[id] = 0; }
            }
        }
    }
    if (st) for (int i = i0; i < i1; ++i) { a.from[i] = a.to[i] = -1; a.rows[i] = 0; }
    if (t == 0) { *a.status = st; if (!st) *a.n_free = top - N; }
}

// ---- rows and pages in every layer -----------------------------------------------------------------------------------
#define LG_LAYERS 64                // of a launch: they travel as its arguments
struct PageLayer { uint16_t *k, *v; long long row_stride, page_stride; int units; };          // units: 8 values, 16 bytes
struct PageLayers { PageLayer l[LG_LAYERS]; };

// The rows of an accepted path to the places behind the committed ones.  Rows only move down and in order (path[k] > path[k - 1]), so a thread that takes 16 bytes of them all, up to eight
// at a time, has read every row before it is written over.  Bound by memory: 2 bytes read and 2 written a value; where the rows lie is a chain of lengths, path and pages ahead of that, which is why
// a workgroup takes keys and values of a layer together, two places of 16 bytes a thread.  64 sequences of 48 layers of 8 heads of 256, 176 MB read and written: 28 to 30 us where caches hold a part of it (5.8 TB/s),
// 44 where they do not (4.0); one sequence of 42 layers 3.6.
typedef uint32_t lg_u4 __attribute__((ext_vector_type(4)));          // (arrays of HIP's own uint4 end up in scratch memory)
#define LG_MOVE_AT_ONCE 8
#define LG_MOVE_PLACES  512         // of a workgroup
__global__ __launch_bounds__(256) void lg_k_page_compact(PageLayers ls, const int32_t *table, const int32_t *len, const int32_t *start, const int32_t *path, const int32_t *count, int max_tree,
                                                        int max_blocks, int shift, int n_pages) {
    __shared__ long long s_src[64], s_dst[64];
    __shared__ int s_n;
    const int seq = blockIdx.z, lane = threadIdx.x;
    const PageLayer &L = ls.l[blockIdx.y];
    if (lane < 64) {
        const int total = len[seq], kept = count[seq];
        const long long n = (long long)start[seq + 1] - start[seq];
        const int mine = lane < max_tree ? path[(long long)seq * max_tree + lane] : -1;
        const bool fits = n >= 1 && n <= max_tree && total >= n && total <= (long long)max_blocks << shift;
        const int before = __shfl(mine, lane ? lane - 1 : 0);
        const bool ok = fits && lane < kept && mine >= 0 && mine < n && (lane == 0 || mine > before);
        const lg_u64 not_ok = ~__ballot(ok);
        const int last = not_ok ? (int)__builtin_ctzll(not_ok) : 64;   // rows from here on stay where they are
        const int P = 1 << shift;
        bool moves = lane < last && mine != lane;
        long long src = 0, dst = 0;
        if (moves) {
            const int32_t *row = table + (long long)seq * max_blocks;
            const int base = total - (int)n, sp = base + mine, dp = base + lane, a = row[sp >> shift], b = row[dp >> shift];
            moves = a >= 0 && a < n_pages && b >= 0 && b < n_pages;
            src = a * L.page_stride + (sp & (P - 1)) * L.row_stride;
            dst = b * L.page_stride + (dp & (P - 1)) * L.row_stride;
        }
        const lg_u64 all = __ballot(moves);
        if (moves) { const int k = __popcll(all & ((1ull << lane) - 1)); s_src[k] = src; s_dst[k] = dst; }
        if (lane == 0) s_n = __popcll(all);
    }
    __syncthreads();
    const int n = s_n, u0 = (int)(blockIdx.x * LG_MOVE_PLACES + threadIdx.x), u1 = u0 + LG_MOVE_PLACES / 2;
    if (u0 >= 2 * L.units) return;
    const bool both = u1 < 2 * L.units;
    auto place = [&](int u) { return (u < L.units ? L.k : L.v) + (u < L.units ? u : u - L.units) * 8; };
    uint16_t *const p0 = place(u0), *const p1 = place(both ? u1 : u0);
    auto move = [&](auto most, int k0) {            // (behind the last one the last again: no branch between loads)
        constexpr int N = decltype(most)::value;
        lg_u4 x[N], y[N];
        #pragma unroll
        for (int k = 0; k < N; ++k) {
            const long long at = s_src[k0 + k < n ? k0 + k : n - 1];
            x[k] = *(const lg_u4 *)(p0 + at);
            y[k] = *(const lg_u4 *)(p1 + at);
        }
        #pragma unroll
        for (int k = 0; k < N; ++k)
            if (k0 + k < n) {
                const long long at = s_dst[k0 + k];
                *(lg_u4 *)(p0 + at) = x[k];
                if (both) *(lg_u4 *)(p1 + at) = y[k];
            }
    };
    for (int k0 = 0; k0 < n; k0 += LG_MOVE_AT_ONCE) {
        if (n - k0 > 4) move(std::integral_constant<int, LG_MOVE_AT_ONCE>{}, k0);
        else if (n - k0 > 2) move(std::integral_constant<int, 4>{}, k0);
        else move(std::integral_constant<int, 2>{}, k0);
    }
}
// The first rows[i] rows of page from[i] to page to[i]: a workgroup takes every `parts`-th 4096 bytes of K or V of one pair in one layer.  Bound by memory: 1.81 GB read and written 372 us, 4.9 TB/s, as much as any copy; nine pages of 42 layers, 55 MB, 8 to 9 us.
__global__ __launch_bounds__(256) void lg_k_page_copy(PageLayers ls, const int32_t *from, const int32_t *to, const int32_t *rows, int shift, int n_pages, int parts) {
    const int i = blockIdx.z, a = from[i], b = to[i], n = rows[i];
    if (a < 0 || a >= n_pages || b < 0 || b >= n_pages || a == b || n < 1) return;
    const PageLayer &L = ls.l[blockIdx.y];
    const bool second = (int)blockIdx.x >= parts;
    const int first = second ? blockIdx.x - parts : blockIdx.x, P = 1 << shift, units = (n < P ? n : P) * L.units;
    const uint16_t *const src = (second ? L.v : L.k) + a * L.page_stride;
    uint16_t *const dst = (second ? L.v : L.k) + b * L.page_stride;
    const int step = parts * 256, of = L.units;
    const bool dense = L.row_stride == of * 8;
    auto where = [&](int u) { const int r = dense ? 0 : u / of; return r * L.row_stride + (long long)(u - r * of) * 8; };
    int u = first * 256 + threadIdx.x;
    for (; u + 3 * step < units; u += 4 * step) {
        const long long p0 = where(u), p1 = where(u + step), p2 = where(u + 2 * step), p3 = where(u + 3 * step);
        const uint4 x0 = *(const uint4 *)(src + p0), x1 = *(const uint4 *)(src + p1), x2 = *(const uint4 *)(src + p2), x3 = *(const uint4 *)(src + p3);
        *(uint4 *)(dst + p0) = x0; *(uint4 *)(dst + p1) = x1; *(uint4 *)(dst + p2) = x2; *(uint4 *)(dst + p3) = x3;
    }
    for (; u < units; u += step) *(uint4 *)(dst + where(u)) = *(const uint4 *)(src + where(u));
}
