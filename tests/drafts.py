"""Plain forms of the operators around trees of drafted tokens, shared pages and rules for logits, in 64 bits or whole numbers, and calls of the C ABI with host arrays."""
import ctypes as C
import math

import numpy as np

from serving import pages_of


# ---- trees --------------------------------------------------------------------------------------------------------
def random_parents(rng, n, kind="any"):
    """A tree's parents: a chain, all on row 0, or anything earlier."""
    if kind == "chain":
        return np.arange(n) - 1
    if kind == "star":
        return np.where(np.arange(n) > 0, 0, -1)
    return np.array([-1] + [int(rng.integers(0, j)) for j in range(1, n)][:max(0, n - 1)])[:n]


def starts_of(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)


def ways(parent):
    """Every row's way: itself and the rows above it."""
    out = []
    for j in range(len(parent)):
        out.append([j] + (out[parent[j]] if j else []))
    return out


def bits(rows):
    return np.uint64(sum(1 << int(r) for r in rows))


def tree_plan_ref(start, parent, lens):
    mask, pos, seq = np.zeros(len(parent), np.uint64), np.zeros(len(parent), np.int64), np.zeros(len(parent), np.int64)
    for i, (a, b) in enumerate(zip(start[:-1], start[1:])):
        for j, way in enumerate(ways(parent[a:b])):
            mask[a + j], pos[a + j], seq[a + j] = bits(way), lens[i] - (b - a) + len(way) - 1, i
    return mask, pos, seq


def accept_ref(start, parent, token, after, lens, most):
    path, count, ends, last = np.full((len(lens), most), -1), [], [], []
    for i, (a, b) in enumerate(zip(start[:-1], start[1:])):
        way = [0] if b > a else []
        while way:
            fits = [j for j in range(way[-1] + 1, b - a) if parent[a + j] == way[-1] and token[a + j] == after[a + way[-1]] and after[a + way[-1]] >= 0]
            if not fits:
                break
            way.append(fits[0])
        path[i, :len(way)] = way
        count.append(len(way)), ends.append(lens[i] - (b - a) + len(way)), last.append(after[a + way[-1]] if way else -1)
    return path, np.array(count), np.array(ends), np.array(last)


def tree_attend_ref(q, k, v, table, lens, start, mask, pos, page, n_pages, n_head_kv, window, scale, max_len):
    """q [rows][H][hd]; k, v [n_pages][page][kv][hd] binary16.  (out, bound): the result, and how far a kernel of the documented roundings may be from it."""
    rows, H, hd = q.shape
    G = H // n_head_kv
    out, bound = np.zeros((rows, H, hd)), np.zeros((rows, H, 1))
    for i, (a, b) in enumerate(zip(start[:-1], start[1:])):
        n, L = int(b - a), int(lens[i])
        if n <= 0 or L < n or L > max_len or L > table.shape[1] * page:
            continue
        done = L - n
        for j in range(n):
            if pos[a + j] < done:
                continue
            least = pos[a + j] - window + 1 if window else -1
            sees = np.arange(max(0, least), done)
            tree = [x for x in range(n) if int(mask[a + j]) >> x & 1 and (not window or pos[a + x] >= least)]
            sees = np.concatenate([sees, done + np.array(tree, np.int64)]).astype(np.int64)
            sees = sees[(table[i, sees // page] >= 0) & (table[i, sees // page] < n_pages)]
            if not sees.size:
                continue
            at = (table[i, sees // page], sees % page)
            kk, vv = k[at].astype(np.float64), v[at].astype(np.float64)
            for h in range(H):
                qq = q[a + j, h].astype(np.float64)
                x = scale * (kk[:, h // G] @ qq)
                e = np.exp(x - x.max())
                out[a + j, h] = e @ vv[:, h // G] / e.sum()
                size = abs(scale) * np.max(np.abs(kk[:, h // G]) @ np.abs(qq))
                bound[a + j, h] = tolerance(size, hd, sees.size) * np.max(np.abs(vv[:, h // G]))
    return out, bound


def tolerance(size, hd, keys):
    """Relative to the largest value.  A score: its query in 22 bits (2^-21 with both truncations), 2 hd products (two for each part of a query's value) added in f32 in any order, and
    the factor's three roundings and the product with it, all relative to `size`, the sum of the products' magnitudes.  Its exponential moves by as much, and by 2^-21 for the instruction and
    the argument's own rounding, 2^-21 for its two binary16 parts; numerator and denominator add 2 `keys` terms in f32 (2^-24 each, either side), and 16 joins and the division."""
    score = size * (2.0 ** -21 + (2 * hd + 6) * 2.0 ** -24)
    return 2 * (score + 2.0 ** -20) + 2 * (2 * keys + 16) * 2.0 ** -24


# ---- pages --------------------------------------------------------------------------------------------------------
def compact_ref(pools, page, n_pages, table, lens, start, path, count):
    """pools [layers][2][n_pages][page][width]; the rows of every path, one after another."""
    out = pools.copy()
    for i, (a, b) in enumerate(zip(start[:-1], start[1:])):
        n, L = int(b - a), int(lens[i])
        if n < 1 or n > path.shape[1] or L < n or L > table.shape[1] * page:
            continue
        before = -1
        for k in range(min(int(count[i]), path.shape[1])):
            if not before < path[i, k] < n:
                break
            before = int(path[i, k])
            src, dst = L - n + before, L - n + k
            s, d = int(table[i, src // page]), int(table[i, dst // page])
            if before != k and 0 <= s < n_pages and 0 <= d < n_pages:
                out[:, :, d, dst % page] = pools[:, :, s, src % page]
    return out


def fork_ref(page, src, old, new, table, shares, stack, n_free):
    """(from, to, rows, status, table, shares, stack, height), row by row."""
    n, n_pages, most = len(src), stack.size, table.shape[1] * page
    status = 0
    for i in range(n):
        named = 0 <= src[i] < n
        if src[i] < -1 or src[i] >= n:
            status |= 4
        elif new[i] > (old[src[i]] if named else 0):
            status |= 1
        if not 0 <= old[i] <= most or new[i] < 0:
            status |= 1
    nothing = np.full(n, -1, np.int32), np.full(n, -1, np.int32), np.zeros(n, np.int32)
    same = table, shares, stack, n_free
    if n_free < 0 or n_free > n_pages:
        status |= 8
    if status:
        return (*nothing, status, *same)
    nb = [int(pages_of(x, page)) for x in new]
    leave, come = [], []
    for i in range(n):
        first = 0 if src[i] != i else nb[i]
        leave += [(i, b) for b in range(first, int(pages_of(old[i], page)))]
        come += [(i, b, int(table[src[i], b])) for b in range(nb[i])] if src[i] != i else []
    ends = {i: int(table[src[i], new[i] // page]) for i in range(n) if src[i] >= 0 and new[i] % page}
    touched = [int(table[x]) for x in leave] + [p for _, _, p in come] + list(ends.values())
    if any(not 0 <= p < n_pages for p in touched):
        return (*nothing, 16, *same)
    holders = {p: int(shares[p]) + 1 for p in touched}
    if any(not 0 <= int(shares[p]) < 4096 for p in touched):
        return (*nothing, 32, *same)
    for x in leave:
        holders[int(table[x])] -= 1
    for _, _, p in come:
        holders[p] += 1
    if any(h < 0 for h in holders.values()):
        return (*nothing, 32, *same)
    s2, height, pushed = [int(x) for x in stack], n_free, []
    for x in leave:
        p = int(table[x])
        if holders[p] == 0 and p not in pushed:
            pushed.append(p)
    height += len(pushed)
    if height > n_pages:
        return (*nothing, 8, *same)
    for k, p in enumerate(pushed):
        s2[height - 1 - k] = p
    by_page = {}
    for i, p in ends.items():
        by_page.setdefault(p, []).append(i)
    copies = []
    for p, rows in by_page.items():
        if len(rows) > holders[p]:
            return (*nothing, 32, *same)
        keeper = min(rows, key=lambda i: (src[i] != i, i)) if len(rows) == holders[p] else None
        copies += [i for i in rows if i != keeper]
    copies.sort()
    if len(copies) > height:
        return (*nothing, 2, *same)
    t2, sh2 = table.copy(), shares.copy()
    for p in touched:
        sh2[p] = max(0, holders[p] - sum(1 for i in copies if ends[i] == p) - 1)
    for i in range(n):
        if src[i] != i:
            t2[i, :max(nb[i], int(pages_of(old[i], page)))] = -1
            t2[i, :nb[i]] = table[src[i], :nb[i]] if src[i] >= 0 else -1
        else:
            t2[i, nb[i]:int(pages_of(old[i], page))] = -1
    frm, to, rows = nothing
    for i in copies:
        height -= 1
        p = s2[height]
        if not 0 <= p < n_pages:
            return (np.full(n, -1, np.int32), np.full(n, -1, np.int32), np.zeros(n, np.int32), 16, *same)
        frm[i], to[i], rows[i] = ends[i], p, new[i] % page
        t2[i, new[i] // page], sh2[p] = p, 0
    return frm, to, rows, 0, t2, sh2, np.array(s2, np.int32), height


# ---- rules --------------------------------------------------------------------------------------------------------
def rules_ref(logits, seq, penalty, hist, hist_len, tree, bias, allow, allow_row):
    """logits [rows][V]; penalty: (repetition, presence, frequency, prompt) of each sequence or None; tree: (mask, start, tokens) or None; bias: (start, tokens, values) or None.
    In 64 bits from the f32 values."""
    rows, V = logits.shape
    out = logits.astype(np.float64)
    n_seq = len(penalty) if penalty is not None else len(bias[0]) - 1 if bias is not None else 0
    for r in range(rows):
        i = int(seq[r]) if seq is not None else r
        named = 0 <= i < n_seq
        if penalty is not None and named:
            rep, pres, freq = (float(np.float32(x)) for x in penalty[i][:3])
            rep, pres, freq = rep if rep > 0 else 1.0, 0.0 if pres != pres else pres, 0.0 if freq != freq else freq
            count, seen = {}, set()
            if hist is not None:
                text = hist[i, :max(0, min(int(hist_len[i]), hist.shape[1]))].tolist()
                seen |= set(text)
                for t in text[max(0, penalty[i][3]):]:
                    count[t] = count.get(t, 0) + 1
            if tree is not None:
                for k in range(64):
                    at = int(tree[1][i]) + k
                    if int(tree[0][r]) >> k & 1 and 0 <= at < rows:
                        t = int(tree[2][at])
                        seen.add(t)
                        count[t] = count.get(t, 0) + 1
            with np.errstate(all="ignore"):
                for t in seen:
                    if not 0 <= t < V:
                        continue
                    if rep != 1.0:
                        out[r, t] = out[r, t] / rep if out[r, t] > 0 else out[r, t] * rep
                    if t in count:
                        out[r, t] -= pres
                        if freq:
                            out[r, t] -= freq * count[t]
        if bias is not None and named:
            start, toks, vals = bias
            last = {}
            for e in range(max(0, int(start[i])), min(int(start[i + 1]), len(toks))):
                last[int(toks[e])] = float(vals[e])
            for t, x in last.items():
                if 0 <= t < V:
                    out[r, t] += x
        if allow is not None:
            g = int(allow_row[r]) if allow_row is not None else r
            if 0 <= g < len(allow):
                on = np.unpackbits(np.ascontiguousarray(allow[g]).view(np.uint8), bitorder="little")[:V].astype(bool)
                out[r, ~on] = -math.inf
    return out


# ---- calls --------------------------------------------------------------------------------------------------------
def layers_of(lg, pools, kv, hd, dev):
    """(struct lg_hip_pages [layers], device pointer) of host pools [layers][2][n_pages][page][kv * hd]."""
    p = dev.up(pools)
    n, _, n_pages, page, width = pools.shape
    step = n_pages * page * width * 2
    return (lg.hiplib.Pages * n)(*(lg.hiplib.Pages(p.value + 2 * i * step, p.value + (2 * i + 1) * step, n_pages, page, kv, hd, width, width * page) for i in range(n))), p


def tree_plan(dev, start, parent, lens, most, n_rows=None):
    n, rows = len(lens), len(parent) if n_rows is None else n_rows
    p = [dev.up(x, t) for x, t in ((start, np.int32), (parent if len(parent) else [0], np.int32), (lens, np.int32), (np.full(max(len(parent), 1), 77), np.uint64),
                                   (np.full(max(len(parent), 1), 77), np.int32), (np.full(max(len(parent), 1), 77), np.int32), (np.full(n, 77), np.int32))]
    dev.check(dev.H.lg_hip_tree_plan(n, most, rows, *p, None), "tree_plan")
    got = dev.back(p[3], len(parent), np.uint64), dev.back(p[4], len(parent), np.int32), dev.back(p[5], len(parent), np.int32), dev.back(p[6], n, np.int32)
    dev.free()
    return got


def tree_accept(dev, start, parent, token, after, lens, most, n_rows=None):
    n, rows = len(lens), len(parent) if n_rows is None else n_rows
    p = [dev.up(x if len(x) else [0], np.int32) for x in (start, parent, token, after, lens, np.full(n * most, 77), np.full(n, 77), np.full(n, 77), np.full(n, 77))]
    dev.check(dev.H.lg_hip_tree_accept(n, most, rows, *p, None), "tree_accept")
    got = (dev.back(p[5], (n, most), np.int32), *(dev.back(x, n, np.int32) for x in p[6:]))
    dev.free()
    return got


def tree_attend(lg, dev, q, k, v, table, lens, start, mask, pos, most, n_head_kv, window, scale, max_len, pad=0, n_rows=None, fill=77.0):
    """Rows of q and out `pad` values further apart than they are long."""
    rows, H, hd = q.shape
    n_pages, page = k.shape[:2]
    wide = np.full((rows, H * hd + pad), np.nan, np.float32)
    wide[:, :H * hd] = q.reshape(rows, -1)
    out = np.full((rows, H * hd + pad + (pad > 0)), fill, np.float32)      # (an odd distance, where there is any)
    n = len(lens)
    p = {name: dev.up(x) for name, x in dict(q=wide, k=k, v=v, table=table.astype(np.int32), lens=np.asarray(lens, np.int32), start=np.asarray(start, np.int32),
                                             mask=np.asarray(mask, np.uint64), pos=np.asarray(pos, np.int32), out=out).items()}
    need = dev.H.lg_hip_paged_tree_attention_workspace(n, most, H, n_head_kv, hd, max_len, window)
    work = dev.up(np.full(max(need, 4) // 4, np.nan, np.float32))
    g = lg.hiplib.Pages(p["k"].value, p["v"].value, n_pages, page, n_head_kv, hd, n_head_kv * hd, n_head_kv * hd * page)
    dev.check(dev.H.lg_hip_paged_tree_attention(C.byref(g), p["q"], wide.shape[1], rows if n_rows is None else n_rows, n, most, H, p["table"], table.shape[1], p["lens"], p["start"], p["mask"],
                                                p["pos"], max_len, window, scale, p["out"], out.shape[1], work, need, None), "paged_tree_attention")
    got = dev.back(p["out"], out.shape, np.float32)
    dev.free()
    assert (got[:, H * hd:] == fill).all(), "values between the rows were written"
    return got[:, :H * hd].reshape(rows, H, hd)


def fork(dev, page, src, old, new, table, shares, stack, n_free):
    n = len(src)
    p = [dev.up(x if np.size(x) else [0], np.int32) for x in (src, old, new, table, shares, stack, [n_free], np.full(n, 77), np.full(n, 77), np.full(n, 77), [77])]
    need = dev.H.lg_hip_paged_fork_workspace(n, stack.size, table.shape[1])
    work = dev.up(np.full(max(need, 4) // 4, -123456789, np.int32))
    dev.check(dev.H.lg_hip_paged_fork(n, page, stack.size, table.shape[1], *p, work, need, None), "paged_fork")
    got = (*(dev.back(x, n, np.int32) for x in p[7:10]), int(dev.back(p[10], 1, np.int32)[0]), dev.back(p[3], table.shape, np.int32), dev.back(p[4], shares.shape, np.int32),
           dev.back(p[5], stack.shape, np.int32), int(dev.back(p[6], 1, np.int32)[0]))
    dev.free()
    return got


def penalties(rows):
    raw = np.zeros(len(rows), np.dtype([("r", "f4"), ("a", "f4"), ("b", "f4"), ("n", "i4")]))
    for i, x in enumerate(rows):
        raw[i] = tuple(x)
    return raw


def adjust(lg, dev, logits, seq=None, penalty=None, hist=None, hist_len=None, tree=None, bias=None, allow=None, allow_row=None, pad=0, in_place=False, n_seq=None):
    rows, V = logits.shape
    wide = np.full((rows, V + pad), 55.0, np.float32)
    wide[:, :V] = logits
    r = lg.hiplib.LogitRules(n_seq=n_seq if n_seq is not None else len(penalty) if penalty is not None else len(bias[0]) - 1 if bias is not None else 0)
    up = (lambda a, t: dev.up(np.asarray(a), t).value)  # noqa: E731
    if seq is not None:
        r.seq = up(seq, np.int32)
    if penalty is not None:
        r.penalty = dev.up(penalties(penalty).view(np.uint8)).value
    if hist is not None:
        r.hist, r.hist_len, r.hist_stride = up(hist, np.int32), up(hist_len, np.int32), hist.shape[1]
    if tree is not None:
        r.tree_mask, r.tree_start, r.tree_tok = up(tree[0], np.uint64), up(tree[1], np.int32), up(tree[2], np.int32)
    if bias is not None:
        r.n_bias, r.bias_start, r.bias_tok, r.bias = len(bias[1]), up(bias[0], np.int32), up(bias[1], np.int32), up(bias[2], np.float32)
    if allow is not None:
        r.n_allow, r.allow, r.allow_stride = len(allow), dev.up(np.asarray(allow, np.uint32)).value, allow.shape[1]
        if allow_row is not None:
            r.allow_row = up(allow_row, np.int32)
    x = dev.up(wide)
    out = x if in_place else dev.up(np.full(wide.shape, 77.0, np.float32))
    dev.check(dev.H.lg_hip_adjust_logits(C.byref(r), x, V + pad, rows, V, out, V + pad, None), "adjust_logits")
    got = dev.back(out, wide.shape, np.float32)
    if not in_place:
        assert np.array_equal(dev.back(x, wide.shape, np.float32), wide, equal_nan=True), "the logits themselves were written"
    dev.free()
    assert (got[:, V:] == (55.0 if in_place else 77.0)).all(), "values between the rows were written"
    return got[:, :V]
