"""Plain forms of the operators of a batched decode step (plan, write, attend, sample) in 64 bits, and calls of the C ABI with host arrays."""
import ctypes as C
import math

import numpy as np

from test_zz_no_alloc import DeviceBuffers

ONE = 1 << 44


def pages_of(n, page):
    return -(-np.asarray(n, np.int64) // page)


# ---- plain forms --------------------------------------------------------------------------------------------------
def plan_ref(page, old, new, table, stack, n_free, n_slots):
    """(start, slots, status, table, stack, n_free) after a step, sequence by sequence."""
    n_pages, most = stack.size, table.shape[1] * page
    n = len(old)
    bad = (np.zeros(n + 1, np.int32), np.full(n_slots, -1, np.int32))
    status = 0
    if any(x < 0 or x > most for x in [*old, *new]):
        return (*bad, 1, table, stack, n_free)
    need = int(np.maximum(0, pages_of(new, page) - pages_of(old, page)).sum()) if n else 0
    freed = int(np.maximum(0, pages_of(old, page) - pages_of(new, page)).sum()) if n else 0
    total = int(np.maximum(0, np.asarray(new, np.int64) - np.asarray(old, np.int64)).sum()) if n else 0
    if n_free < 0 or n_free > n_pages or n_free + freed > n_pages:
        status |= 8
    elif need > n_free + freed:
        status |= 2
    if total > n_slots:
        status |= 4
    if status:
        return (*bad, status, table, stack, n_free)
    t2, s2 = table.copy(), [int(x) for x in stack]
    put = [(i, b) for i in range(n) for b in range(pages_of(new[i], page), pages_of(old[i], page))]
    for i, b in put:
        if not 0 <= table[i, b] < n_pages:
            return (*bad, 16, table, stack, n_free)
        t2[i, b] = -1
    for (i, b), at in zip(put, range(n_free + freed - 1, -1, -1)):
        s2[at] = int(table[i, b])
    top = n_free + freed
    for i in range(n):
        if new[i] > old[i] and old[i] % page and not 0 <= table[i, old[i] // page] < n_pages:
            return (*bad, 16, table, stack, n_free)
        for b in range(pages_of(old[i], page), pages_of(new[i], page)):
            top -= 1
            if not 0 <= s2[top] < n_pages:
                return (*bad, 16, table, stack, n_free)
            t2[i, b] = s2[top]
    start, slots = [0], []
    for i in range(n):
        slots += [int(t2[i, p // page]) * page + p % page for p in range(old[i], new[i])]
        start.append(len(slots))
    slots += [-1] * (n_slots - len(slots))
    return np.array(start, np.int32), np.array(slots, np.int32), 0, t2, np.array(s2, np.int32), top


def attend_ref(q, k, v, table, lens, page, n_pages, n_head_kv, window, scale, max_len):
    """q [n][H][hd]; k, v [n_pages][page][kv][hd] binary16.  Returns (out, bound) in 64 bits: the result, and how far a
    kernel of the documented roundings may be from it (see tolerance)."""
    n, H, hd = q.shape
    G = H // n_head_kv
    out, bound = np.zeros((n, H, hd)), np.zeros((n, H, 1))
    for i in range(n):
        L = max(0, min(int(lens[i]), max_len, table.shape[1] * page))
        pos = np.arange(max(0, L - window) if window else 0, L)
        pos = pos[(table[i, pos // page] >= 0) & (table[i, pos // page] < n_pages)]
        if not pos.size:
            continue
        rows = (table[i, pos // page], pos % page)
        kk, vv = k[rows].astype(np.float64), v[rows].astype(np.float64)             # [keys][kv][hd]
        for h in range(H):
            x = scale * (kk[:, h // G] @ q[i, h].astype(np.float64))
            e = np.exp(x - x.max())
            out[i, h] = e @ vv[:, h // G] / e.sum()
            size = abs(scale) * np.max(np.abs(kk[:, h // G]) @ np.abs(q[i, h].astype(np.float64)))
            bound[i, h] = tolerance(size, hd, pos.size) * np.max(np.abs(vv[:, h // G]))
    return out, bound


def tolerance(size, hd, keys):
    """Relative to the largest value.  A score: its query in 22 bits (2^-21 with both truncations), hd products added in f32 in any order
    (hd 2^-24), the two halves added and the scale applied (4 more roundings), all relative to `size`, the sum of the products'
    magnitudes.  Its exponential moves by as much, and by 2^-21 for the instruction and the argument's own rounding, 2^-21 for its two
    binary16 parts; numerator and denominator add `keys` terms in f32 (2^-24 each, either side), and 16 joins and the division."""
    score = size * (2.0 ** -21 + (hd + 4) * 2.0 ** -24)
    return 2 * (score + 2.0 ** -20) + 2 * (keys + 16) * 2.0 ** -24


def within(got, want, bound, what=""):
    off = np.abs(got - want)
    bad = np.argwhere(~(off <= bound))
    worst = float(np.nanmax(off / np.maximum(bound, 1e-300))) if off.size else 0.0
    assert not bad.size, f"{what}: {len(bad)} of {off.size} values outside, the first at {bad[0].tolist()}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}; {worst:.3g} times the bound"


def weights(l, T):
    """Whole-number weights of a row, and its largest logit (-inf: none)."""
    l = np.where(np.isnan(l), -np.inf, np.asarray(l, np.float64))
    top = l.max()
    if top == -np.inf:
        return np.zeros(l.size, np.int64), top
    with np.errstate(all="ignore"):
        d = np.where(l == top, 0.0, np.where(np.isinf(l), -np.inf, (l - top) / np.float64(np.float32(T))))
    return np.rint(np.exp(d) * ONE).astype(np.int64), top


def sample_ref(l, T, k, p, m, u):
    """(token, probability, kept, clear): `clear` is false where the last bits of some weights could decide.  A weight other than the largest
    logit's may be one unit off (the exponential's own rounding), so a sum of them as many units as it has terms."""
    T, p, m, u = (np.float32(x) for x in (T, p, m, u))
    greedy = not T > 0
    w, top = weights(l, 1.0 if greedy else T)
    if top == -np.inf:
        return -1, 0.0, 0, True
    order = np.lexsort((np.arange(w.size), -np.where(np.isnan(l), -np.inf, l)))
    order = order[w[order] > 0]
    n, clear = order.size, True
    if k > 0:
        n = min(n, int(k))
    if greedy:
        n = 1
    slack = int((w[order[:n]] < ONE).sum())
    slack += 2 * (slack > 0)
    if p < 1:
        sums = []
        for x in w[order[:n]].tolist():
            sums.append(x + (sums[-1] if sums else 0))
        want = max(1, math.ceil(float(p) * float(sums[-1])))
        border = int(np.searchsorted(np.array(sums, np.uint64), np.uint64(want)))
        clear &= all(abs(want - s) > slack or not slack for s in sums[max(0, border - 1):border + 2])
        n = min(n, border + 1)
    keep = order[:n]
    if m > 0:
        least = min(1.0, float(m)) * ONE
        clear &= bool(np.all((np.abs(w[order] - least) > 2) | (w[order] == ONE)))
        keep = keep[w[keep] >= least]
    keep = np.sort(keep)
    run = []
    for x in w[keep].tolist():
        run.append(x + (run[-1] if run else 0))
    S = run[-1]
    r = min(math.floor(min(max(float(u), 0.0), 1.0) * float(S)), S - 1) if u == u else 0
    j = int(np.searchsorted(np.array(run, np.uint64), np.uint64(r), side="right"))
    if slack:
        clear &= run[j] - r > slack and (r == 0 or j == 0 or r - run[j - 1] > slack)
    return int(keep[j]), int(w[keep[j]]) / S, int(keep.size), clear


# ---- calls --------------------------------------------------------------------------------------------------------
class Device(DeviceBuffers):
    """Arrays on the device and the C ABI's calls on them, on the default stream unless told otherwise."""

    def __init__(self, lg):
        self.lg, self.H = lg, lg.hiplib.load_hip()
        super().__init__()

    def up(self, a, dtype=None):
        return self.upload(np.ascontiguousarray(a, dtype))

    def room(self, nbytes):
        p = C.c_void_p()
        assert self.rt.hipMalloc(C.byref(p), C.c_size_t(max(int(nbytes), 256))) == 0
        self.held.append(p)
        return p

    def put(self, p, arr):
        arr = np.ascontiguousarray(arr)
        assert self.rt.hipMemcpy(p, arr.ctypes.data_as(C.c_void_p), C.c_size_t(arr.nbytes), 1) == 0

    def back(self, p, shape, dtype):
        out = np.zeros(shape, dtype)
        self.download(p, out)
        return out

    def check(self, rc, what):
        self.lg.hiplib.hip_check(rc, what)


def plan(dev, page, old, new, table, stack, n_free, n_slots, stream=None):
    n = len(old)
    p = [dev.up(x, np.int32) for x in (old, new, table, stack, [n_free], np.full(n + 1, 77), np.full(max(n_slots, 1), 77), [77])]
    need = dev.H.lg_hip_paged_plan_workspace(n)
    rc = dev.H.lg_hip_paged_plan(n, page, stack.size, table.shape[1], *p[:7], n_slots, p[7], dev.room(need), need, stream)
    dev.check(rc, "paged_plan")
    start, slots, status = dev.back(p[5], n + 1, np.int32), dev.back(p[6], max(n_slots, 1), np.int32)[:n_slots], int(dev.back(p[7], 1, np.int32)[0])
    got = (start, slots, status, dev.back(p[2], table.shape, np.int32), dev.back(p[3], stack.shape, np.int32), int(dev.back(p[4], 1, np.int32)[0]))
    dev.free()
    return got


def sample(dev, logits, params, u, stride=None):
    rows, V = logits.shape
    stride = stride or V
    wide = np.full((rows, stride), np.inf, np.float32)                 # what lies between the rows is not theirs
    wide[:, :V] = logits
    raw = np.zeros(rows, np.dtype([("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")]))
    for i, x in enumerate(params):
        raw[i] = x
    p = [dev.up(wide), dev.up(raw.view(np.uint8)), dev.up(u, np.float32), dev.up(np.full(rows, 77), np.int32), dev.up(np.full(rows, 77.0), np.float32), dev.up(np.full(rows, 77), np.int32)]
    need = dev.H.lg_hip_sample_workspace(rows, V)
    dev.check(dev.H.lg_hip_sample(p[0], stride, rows, V, *p[1:], dev.room(need), need, None), "sample")
    got = dev.back(p[3], rows, np.int32), dev.back(p[4], rows, np.float32), dev.back(p[5], rows, np.int32)
    dev.free()
    return got
