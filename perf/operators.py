"""Operators of a batched decode step: what a program that serves many sequences at once calls between its matrix products.

  plan    block tables, slots of the new tokens and the stack of free pages, from the lengths before and after a step
  write   the K and V rows of new tokens into their slots, as binary16
  attend  attention of one new token per sequence over the pages of its table
  sample  tokens drawn from logits rows by given random numbers (temperature, top-k, top-p, min-p)

With `own` false, `run` computes them from elementary torch operations; with it true, it calls the C ABI of liblg_hip.so
(include/lg_hip.h) as a program bound to it by FFI does.  Head layouts, windows, cache lengths and vocabularies are those of
little-gemma_amd/synth.py: the E4B shape (8 query and 2 key heads of 256, window 512, 262144 tokens), the 12B shape
(16 and 8 heads of 256, window 1024) and the tiny ones (8 and 2 heads of 64, 8192 tokens).
"""
import ctypes as C
import math

import numpy as np
import torch

own = False
ONE = 2.0 ** 44                      # the weight of a row's largest logit, in the whole numbers that sampling sums


# ---- the cases ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one more token for every conversation of a server, pages of 16: the call before each decode step
        dict(name="plan decode 64", kind="plan", n_seq=64, page=16, ctx=4096, grow=1, shrink=0),
        # prompts of up to 2000 tokens come in while other conversations take rejected drafts back
        dict(name="plan prompts 333", kind="plan", n_seq=333, page=32, ctx=8191, grow=2000, shrink=7),
        # the new rows of a decode step of 64 conversations, E4B heads
        dict(name="write decode 64", kind="write", n_tok=64, kv=2, hd=256, page=16, fused=8),
        # prompts of together 20011 tokens, 12B heads
        dict(name="write prompts 20011", kind="write", n_tok=20011, kv=8, hd=256, page=64, fused=16),
        # the smallest call: one short conversation of the tiny model
        dict(name="attend tiny", kind="attend", n_seq=1, heads=8, kv=2, hd=64, page=16, ctx=100, window=0, ragged=False, scaled=False),
        # a sliding layer of the E4B shape for 64 conversations of all lengths
        dict(name="attend e4b window", kind="attend", n_seq=64, heads=8, kv=2, hd=256, page=16, ctx=4096, window=512, ragged=True, scaled=False),
        # a global layer of it for 61
        dict(name="attend e4b global", kind="attend", n_seq=61, heads=8, kv=2, hd=256, page=32, ctx=8192, window=0, ragged=True, scaled=False),
        # one long document, 12B heads: few rows, a long axis
        dict(name="attend 12b long", kind="attend", n_seq=1, heads=16, kv=8, hd=256, page=64, ctx=100003, window=0, ragged=False, scaled=False),
        # a full server of the larger model
        dict(name="attend 12b full", kind="attend", n_seq=24, heads=16, kv=8, hd=256, page=32, ctx=16384, window=0, ragged=False, scaled=False),
        # chat: one row, the settings that models of this family recommend
        dict(name="sample chat", kind="sample", rows=1, vocab=262144, mode="chat"),
        # a verify block of 5 rows by nucleus sampling alone: no bound on how many tokens stay
        dict(name="sample nucleus 5", kind="sample", rows=5, vocab=262144, mode="nucleus"),
        # a batch in which every conversation brings its own settings, some rows masked by a grammar
        dict(name="sample mixed 64", kind="sample", rows=64, vocab=262144, mode="mixed"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("plan", "write", "attend", "sample"), (2, 2, 5, 4))[0]
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "plan":
        grow = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 2000)
        return dict(kind=kind, n_seq=_log_uniform(rng, 1, 333), page=page, ctx=_log_uniform(rng, 33, 8191), grow=grow, shrink=rng.choice((0, 1, 7, 300)))
    if kind == "write":
        kv, hd = rng.choice(((2, 64), (2, 128), (2, 256), (8, 256), (1, 512), (4, 128)))
        return dict(kind=kind, n_tok=_log_uniform(rng, 1, 20011), kv=kv, hd=hd, page=page, fused=rng.choice((0, kv, 2 * kv, 4 * kv)))
    if kind == "attend":
        heads, kv, hd = rng.choice(((8, 2, 64), (8, 2, 128), (8, 2, 256), (16, 8, 256), (8, 1, 512), (8, 8, 128), (5, 1, 64), (12, 4, 256)))
        window = 0 if rng.random() < 0.5 else rng.choice((128, 512, 1024, 333))
        ctx = _log_uniform(rng, 1, 60000)
        keys = 24 * 16384 * 8 * 256 // (kv * hd)                       # of the largest listed case
        n_seq = _log_uniform(rng, 1, max(1, min(128, keys // ctx)))
        return dict(kind=kind, n_seq=n_seq, heads=heads, kv=kv, hd=hd, page=page, ctx=ctx, window=window, ragged=rng.random() < 0.6, scaled=rng.random() < 0.3)
    vocab = rng.choice((8192, 262144, _log_uniform(rng, 300, 262144)))
    rows = _log_uniform(rng, 1, 64)
    return dict(kind=kind, rows=rows, vocab=vocab, mode=rng.choice(("chat", "nucleus", "plain", "min_p", "mixed")))


# ---- states -------------------------------------------------------------------------------------------------------
class _State:
    pass


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _quantiles(n, most, ragged):
    """Lengths of n sequences: all `most`, or from a free place (0) up to it, half of them under a quarter."""
    if not ragged:
        return np.full(n, most, np.int64)
    return np.round(most * (np.arange(1 if n < 8 else 0, n + (1 if n < 8 else 0)) / (n if n < 8 else n - 1)) ** 2).astype(np.int64)


def _plan_lengths(c):
    """(before, after) a step: growth by `grow` (1) or by up to it, every third sequence taking up to `shrink` back."""
    n = c["n_seq"]
    before = _quantiles(n, c["ctx"], True)
    after = before + (1 if c["grow"] == 1 else np.ceil(c["grow"] * ((np.arange(n) * 7 % n + 1) / n) ** 2).astype(np.int64))
    if c["shrink"]:
        back = np.arange(n) % 3 == 2
        after[back] = np.maximum(0, before[back] - 1 - np.arange(n)[back] % c["shrink"])
    return before, after


def _pages(n, page):
    return -(-n // page)


def _prepare_plan(s, c, rng):
    before, after = _plan_lengths(c)
    at = rng.permutation(c["n_seq"])
    before, after = before[at], after[at]
    P = c["page"]
    most = int(max(before.max(), after.max()))
    s.blocks = _pages(most, P) + 1
    held, wants = _pages(before, P), _pages(np.maximum(before, after), P)
    s.n_pages = int(wants.sum()) + 64
    ids = rng.permutation(s.n_pages)
    table = np.full((c["n_seq"], s.blocks), -1, np.int32)
    first = np.cumsum(held) - held
    cols = np.arange(s.blocks)[None, :]
    inside = cols < held[:, None]
    table[inside] = ids[(first[:, None] + cols)[inside]]
    stack = np.zeros(s.n_pages, np.int32)
    free = ids[int(held.sum()):]
    stack[:free.size] = free
    s.n_new, s.n_back = int(np.maximum(0, after - before).sum()), int(np.maximum(0, before - after).sum())
    s.n_slots = max(s.n_new, s.n_back) + 3                             # a captured step's fixed room
    s.len_old, s.len_new, s.table, s.stack, s.n_free = _i32(before), _i32(after), _i32(table), _i32(stack), _i32([free.size])
    s.start, s.slots, s.status = _i32(np.zeros(c["n_seq"] + 1)), _i32(np.zeros(s.n_slots)), _i32([0])
    s.start2, s.slots2, s.status2 = _i32(np.zeros(c["n_seq"] + 1)), _i32(np.zeros(s.n_slots)), _i32([0])


def _rows_of(gen, n, heads, kv, hd):
    """Rows as a fused q/k/v product leaves them: [n][(heads + 2 kv) * hd] floats, and their three parts."""
    x = torch.randn((n, (heads + 2 * kv) * hd), generator=gen, device="cuda")
    return x, x[:, :heads * hd], x[:, heads * hd:(heads + kv) * hd], x[:, (heads + kv) * hd:]


def _prepare_write(s, c, rng, gen):
    n, P, width = c["n_tok"], c["page"], c["kv"] * c["hd"]
    s.n_pages = _pages(n, P) + 5
    s.x, _, s.k, s.v = _rows_of(gen, n, c["fused"], c["kv"], c["hd"])
    # runs of tokens of many sequences; every 29th place is padding
    slots = (rng.permutation(s.n_pages)[:, None] * P + np.arange(P)[None, :]).reshape(-1)[:n]
    slots[28::29] = -1
    s.slots = _i32(slots)
    s.kpool, s.vpool = (torch.zeros((s.n_pages, P, width), dtype=torch.float16, device="cuda") for _ in range(2))


def _lengths(c):
    return _quantiles(c["n_seq"], c["ctx"], c["ragged"])


def _prepare_attend(s, c, rng, gen):
    n, P, hd, kv = c["n_seq"], c["page"], c["hd"], c["kv"]
    lens = rng.permutation(_lengths(c))
    s.blocks = max(1, _pages(c["ctx"], P))
    held = _pages(lens, P)
    s.n_pages = int(held.sum()) + 3
    ids = rng.permutation(s.n_pages)
    table = np.full((n, s.blocks), -1, np.int32)
    cols = np.arange(s.blocks)[None, :]
    inside = cols < held[:, None]
    table[inside] = ids[((np.cumsum(held) - held)[:, None] + cols)[inside]]
    s.table, s.lens, s.max_len = _i32(table), _i32(lens), c["ctx"]
    s.kpool, s.vpool = (torch.randn((s.n_pages, P, kv * hd), generator=gen, device="cuda", dtype=torch.float16) for _ in range(2))
    # scores of a spread of 2, where attention picks some keys and averages over many
    s.scale = hd ** -0.5 if c["scaled"] else 1.0
    s.x, s.q, _, _ = _rows_of(gen, n, c["heads"], kv, hd)
    s.x *= 2.0 if c["scaled"] else 2.0 * hd ** -0.5
    s.out = torch.zeros((n, c["heads"] * hd), device="cuda")


MODES = {  # temperature, top-k, top-p, min-p
    "chat": ((1.0, 64, 0.95, 0.0),),
    "nucleus": ((0.8, 0, 0.9, 0.0),),
    "plain": ((1.0, 0, 1.0, 0.0),),
    "min_p": ((1.5, 0, 1.0, 0.05),),
    "mixed": ((1.0, 64, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 5000, 0.98, 0.0), (1.5, 0, 1.0, 0.1),
              (1.0, 0, 1.0, 0.0), (0.6, 1, 1.0, 0.0), (2.0, 200, 0.5, 0.02)),
}


def _prepare_sample(s, c, rng, gen):
    rows, V = c["rows"], c["vocab"]
    z = torch.randn((rows, V), generator=gen, device="cuda") * 3.0
    # a few likely tokens in every row, from nearly certain to hardly any
    peaks = torch.randint(0, V, (rows, 24), generator=gen, device="cuda")
    lift = 14.0 * torch.rand((rows, 24), generator=gen, device="cuda") * torch.rand((rows, 1), generator=gen, device="cuda")
    z.scatter_add_(1, peaks, lift)
    l = 30.0 * torch.tanh(z / 30.0)
    if c["mode"] == "mixed":
        r = torch.arange(rows, device="cuda")
        l = torch.where((r % 4 == 1)[:, None], l.to(torch.bfloat16).to(torch.float32), l)           # a head that answers in bfloat16: many ties
        l = torch.where((r % 7 == 3)[:, None] & (torch.rand((rows, V), generator=gen, device="cuda") < 0.7), float("-inf"), l)
    s.logits = l.contiguous()
    m = MODES[c["mode"]]
    p = [m[i % len(m)] for i in range(rows)]
    s.temp, s.top_p, s.min_p = (torch.tensor([x[j] for x in p], dtype=torch.float32, device="cuda") for j in (0, 2, 3))
    s.top_k = _i32([x[1] for x in p])
    raw = np.zeros(rows, np.dtype([("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")]))
    for j, name in enumerate("tkpm"):
        raw[name] = [x[j] for x in p]
    s.params = torch.from_numpy(raw.view(np.uint8).reshape(rows, 16).copy()).cuda()                 # as struct lg_hip_sampling
    s.u = torch.rand(rows, generator=gen, device="cuda")
    s.tok, s.kept, s.prob = _i32(np.zeros(rows)), _i32(np.zeros(rows)), torch.zeros(rows, device="cuda")


def prepare(case, seed):
    s, rng = _State(), np.random.default_rng(seed)
    s.case = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "plan":
        _prepare_plan(s, case, rng)
    elif case["kind"] == "write":
        _prepare_write(s, case, rng, gen)
    elif case["kind"] == "attend":
        _prepare_attend(s, case, rng, gen)
    else:
        _prepare_sample(s, case, rng, gen)
    s.device, s.calls = torch.cuda.current_device(), {}
    return s


# ---- the framework's calls ----------------------------------------------------------------------------------------
_lib = None


def _own():
    global _lib
    if _lib is None:
        import importlib
        _lib = importlib.import_module("little-gemma_amd").hiplib
        _lib.load_hip()
    return _lib


def _pool(s):
    c = s.case
    width = c["kv"] * c["hd"]
    return _own().Pages(s.kpool.data_ptr(), s.vpool.data_ptr(), s.n_pages, c["page"], c["kv"], c["hd"], width, width * c["page"])


def _bound(s, stream):
    """The call of a state on a stream with its arguments in place, as a serving loop keeps it: pointers, handles, working memory of the stream's own.
    (call, arguments of each call in turn, the memory)"""
    L, c, work = _own(), s.case, []
    H, p, stream = L.load_hip(), (lambda t: C.c_void_p(t.data_ptr())), C.c_void_p(stream)

    def memory(n):
        work.append(torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"))
        return p(work[0]), C.c_size_t(n)

    if c["kind"] == "plan":
        w = memory(H.lg_hip_paged_plan_workspace(c["n_seq"]))
        head = (c["n_seq"], c["page"], s.n_pages, s.blocks)
        a = (*head, p(s.len_old), p(s.len_new), p(s.table), p(s.stack), p(s.n_free), p(s.start), p(s.slots), s.n_slots, p(s.status), *w, stream)
        b = (*head, p(s.len_new), p(s.len_old), p(s.table), p(s.stack), p(s.n_free), p(s.start2), p(s.slots2), s.n_slots, p(s.status2), *w, stream)
        return H.lg_hip_paged_plan, (a, b), work
    if c["kind"] == "write":
        return H.lg_hip_paged_write, ((C.byref(_pool(s)), p(s.k), p(s.v), s.x.shape[1], p(s.slots), c["n_tok"], stream),), work
    if c["kind"] == "attend":
        w = memory(H.lg_hip_paged_attention_workspace(c["n_seq"], c["heads"], c["kv"], c["hd"], s.max_len, c["window"]))
        return H.lg_hip_paged_attention, ((C.byref(_pool(s)), p(s.q), s.x.shape[1], c["n_seq"], c["heads"], p(s.table), s.blocks, p(s.lens), s.max_len,
                                           c["window"], s.scale, p(s.out), s.out.shape[1], *w, stream),), work
    w = memory(H.lg_hip_sample_workspace(c["rows"], c["vocab"]))
    return H.lg_hip_sample, ((p(s.logits), c["vocab"], c["rows"], c["vocab"], p(s.params), p(s.u), p(s.tok), p(s.prob), p(s.kept), *w, stream),), work


def _run_own(s):
    # the stream that is current now (its handle alone: 0.1 us, a Stream object 2.8)
    stream = torch._C._cuda_getCurrentRawStream(s.device)
    if stream not in s.calls:
        s.calls[stream] = _bound(s, stream)
    f, passes, _ = s.calls[stream]
    for args in passes:
        rc = f(*args)
        if rc:
            _own().hip_check(rc, s.case["kind"])


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _plan(s, len_old, len_new, start, slots, status):
    P, n = s.case["page"], s.case["n_seq"]
    a, b = len_old.long(), len_new.long()
    na, nb = (a + P - 1) // P, (b + P - 1) // P
    freed, need, new = (na - nb).clamp(min=0), (nb - na).clamp(min=0), (b - a).clamp(min=0)
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    F, N, T = (torch.cat([zero, x.cumsum(0)]) for x in (freed, need, new))
    top = s.n_free.long() + F[-1:]                                     # the stack's height once the freed pages are on it
    col = torch.arange(s.blocks, device="cuda")[None, :]
    table = s.table.long()
    # push: one scatter over the table's places, those that free nothing go to a place behind the stack
    e = F[:n, None] + col - nb[:, None]
    gone = (col >= nb[:, None]) & (col < na[:, None])
    stack = torch.cat([s.stack.long(), zero]).scatter(0, torch.where(gone, top - 1 - e, s.n_pages).reshape(-1), table.reshape(-1))[:-1]
    # pop
    e = N[:n, None] + col - na[:, None]
    come = (col >= na[:, None]) & (col < nb[:, None])
    table = torch.where(come, stack[(top - 1 - e).clamp(0, s.n_pages - 1)], torch.where(gone, -1, table))
    s.table.copy_(table)
    s.stack.copy_(stack)
    s.n_free.copy_(top - N[-1:])
    start.copy_(T)
    j = torch.arange(s.n_slots, device="cuda")
    i = torch.searchsorted(T[1:], j, right=True).clamp(max=n - 1)
    pos = (a[i] + j - T[i]).clamp(min=0)
    slots.copy_(torch.where(j < T[-1:], table[i, (pos // P).clamp(max=s.blocks - 1)] * P + pos % P, -1))
    status.zero_()


def _write(s):
    n = s.n_pages * s.case["page"]
    idx = s.slots.long()
    ok = (idx >= 0) & (idx < n)
    for pool, rows in ((s.kpool, s.k), (s.vpool, s.v)):
        flat = pool.view(n, -1)
        flat[idx[ok]] = rows[ok].to(torch.float16)


def _attend(s):
    c, P, G = s.case, s.case["page"], s.case["heads"] // s.case["kv"]
    n, hd, kv = c["n_seq"], c["hd"], c["kv"]
    span = s.max_len if not c["window"] else min(s.max_len, c["window"])
    lens = s.lens.long()
    first = (lens - span).clamp(min=0)
    pos = first[:, None] + torch.arange(span, device="cuda")[None, :]                                # [n][span]
    seen = pos < lens[:, None]
    page = torch.gather(s.table.long(), 1, (pos // P).clamp(max=s.blocks - 1)).clamp(min=0)
    row = torch.where(seen, page * P + pos % P, 0).reshape(-1)
    # few sequences at a time where the gathered rows would not fit the card twice over
    outs, step = [], max(1, (1 << 31) // (span * kv * hd))
    for i in range(0, n, step):
        m = min(step, n - i)
        r, ok = row[i * span:(i + m) * span], seen[i:i + m, None, None, :]
        k = s.kpool.view(-1, kv, hd)[r].float().view(m, span, kv, hd).permute(0, 2, 3, 1).contiguous()
        q = s.q[i:i + m].reshape(m, kv, G, hd) * s.scale
        x = torch.where(ok, torch.matmul(q, k), float("-inf"))
        top = x.amax(-1, keepdim=True)
        e = torch.where(ok, torch.exp(x - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
        del k, x
        v = s.vpool.view(-1, kv, hd)[r].float().view(m, span, kv, hd).permute(0, 2, 1, 3).contiguous()
        o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        outs.append(torch.where(lens[i:i + m, None, None, None] > 0, o, 0.0).reshape(m, -1))
    s.out.copy_(torch.cat(outs))


def _sample(s):
    V = s.case["vocab"]
    l = torch.where(torch.isnan(s.logits), float("-inf"), s.logits)
    order = torch.sort(l, dim=1, descending=True, stable=True)
    x = order.values.double()
    top = x[:, :1]
    greedy = ~(s.temp > 0)
    T = torch.where(greedy, 1.0, s.temp.double())[:, None]
    d = torch.where(x == top, 0.0, torch.where(torch.isinf(x), float("-inf"), (x - top) / T))
    w = torch.round(torch.exp(d) * ONE).long()                                                       # whole numbers: their sums have no order
    rank = torch.arange(V, device="cuda")[None, :]
    k = torch.where(greedy, 1, torch.where(s.top_k > 0, s.top_k.long(), V))[:, None]
    w = torch.where(rank < k, w, 0)
    run = w.cumsum(1)
    need = torch.ceil(s.top_p.double()[:, None] * run[:, -1:].double()).long().clamp(min=1)
    w = torch.where((run - w < need) | ~(s.top_p < 1)[:, None], w, 0)
    w = torch.where((w.double() >= s.min_p.double()[:, None] * ONE) | ~(s.min_p > 0)[:, None], w, 0)
    by_index = torch.zeros_like(w).scatter(1, order.indices, w)
    run = by_index.cumsum(1)
    total = run[:, -1:]
    r = torch.minimum(torch.floor(s.u.double()[:, None].clamp(min=0) * total.double()).long(), total - 1)
    tok = (run <= r).sum(1).clamp(max=V - 1)
    any_ = (total > 0)[:, 0] & ~torch.isneginf(top[:, 0])
    s.tok.copy_(torch.where(any_, tok, -1))
    s.kept.copy_(torch.where(any_, (w > 0).sum(1), 0))
    s.prob.copy_(torch.where(any_, by_index.gather(1, tok[:, None])[:, 0].double() / total[:, 0].clamp(min=1).double(), 0.0))


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    kind = s.case["kind"]
    if own:
        _run_own(s)
    elif kind == "plan":
        _plan(s, s.len_old, s.len_new, s.start, s.slots, s.status)
        _plan(s, s.len_new, s.len_old, s.start2, s.slots2, s.status2)
    elif kind == "write":
        _write(s)
    elif kind == "attend":
        _attend(s)
    else:
        _sample(s)
    if kind == "plan":               # a step's plan, and the plan that takes the step back: the pages are as before
        return {"start": s.start, "slots": s.slots, "status": s.status, "table": s.table, "stack": s.stack, "free": s.n_free,
                "back_start": s.start2, "back_slots": s.slots2, "back_status": s.status2}
    if kind == "write":
        return {"k": s.kpool, "v": s.vpool}
    if kind == "attend":
        return {"out": s.out}
    return {"token": s.tok, "prob": s.prob, "kept": s.kept}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "plan":
        a, b = _plan_lengths(c)
        moved = np.abs(_pages(b, c["page"]) - _pages(a, c["page"])).sum()
        grown, back = np.maximum(0, b - a).sum(), np.maximum(0, a - b).sum()
        slots = max(grown, back) + 3
        # lengths twice, starts, slots, the table's entry of each written block, and for a page that moves a stack and a table entry
        return {"bytes": float(2 * (8 * c["n_seq"] + 4 * (c["n_seq"] + 1) + 4 * slots) + 4 * (grown + back) / c["page"] + 2 * 8 * moved), "flops": 0.0}
    if c["kind"] == "write":
        n = c["n_tok"] - c["n_tok"] // 29
        return {"bytes": float(n * 2 * c["kv"] * c["hd"] * (4 + 2) + 4 * c["n_tok"]), "flops": 0.0}
    if c["kind"] == "attend":
        lens = _lengths(c)
        keys = int((np.minimum(lens, c["window"]) if c["window"] else lens).sum())
        rows = 2 * 4 * c["n_seq"] * c["heads"] * c["hd"]
        return {"bytes": float(4 * keys * c["kv"] * c["hd"] + rows + 4 * keys / c["page"]), "flops": 4.0 * c["heads"] * c["hd"] * keys}
    return {"bytes": float(c["rows"] * (4 * c["vocab"] + 32)), "flops": 20.0 * c["rows"] * c["vocab"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_sample(s):
    """Row by row from the definition: the border of each filter by sorted values, the draw by searching the running sums."""
    V, toks, probs, kepts = s.case["vocab"], [], [], []
    for i in range(s.case["rows"]):
        l = s.logits[i].double()
        T, k, p, m, u = (float(x[i]) for x in (s.temp, s.top_k, s.top_p, s.min_p, s.u))
        best = l[~torch.isnan(l)].max().item() if bool((l > -math.inf).any()) else -math.inf
        if best == -math.inf:
            toks.append(-1), probs.append(0.0), kepts.append(0)
            continue
        ids = torch.nonzero(l > -math.inf)[:, 0]
        ids = ids[torch.argsort(-l[ids], stable=True)]
        w = torch.where(l[ids] == best, 1.0, torch.exp((l[ids] - best) / (T if T > 0 else 1.0))) * ONE
        w = torch.floor(w + 0.5).long()
        n = min(int(k), len(ids)) if k > 0 else len(ids)
        if T <= 0:
            n = 1
        if p < 1:
            sums = w[:n].cumsum(0)
            want = max(1, math.ceil(p * float(sums[-1])))
            n = min(n, int((sums < want).sum()) + 1)
        keep = torch.arange(len(ids), device="cuda") < n
        keep &= w > 0
        if m > 0:
            keep &= w.double() >= m * ONE
        ids, w = ids[keep], w[keep]
        ids, by = torch.sort(ids)
        sums = w[by].cumsum(0)
        total = int(sums[-1])
        r = min(math.floor(max(u, 0.0) * float(total)), total - 1)
        j = int((sums <= r).sum())
        toks.append(int(ids[j])), probs.append(int(w[by][j]) / total), kepts.append(len(ids))
    return {"token": np.array(toks, np.int32), "prob": np.array(probs, np.float64), "kept": np.array(kepts, np.int32)}


def _exact_attend(s):
    c, P, G = s.case, s.case["page"], s.case["heads"] // s.case["kv"]
    lens, table = s.lens.cpu().numpy(), s.table.cpu().numpy()
    out = torch.zeros((c["n_seq"], c["kv"], G, c["hd"]), dtype=torch.float64, device="cuda")
    for i, n in enumerate(int(x) for x in lens):
        if not n:
            continue
        lo = max(0, n - c["window"]) if c["window"] else 0
        ids = torch.from_numpy(table[i, :_pages(n, P)].astype(np.int64)).cuda()
        k, v = (pool[ids].reshape(-1, c["kv"], c["hd"])[lo:n].double().transpose(0, 1).contiguous() for pool in (s.kpool, s.vpool))
        q = s.q[i].double().view(c["kv"], G, c["hd"]) * s.scale
        x = torch.matmul(k, q.transpose(1, 2).contiguous()).transpose(1, 2).contiguous()               # [kv][G][keys]
        e = torch.exp(x - x.amax(-1, keepdim=True))
        out[i] = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    return {"out": out.view(c["n_seq"], -1)}


def exact(case, seed):
    if case["kind"] == "plan":
        return None                  # whole numbers only
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "attend":
        return _exact_attend(s)
    # the nearest binary16 value of every row's, by its neighbours' distance: 11 significant bits, 2^-24 apart below 2^-14
    def rounded(x):
        x = x.double()
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14))) - 10.0)
        return torch.round(x / step) * step

    out = {}
    n = s.n_pages * case["page"]
    ok = s.slots >= 0
    for name, rows in (("k", s.k), ("v", s.v)):
        pool = torch.zeros((n, rows.shape[1]), dtype=torch.float64, device="cuda")
        pool[s.slots[ok].long()] = rounded(rows[ok])
        out[name] = pool.view(s.n_pages, case["page"], -1)
    return out
