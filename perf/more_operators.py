"""Operators of a batched step that verifies trees of drafted tokens and shares pages between sequences, beside those of perf/operators.py:

  tree     trees of drafted tokens: every row's ancestors and position before the step, the accepted path after it
  attend   attention of every token of the trees over the pages of its sequence: the committed positions and the token's ancestors
  compact  the K and V rows of an accepted path, moved to the positions they are accepted at, in every layer
  fork     sequences that come to share the pages of others, the pages that are not full copied in every layer, and an end of them
  logits   penalties for repeated tokens, biases and grammar masks, ahead of sampling

With `own` false, `run` computes them from elementary torch operations; with it true, it calls the C ABI of liblg_hip.so
(include/lg_hip.h) as a program bound to it by FFI does.  Head layouts, windows, layers, cache lengths and vocabularies are those of
little-gemma_amd/synth.py: the E4B shape (8 query and 2 key heads of 256, window 512, 42 layers, 262144 tokens), the 12B shape
(16 and 8 heads of 256, window 1024, 48 layers) and the tiny ones (8 and 2 heads of 64, 8192 tokens).
"""
import ctypes as C
import math

import numpy as np
import torch

own = False


# ---- the cases ----------------------------------------------------------------------------------------------------
def listed():
    return [
        # one conversation with a small tree: the bookkeeping around one verify step
        dict(name="tree 1", kind="tree", n_seq=1, nodes=8, chain=False),
        # a full server with the largest trees
        dict(name="tree 256", kind="tree", n_seq=256, nodes=64, chain=False),
        # the smallest call: a chain of four drafts for one short conversation of the tiny model
        dict(name="attend tiny chain", kind="attend", n_seq=1, nodes=5, chain=True, heads=8, kv=2, hd=64, page=16, ctx=100, window=0, ragged=False, scaled=False),
        # a sliding layer of the E4B shape, 64 conversations of all lengths, trees of up to 16
        dict(name="attend e4b window", kind="attend", n_seq=64, nodes=16, chain=False, heads=8, kv=2, hd=256, page=16, ctx=4096, window=512, ragged=True, scaled=False),
        # a global layer of it, 24 conversations with the largest trees: products count here
        dict(name="attend e4b global", kind="attend", n_seq=24, nodes=64, chain=False, heads=8, kv=2, hd=256, page=32, ctx=8192, window=0, ragged=True, scaled=False),
        # one long document, 12B heads
        dict(name="attend 12b long", kind="attend", n_seq=1, nodes=16, chain=False, heads=16, kv=8, hd=256, page=64, ctx=100003, window=0, ragged=False, scaled=False),
        # one conversation of the E4B shape after a verify step
        dict(name="compact 1", kind="compact", n_seq=1, nodes=16, kv=2, hd=256, layers=42, page=16, ctx=777),
        # a server of the 12B shape
        dict(name="compact 64", kind="compact", n_seq=64, nodes=32, kv=8, hd=256, layers=48, page=32, ctx=300),
        # eight answers to one prompt
        dict(name="fork 8", kind="fork", n_src=1, n_fork=8, page=64, ctx=1000, back=0, kv=2, hd=256, layers=42),
        # three more answers for each of 61 conversations, some from a few tokens back
        dict(name="fork 61 by 4", kind="fork", n_src=61, n_fork=183, page=32, ctx=333, back=20, kv=8, hd=256, layers=48),
        # chat: one row, a page of history, no grammar
        dict(name="logits chat", kind="logits", n_seq=1, nodes=0, vocab=262144, hist=3001, mode="penalties"),
        # the rows of four trees, longer histories, biases, a grammar on some rows
        dict(name="logits trees", kind="logits", n_seq=4, nodes=16, vocab=262144, hist=8192, mode="all"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((8, 2, 64), (8, 2, 128), (8, 2, 256), (16, 8, 256), (8, 1, 512), (8, 8, 128), (5, 1, 64), (12, 4, 256))


def draw(rng):
    kind = rng.choices(("tree", "attend", "compact", "fork", "logits"), (2, 6, 2, 3, 3))[0]
    page = rng.choice((16, 32, 64, 128, 256))
    if kind == "tree":
        return dict(kind=kind, n_seq=_log_uniform(rng, 1, 256), nodes=_log_uniform(rng, 1, 64), chain=rng.random() < 0.2)
    if kind == "attend":
        heads, kv, hd = rng.choice(HEADS)
        window = 0 if rng.random() < 0.5 else rng.choice((128, 512, 1024, 333))
        ctx, nodes = _log_uniform(rng, 1, 60000), _log_uniform(rng, 1, 64)
        keys = min(100003 * 8 * 256 // (kv * hd), 24 * 8192 * 8 * 256 * 64 // 3 // (heads * hd * nodes))      # of the listed cases
        n_seq = _log_uniform(rng, 1, max(1, min(128, keys // ctx)))
        return dict(kind=kind, n_seq=n_seq, nodes=nodes, chain=rng.random() < 0.2, heads=heads, kv=kv, hd=hd, page=page, ctx=ctx, window=window,
                    ragged=rng.random() < 0.6, scaled=rng.random() < 0.3)
    if kind == "compact":
        kv, hd = rng.choice(((2, 64), (2, 128), (2, 256), (8, 256), (1, 512), (4, 128)))
        layers = rng.choice((1, 6, 42, 48))
        n_seq = _log_uniform(rng, 1, 64)
        return dict(kind=kind, n_seq=n_seq, nodes=_log_uniform(rng, 2, 64), kv=kv, hd=hd, layers=layers, page=min(page, 64), ctx=_log_uniform(rng, 1, 300))
    if kind == "fork":
        kv, hd = rng.choice(((2, 64), (2, 128), (2, 256), (8, 256), (1, 512), (4, 128)))
        n_src = _log_uniform(rng, 1, 61)
        return dict(kind=kind, n_src=n_src, n_fork=_log_uniform(rng, 1, 3 * n_src), page=min(page, 64), ctx=_log_uniform(rng, 17, 333 if n_src > 8 else 2000),
                    back=rng.choice((0, 1, 20)), kv=kv, hd=hd, layers=rng.choice((1, 6, 42)))
    vocab = rng.choice((8192, 262144, _log_uniform(rng, 300, 262144)))
    nodes = 0 if rng.random() < 0.5 else _log_uniform(rng, 1, 64)
    n_seq = _log_uniform(rng, 1, max(1, 64 // max(nodes, 1)))
    return dict(kind=kind, n_seq=n_seq, nodes=nodes, vocab=vocab, hist=_log_uniform(rng, 1, 32768), mode=rng.choice(("penalties", "grammar", "all")))


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


def _pages(n, page):
    return -(-n // page)


def _sizes(n, nodes):
    """Rows of each tree: one is the largest, the others have at least half as many."""
    return nodes - np.arange(n) * 5 % (nodes // 2 + 1)


def _parents(rng, sizes, chain):
    """Trees in breadth: node 0 is the token chosen last, the others hang on earlier ones, likelier on the first children.  [rows], -1 for roots."""
    out = []
    for n in sizes:
        j = np.arange(n)
        out.append(j - 1 if chain else np.where(j > 0, np.floor((j - 1) / 2.5 * rng.uniform(0.3, 1.0, n)), -1).astype(np.int64))
    return np.concatenate(out) if out else np.zeros(0, np.int64)


def _starts(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)


def _ancestors(start, parent):
    """(sets as 64 bits, depths) of every row."""
    mask, depth = np.zeros(parent.size, np.uint64), np.zeros(parent.size, np.int64)
    for a, b in zip(start[:-1], start[1:]):
        for j in range(b - a):
            p = parent[a + j]
            if j:
                mask[a + j], depth[a + j] = mask[a + p], depth[a + p] + 1
            mask[a + j] |= np.uint64(1) << np.uint64(j)
    return mask, depth


def _bits(mask):
    return torch.from_numpy(mask.view(np.int64).copy()).cuda()


def _table(rng, held, blocks, spare=0):
    """(table, free ids, number of pages): distinct random pages for what is held."""
    n_pages = int(held.sum()) + 3 + spare
    ids = rng.permutation(n_pages)
    table = np.full((len(held), blocks), -1, np.int32)
    cols = np.arange(blocks)[None, :]
    inside = cols < held[:, None]
    table[inside] = ids[((np.cumsum(held) - held)[:, None] + cols)[inside]]
    return table, ids[int(held.sum()):], n_pages


def _prepare_tree(s, c, rng):
    sizes = _sizes(c["n_seq"], c["nodes"])
    start = _starts(sizes)
    s.rows = int(start[-1])
    parent = _parents(rng, sizes, c["chain"])
    token = rng.integers(0, 262144, s.rows)
    after = rng.integers(0, 262144, s.rows)
    for a, b in zip(start[:-1], start[1:]):                             # two thirds of the picked tokens are one of the drafts behind the row
        for j in range(1, b - a):
            if rng.random() < 0.67:
                after[a + parent[a + j]] = token[a + j]
    s.start, s.parent, s.token, s.next = _i32(start), _i32(parent), _i32(token), _i32(after)
    s.lens = _i32(rng.integers(0, 8192, c["n_seq"]) + sizes)            # with the trees' rows
    s.mask, s.pos, s.seq, s.status = _bits(np.zeros(s.rows, np.uint64)), _i32(np.zeros(s.rows)), _i32(np.zeros(s.rows)), _i32(np.zeros(c["n_seq"]))
    s.path, s.count, s.len_out, s.last = _i32(np.zeros((c["n_seq"], c["nodes"]))), _i32(np.zeros(c["n_seq"])), _i32(np.zeros(c["n_seq"])), _i32(np.zeros(c["n_seq"]))


def _lengths(c):
    return _quantiles(c["n_seq"], c["ctx"], c["ragged"])


def _prepare_attend(s, c, rng, gen):
    n, P, hd, kv, H = c["n_seq"], c["page"], c["hd"], c["kv"], c["heads"]
    at = rng.permutation(n)
    committed, sizes = _lengths(c)[at], _sizes(n, c["nodes"])[at]
    start = _starts(sizes)
    s.rows = int(start[-1])
    parent = _parents(rng, sizes, c["chain"])
    mask, depth = _ancestors(start, parent)
    s.parent_host, s.start_host, s.committed_host = parent, start, committed
    s.max_len = c["ctx"] + c["nodes"]
    s.blocks = _pages(s.max_len, P)
    table, _, s.n_pages = _table(rng, _pages(committed + sizes, P), s.blocks)
    s.table, s.lens, s.start, s.mask = _i32(table), _i32(committed + sizes), _i32(start), _bits(mask)
    s.pos = _i32(np.repeat(committed, sizes) + depth)
    s.kpool, s.vpool = (torch.randn((s.n_pages, P, kv * hd), generator=gen, device="cuda", dtype=torch.float16) for _ in range(2))
    # scores of a spread of 2, where attention picks some keys and averages over many; queries are parts of rows as a fused q/k/v product leaves them
    s.scale = hd ** -0.5 if c["scaled"] else 1.0
    s.x = torch.randn((s.rows, (H + 2 * kv) * hd), generator=gen, device="cuda")
    s.x *= 2.0 if c["scaled"] else 2.0 * hd ** -0.5
    s.q = s.x[:, :H * hd]
    s.out = torch.zeros((s.rows, H * hd), device="cuda")


def _counts(c):
    """How many rows of each tree are accepted."""
    return 1 + (np.arange(c["n_seq"]) * 7 + 3) % max(1, min(8, c["nodes"] // 2))


def _prepare_compact(s, c, rng, gen):
    n, P, T = c["n_seq"], c["page"], c["nodes"]
    committed, sizes, counts = _quantiles(n, c["ctx"], True), np.full(n, T), _counts(c)
    s.blocks = _pages(c["ctx"] + T, P)
    table, _, s.n_pages = _table(rng, _pages(committed + sizes, P), s.blocks)
    path = np.full((n, T), -1, np.int64)
    for i, m in enumerate(counts):
        path[i, 0] = 0
        path[i, 1:m] = np.sort(rng.choice(np.arange(m, T), m - 1, replace=False)) if m > 1 else []
    s.table, s.lens, s.start, s.path, s.count = _i32(table), _i32(committed + sizes), _i32(_starts(sizes)), _i32(path), _i32(counts)
    s.pools = torch.randn((c["layers"], 2, s.n_pages, P, c["kv"] * c["hd"]), generator=gen, device="cuda", dtype=torch.float16)


def _fork_lengths(c):
    """(lengths of the sources, source of each fork, its length)."""
    lens = _quantiles(c["n_src"], c["ctx"], c["n_src"] > 1)
    of = np.arange(c["n_fork"]) % c["n_src"]
    return lens, of, np.maximum(0, lens[of] - np.arange(c["n_fork"]) * 3 % (c["back"] + 1))


def _prepare_fork(s, c, rng, gen):
    lens, of, ends = _fork_lengths(c)
    a, b, P = c["n_src"], c["n_fork"], c["page"]
    s.n, s.blocks = a + b, _pages(c["ctx"], P) + 1
    held = np.concatenate([_pages(lens, P), np.zeros(b, np.int64)])
    table, free, s.n_pages = _table(rng, held, s.blocks, b)
    stack = np.zeros(s.n_pages, np.int32)
    stack[:free.size] = free
    s.table, s.stack, s.n_free, s.shares = _i32(table), _i32(stack), _i32([free.size]), _i32(np.zeros(s.n_pages))
    me = np.arange(a)
    s.len_a, s.len_b = _i32(np.concatenate([lens, np.zeros(b)])), _i32(np.concatenate([lens, ends]))
    s.src, s.gone = _i32(np.concatenate([me, of])), _i32(np.concatenate([me, np.full(b, -1)]))
    s.copy_from, s.copy_to, s.copy_rows, s.status = (_i32(np.zeros(k)) for k in (s.n, s.n, s.n, 1))
    s.back_from, s.back_to, s.back_rows, s.back_status = (_i32(np.zeros(k)) for k in (s.n, s.n, s.n, 1))
    s.pools = torch.randn((c["layers"], 2, s.n_pages, P, c["kv"] * c["hd"]), generator=gen, device="cuda", dtype=torch.float16)


PENALTIES = ((1.1, 0.0, 0.0), (1.0, 0.5, 0.25), (1.3, 0.1, 0.05), (1.0, 0.0, 0.0))      # repetition, presence, frequency


def _masked(c):
    """Rows that a grammar holds."""
    rows = c["n_seq"] * max(c["nodes"], 1)
    return np.zeros(rows, bool) if c["mode"] == "penalties" else np.arange(rows) % (1 if c["mode"] == "grammar" else 3) == 0


def _history(c):
    return np.maximum(1, _quantiles(c["n_seq"], c["hist"], c["n_seq"] > 1))


def _prepare_logits(s, c, rng, gen):
    n, V, T = c["n_seq"], c["vocab"], c["nodes"]
    s.rows = n * max(T, 1)
    s.logits = 30.0 * torch.tanh(torch.randn((s.rows, V), generator=gen, device="cuda") / 10.0)
    s.out = torch.zeros_like(s.logits)
    s.seq = _i32(np.arange(s.rows) // max(T, 1))
    # tokens of a text: few of them often, most of them never
    s.hist = torch.floor(V * torch.rand((n, c["hist"]), generator=gen, device="cuda") ** 4).to(torch.int32)
    s.hist_len = _i32(_history(c))
    s.use = c["mode"] != "grammar"
    raw = np.zeros(n, np.dtype([("r", "f4"), ("a", "f4"), ("b", "f4"), ("n", "i4")]))               # as struct lg_hip_penalty
    for i in range(n):
        raw[i] = (*PENALTIES[i % 3 if n < 4 else i % 4], _history(c)[i] // 3)
    s.penalty_host = raw
    s.penalty = torch.from_numpy(raw.view(np.uint8).copy()).cuda()
    s.rep, s.pres, s.freq = (torch.tensor(raw[k].copy(), device="cuda") for k in "rab")
    s.prompt = _i32(raw["n"])
    s.tree = T > 0
    if s.tree:
        start = _starts(np.full(n, T))
        mask, _ = _ancestors(start, _parents(rng, np.full(n, T), False))
        s.mask_host, s.mask, s.start = mask, _bits(mask), _i32(start)
        s.token = _i32(rng.integers(0, V, s.rows))
    s.bias_n = 0
    if c["mode"] == "all":
        per = min(300, V // 2)
        s.bias_n = n * per
        s.bias_start = _i32(np.arange(n + 1) * per)
        s.bias_tok = _i32(np.concatenate([rng.choice(V, per, replace=False) for _ in range(n)]))
        s.bias = torch.randn(s.bias_n, generator=gen, device="cuda") * 4.0
    s.allow_n, s.words = int(_masked(c).sum()), (V + 31) // 32
    if s.allow_n:
        # grammars of a state each: a thirtieth of the vocabulary
        allowed = torch.rand((s.allow_n, s.words * 32), generator=gen, device="cuda") < 1 / 30
        weights = torch.tensor([1 << b for b in range(32)], dtype=torch.int64, device="cuda")
        w = (allowed.view(s.allow_n, s.words, 32).long() * weights).sum(-1)
        s.allow = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
        s.allow_row = _i32(np.where(_masked(c), np.cumsum(_masked(c)) - 1, -1))


def prepare(case, seed):
    s, rng = _State(), np.random.default_rng(seed)
    s.case = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "tree":
        _prepare_tree(s, case, rng)
    else:
        dict(attend=_prepare_attend, compact=_prepare_compact, fork=_prepare_fork, logits=_prepare_logits)[case["kind"]](s, case, rng, gen)
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


def _pool(s, k, v):
    c = s.case
    width = c["kv"] * c["hd"]
    return _own().Pages(k.data_ptr(), v.data_ptr(), s.n_pages, c["page"], c["kv"], c["hd"], width, width * c["page"])


def _layers(s):
    n = s.case["layers"]
    return (_own().Pages * n)(*(_pool(s, s.pools[i, 0], s.pools[i, 1]) for i in range(n)))


def _rules(s):
    L = _own()
    p = (lambda t: t.data_ptr())  # noqa: E731
    r = L.LogitRules(n_seq=s.case["n_seq"], seq=p(s.seq))
    if s.use:
        r.penalty, r.hist, r.hist_len, r.hist_stride = p(s.penalty), p(s.hist), p(s.hist_len), s.hist.shape[1]
        if s.tree:
            r.tree_mask, r.tree_start, r.tree_tok = p(s.mask), p(s.start), p(s.token)
    if s.bias_n:
        r.n_bias, r.bias_start, r.bias_tok, r.bias = s.bias_n, p(s.bias_start), p(s.bias_tok), p(s.bias)
    if s.allow_n:
        r.n_allow, r.allow, r.allow_row, r.allow_stride = s.allow_n, p(s.allow), p(s.allow_row), s.words
    return r


def _bound(s, stream):
    """The calls of a pass on a stream with their arguments in place, as a serving loop keeps them: pointers, handles, working memory of the stream's own."""
    L, c, keep = _own(), s.case, []
    H, p, stream = L.load_hip(), (lambda t: C.c_void_p(t.data_ptr())), C.c_void_p(stream)

    def memory(n):
        keep.append(torch.empty(max(n, 16), dtype=torch.uint8, device="cuda"))
        return p(keep[-1]), C.c_size_t(n)

    if c["kind"] == "tree":
        shape = (c["n_seq"], c["nodes"], s.rows, p(s.start), p(s.parent))
        return [(H.lg_hip_tree_plan, (*shape, p(s.lens), p(s.mask), p(s.pos), p(s.seq), p(s.status), stream)),
                (H.lg_hip_tree_accept, (*shape, p(s.token), p(s.next), p(s.lens), p(s.path), p(s.count), p(s.len_out), p(s.last), stream))], keep
    if c["kind"] == "attend":
        w = memory(H.lg_hip_paged_tree_attention_workspace(c["n_seq"], c["nodes"], c["heads"], c["kv"], c["hd"], s.max_len, c["window"]))
        keep.append(_pool(s, s.kpool, s.vpool))
        return [(H.lg_hip_paged_tree_attention, (C.byref(keep[-1]), p(s.q), s.x.shape[1], s.rows, c["n_seq"], c["nodes"], c["heads"], p(s.table), s.blocks, p(s.lens),
                                                 p(s.start), p(s.mask), p(s.pos), s.max_len, c["window"], s.scale, p(s.out), s.out.shape[1], *w, stream))], keep
    if c["kind"] == "compact":
        keep.append(_layers(s))
        return [(H.lg_hip_paged_compact, (keep[-1], c["layers"], c["n_seq"], c["nodes"], p(s.table), s.blocks, p(s.lens), p(s.start), p(s.path), p(s.count), stream))], keep
    if c["kind"] == "fork":
        w = memory(H.lg_hip_paged_fork_workspace(s.n, s.n_pages, s.blocks))
        keep.append(_layers(s))
        shape = (s.n, c["page"], s.n_pages, s.blocks)
        pages = (p(s.table), p(s.shares), p(s.stack), p(s.n_free))
        return [(H.lg_hip_paged_fork, (*shape, p(s.src), p(s.len_a), p(s.len_b), *pages, p(s.copy_from), p(s.copy_to), p(s.copy_rows), p(s.status), *w, stream)),
                (H.lg_hip_paged_copy, (keep[-1], c["layers"], s.n, p(s.copy_from), p(s.copy_to), p(s.copy_rows), stream)),
                (H.lg_hip_paged_fork, (*shape, p(s.gone), p(s.len_b), p(s.len_a), *pages, p(s.back_from), p(s.back_to), p(s.back_rows), p(s.back_status), *w, stream))], keep
    keep.append(_rules(s))
    V = c["vocab"]
    return [(H.lg_hip_adjust_logits, (C.byref(keep[-1]), p(s.logits), V, s.rows, V, p(s.out), V, stream))], keep


def _run_own(s):
    # the stream that is current now (its handle alone: a Stream object takes microseconds)
    stream = torch._C._cuda_getCurrentRawStream(s.device)
    if stream not in s.calls:
        s.calls[stream] = _bound(s, stream)
    for f, args in s.calls[stream][0]:
        rc = f(*args)
        if rc:
            _own().hip_check(rc, s.case["kind"])


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _tree_plan(s):
    n, T = s.case["n_seq"], s.case["nodes"]
    start = s.start.long()
    r = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(start[1:], r, right=True)
    j = r - start[seq]
    # reach[i][j][k]: node k is j or above it; squaring doubles the steps
    step = torch.zeros((n, T, T), device="cuda")
    step[seq, j, j] = 1.0
    up = j > 0
    step[seq[up], j[up], s.parent.long()[up]] = 1.0
    for _ in range(max(1, (T - 1).bit_length())):
        step = (torch.matmul(step, step) > 0).float()
    reach = (step > 0).long()[seq, j]                                                               # [rows][T]
    s.mask.copy_((reach << torch.arange(T, device="cuda")).sum(1))                                  # distinct bits: the sum is their union
    size = start[1:] - start[:-1]
    s.pos.copy_((s.lens.long() - size)[seq] + reach.sum(1) - 1)
    s.seq.copy_(seq)
    s.status.zero_()


def _tree_accept(s):
    n, T = s.case["n_seq"], s.case["nodes"]
    start = s.start.long()
    size = (start[1:] - start[:-1])[:, None]
    col = torch.arange(T, device="cuda")[None, :]
    row = (start[:-1, None] + col).clamp(max=max(s.rows - 1, 0))
    inside = col < size
    parent, token = s.parent.long()[row], s.token.long()[row]
    at = torch.zeros((n, 1), dtype=torch.long, device="cuda")
    live = size > 0
    count, path = live.long(), torch.where(live & (col == 0), 0, -1).expand(n, T).clone()
    for k in range(1, T):
        want = s.next.long()[(start[:-1, None] + at).clamp(max=max(s.rows - 1, 0))]
        fits = inside & (col > at) & (parent == at) & (token == want) & (want >= 0)
        first = torch.where(fits, col, T).amin(1, keepdim=True)
        live = live & (first < T)
        at = torch.where(live, first, at)
        path[:, k:k + 1] = torch.where(live, at, -1)
        count = count + live.long()
    s.path.copy_(path)
    s.count.copy_(count[:, 0])
    s.len_out.copy_(s.lens.long() - size[:, 0] + count[:, 0])
    s.last.copy_(torch.where(size[:, 0] > 0, s.next.long()[(start[:-1] + at[:, 0]).clamp(max=max(s.rows - 1, 0))], -1))


def _attend(s):
    c, P, G = s.case, s.case["page"], s.case["heads"] // s.case["kv"]
    n, hd, kv, T, W = c["n_seq"], c["hd"], c["kv"], c["nodes"], c["window"]
    start = s.start.long()
    size = start[1:] - start[:-1]
    lens = s.lens.long()
    committed = lens - size
    span = (c["ctx"] if not W else min(c["ctx"], W)) + T
    t = (committed - (span - T)).clamp(min=0)[:, None] + torch.arange(span, device="cuda")[None, :]      # [n][span]
    page = torch.gather(s.table.long(), 1, (t // P).clamp(max=s.blocks - 1))
    ok = (t < lens[:, None]) & (page >= 0)
    row = torch.where(ok, page * P + t % P, 0)
    node = (t - committed[:, None]).clamp(0, T - 1)                                                 # of positions behind the committed ones
    tail = t >= committed[:, None]
    mine = start[:-1, None] + torch.arange(T, device="cuda")[None, :]                               # [n][T] rows of the trees
    real = torch.arange(T, device="cuda")[None, :] < size[:, None]
    mine = torch.where(real, mine, 0)
    # few sequences at a time where the gathered rows or the scores would take too much room
    step = max(1, (1 << 31) // (span * kv * (2 * hd + 3 * G * T)))
    for i in range(0, n, step):
        m = min(step, n - i)
        part = slice(i, i + m)
        seen = torch.where(tail[part, None, :], (s.mask[mine[part]][:, :, None] >> node[part, None, :]) & 1 > 0, True) & ok[part, None, :]
        if W:
            where = torch.where(tail[part, None, :], s.pos.long()[(start[:-1][part, None] + node[part]).clamp(max=s.rows - 1)][:, None, :], t[part, None, :])
            seen &= where > s.pos.long()[mine[part]][:, :, None] - W
        seen = seen[:, None, :, None, :].expand(m, 1, T, G, span).reshape(m, 1, T * G, span)
        r = row[part].reshape(-1)
        k = s.kpool.view(-1, kv, hd)[r].float().view(m, span, kv, hd).permute(0, 2, 3, 1).contiguous()
        q = (s.q[mine[part].reshape(-1)].reshape(m, T, kv, G, hd) * s.scale).permute(0, 2, 1, 3, 4).reshape(m, kv, T * G, hd)
        x = torch.where(seen, torch.matmul(q, k), float("-inf"))
        top = x.amax(-1, keepdim=True)
        e = torch.where(seen, torch.exp(x - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
        del k, x
        v = s.vpool.view(-1, kv, hd)[r].float().view(m, span, kv, hd).permute(0, 2, 1, 3).contiguous()
        o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        o = o.view(m, kv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(m, T, -1)
        s.out[mine[part][real[part]]] = o[real[part]]


def _move(pools, P, src, dst):
    """Rows `src` of every layer to `dst` (slots): everything is read, then everything is written."""
    n = pools.shape[2] * P
    flat = pools.view(pools.shape[0], 2, n, -1)
    flat[:, :, dst] = flat[:, :, src]


def _compact(s):
    P, T = s.case["page"], s.case["nodes"]
    base = s.lens.long() - (s.start[1:] - s.start[:-1]).long()
    k = torch.arange(T, device="cuda")[None, :]
    path = s.path.long()
    moves = (k < s.count.long()[:, None]) & (path > k)

    def slots(pos):
        return torch.gather(s.table.long(), 1, (pos // P).clamp(0, s.blocks - 1)) * P + pos % P

    _move(s.pools, P, slots(base[:, None] + path.clamp(min=0))[moves], slots(base[:, None] + k)[moves])


def _fork(s, src, len_old, len_new, copy_from, copy_to, copy_rows, status):
    n, P, B, N = s.n, s.case["page"], s.blocks, s.n_pages
    i, col = torch.arange(n, device="cuda"), torch.arange(B, device="cuda")[None, :]
    src, a, b, old = src.long(), len_old.long(), len_new.long(), s.table.long()
    na, nb = (a + P - 1) // P, (b + P - 1) // P
    moved = src != i
    take = old[src.clamp(min=0)]
    leave = (col >= torch.where(moved, 0, nb)[:, None]) & (col < na[:, None])
    come = moved[:, None] & (col < nb[:, None])

    def tally(where, ids, value=1):
        return torch.zeros(N + 1, dtype=torch.long, device="cuda").scatter_add(0, torch.where(where, ids, N).reshape(-1), torch.full((ids.numel(),), value, device="cuda"))

    def lowest(where, ids, keys):
        return torch.full((N + 1,), 1 << 60, device="cuda").scatter_reduce(0, torch.where(where, ids, N).reshape(-1), keys.reshape(-1), "amin")

    holders = torch.cat([s.shares.long() + 1, torch.zeros(1, dtype=torch.long, device="cuda")]) + tally(come, take) + tally(leave, old, -1)
    # pages that nobody holds any longer go on the stack, the first one topmost
    order = torch.arange(n * B, device="cuda").view(n, B)
    at = torch.where(leave, old, N)
    push = leave & (holders[at] == 0) & (lowest(leave, old, order)[at] == order)
    k = push.reshape(-1).cumsum(0).view(n, B)
    top = s.n_free.long() + k[-1, -1]
    stack = torch.cat([s.stack.long(), torch.zeros(1, dtype=torch.long, device="cuda")])
    stack = stack.scatter(0, torch.where(push, top - k, N).reshape(-1), old.reshape(-1))
    # a last page that is not full is its row's own: one row keeps it where no other holds more of it, the others copy
    part = b % P > 0
    last = torch.where(part, torch.gather(take, 1, (b // P).clamp(max=B - 1)[:, None])[:, 0], N)
    key = moved.long() * n + i
    keeps = (tally(part, last)[last] == holders[last]) & (lowest(part, last, key)[last] == key)
    copies = part & ~keeps
    m = copies.long().cumsum(0)
    fresh = stack[(top - m).clamp(0, N - 1)]
    s.shares.copy_((holders - 1 - tally(copies, last))[:N].clamp(min=0))
    table = torch.where(col < nb[:, None], take, torch.where(col < na[:, None], -1, old))
    table = torch.where(copies[:, None] & (col == (b // P)[:, None]), fresh[:, None], table)
    s.table.copy_(table)
    s.stack.copy_(stack[:N])
    s.n_free.copy_(top - m[-1:])
    copy_from.copy_(torch.where(copies, last, -1))
    copy_to.copy_(torch.where(copies, fresh, -1))
    copy_rows.copy_(torch.where(copies, b % P, 0))
    status.zero_()


def _copy(s):
    P = s.case["page"]
    k = torch.arange(P, device="cuda")[None, :]
    rows = (k < s.copy_rows[:, None]) & (s.copy_to >= 0)[:, None]
    _move(s.pools, P, (s.copy_from.long()[:, None] * P + k)[rows], (s.copy_to.long()[:, None] * P + k)[rows])


def _logits(s):
    c, V, n = s.case, s.case["vocab"], s.case["n_seq"]
    l = s.logits
    seq = s.seq.long()
    if s.use:
        place, ones = torch.arange(c["hist"], device="cuda")[None, :], torch.ones((n, c["hist"]), device="cuda")
        seen = place < s.hist_len[:, None]
        made = seen & (place >= s.prompt[:, None])
        base = torch.zeros((n, V), device="cuda")
        any_ = base.scatter_add(1, s.hist.long(), ones * seen)[seq]
        count = base.scatter_add(1, s.hist.long(), ones * made)[seq]
        if s.tree:
            T = c["nodes"]
            on = ((s.mask[:, None] >> torch.arange(T, device="cuda")[None, :]) & 1).float()
            toks = s.token.long().view(n, T)[seq]
            any_, count = any_.scatter_add(1, toks, on), count.scatter_add(1, toks, on)
        rep = s.rep[seq][:, None]
        l = torch.where(any_ > 0, torch.where(l > 0, l / rep, l * rep), l)
        l = torch.where(count > 0, l - s.pres[seq][:, None] - s.freq[seq][:, None] * count, l)
    if s.bias_n:
        b = torch.zeros((n, V), device="cuda").scatter(1, s.bias_tok.long().view(n, -1), s.bias.view(n, -1))
        l = l + b[seq]
    if s.allow_n:
        tok = torch.arange(V, device="cuda")
        bit = (s.allow[:, tok // 32] >> (tok % 32)[None, :]) & 1
        row = s.allow_row.long()
        l = torch.where((row >= 0)[:, None] & (bit[row.clamp(min=0)] == 0), float("-inf"), l)
    s.out.copy_(l)


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(s):
    kind = s.case["kind"]
    if own:
        _run_own(s)
    elif kind == "tree":
        _tree_plan(s)
        _tree_accept(s)
    elif kind == "attend":
        _attend(s)
    elif kind == "compact":
        _compact(s)
    elif kind == "fork":
        _fork(s, s.src, s.len_a, s.len_b, s.copy_from, s.copy_to, s.copy_rows, s.status)
        _copy(s)
        _fork(s, s.gone, s.len_b, s.len_a, s.back_from, s.back_to, s.back_rows, s.back_status)
    else:
        _logits(s)
    if kind == "tree":
        return {"mask": s.mask, "pos": s.pos, "seq": s.seq, "status": s.status, "path": s.path, "count": s.count, "len": s.len_out, "token": s.last}
    if kind == "attend":
        return {"out": s.out}
    if kind == "compact":
        return {"pages": s.pools}
    if kind == "fork":               # the forks have ended again: the pages are as before, but for the copies
        return {"from": s.copy_from, "to": s.copy_to, "rows": s.copy_rows, "status": s.status, "pages": s.pools, "table": s.table, "shares": s.shares,
                "stack": s.stack, "free": s.n_free, "back_from": s.back_from, "back_to": s.back_to, "back_rows": s.back_rows, "back_status": s.back_status}
    return {"logits": s.out}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "tree":
        rows, n = float(_sizes(c["n_seq"], c["nodes"]).sum()), c["n_seq"]
        # parents twice, ancestors, positions, sequences; tokens, picked tokens; starts and lengths twice; status, paths, counts, lengths, tokens
        return {"bytes": rows * (8 + 8 + 4 + 4 + 8) + n * (2 * 8 + 4 + 4 * c["nodes"] + 12.0), "flops": 0.0}
    if c["kind"] == "attend":
        committed, sizes = _lengths(c), _sizes(c["n_seq"], c["nodes"])
        keys = np.minimum(committed, c["window"] - 1) if c["window"] else committed
        rows = 2 * 4 * int(sizes.sum()) * c["heads"] * c["hd"]
        total = int((keys + sizes).sum())
        return {"bytes": float(4 * total * c["kv"] * c["hd"] + rows + 4 * total / c["page"] + 12 * sizes.sum()),
                "flops": 4.0 * c["heads"] * c["hd"] * float((sizes * (keys + 1)).sum())}
    if c["kind"] == "compact":
        return {"bytes": float((_counts(c) - 1).sum()) * 2 * 4 * c["kv"] * c["hd"] * c["layers"] + 4.0 * c["n_seq"] * (c["nodes"] + 4), "flops": 0.0}
    if c["kind"] == "fork":
        _, _, ends = _fork_lengths(c)
        held = int(_pages(ends, c["page"]).sum())
        # rows copied; per page that is shared and given back its entry of either table row and its count twice
        return {"bytes": float((ends % c["page"]).sum()) * 2 * 4 * c["kv"] * c["hd"] * c["layers"] + 2 * held * (8 + 8.0), "flops": 0.0}
    rows, V = c["n_seq"] * max(c["nodes"], 1), c["vocab"]
    b = 8.0 * rows * V + float(_masked(c).sum()) * V / 8
    return {"bytes": b + (4.0 * float(_history(c).sum()) if c["mode"] != "grammar" else 0.0), "flops": 0.0}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_attend(s):
    """Sequence by sequence over its keys alone, what a row sees found by walking up from it."""
    c, P, G, W = s.case, s.case["page"], s.case["heads"] // s.case["kv"], s.case["window"]
    kv, hd = c["kv"], c["hd"]
    table = s.table.cpu().numpy()
    out = torch.zeros((s.rows, c["heads"] * hd), dtype=torch.float64, device="cuda")
    for i, done in enumerate(int(x) for x in s.committed_host):
        a, b = int(s.start_host[i]), int(s.start_host[i + 1])
        n, parent = b - a, s.parent_host[a:b]
        lo = max(0, done - W) // P * P if W else 0
        ids = torch.from_numpy(table[i, lo // P:_pages(done + n, P)].astype(np.int64)).cuda()
        k, v = (pool[ids].reshape(-1, kv, hd)[:done + n - lo].double().transpose(0, 1).contiguous() for pool in (s.kpool, s.vpool))
        seen = np.zeros((n, done + n - lo), bool)
        for j in range(n):
            chain = [j]
            while chain[-1] > 0:
                chain.append(int(parent[chain[-1]]))
            pos = done + len(chain) - 1
            seen[j, max(lo, pos - W + 1 if W else 0) - lo:done - lo] = True
            for up, node in enumerate(chain):
                seen[j, done - lo + node] = not W or up < W
        ok = torch.from_numpy(seen).cuda()[None, :, None, :]
        q = s.q[a:b].double().view(n, kv, G, hd).permute(1, 0, 2, 3).contiguous() * s.scale
        x = torch.matmul(q.reshape(kv, n * G, hd), k.transpose(1, 2).contiguous()).view(kv, n, G, -1)
        x = torch.where(ok, x, -math.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(e.view(kv, n * G, -1), v) / e.sum(-1).view(kv, n * G, 1)
        out[a:b] = o.view(kv, n, G, hd).permute(1, 0, 2, 3).reshape(n, -1)
    return {"out": out}


def _exact_logits(s):
    """Row by row: the tokens of a row's text, each with its count."""
    c = s.case
    out = s.logits.double()
    for r in range(s.rows):
        i = int(s.seq[r])
        if s.use:
            rep, pres, freq, prompt = (x.item() for x in s.penalty_host[i])
            text = s.hist[i, :int(s.hist_len[i])].long()
            new = text[prompt:]
            if s.tree:
                bits = [k for k in range(c["nodes"]) if int(s.mask_host[r]) >> k & 1]
                drafted = s.token.long()[int(s.start[i]):][bits]
                text, new = torch.cat([text, drafted]), torch.cat([new, drafted])
            ids = torch.unique(text)
            x = out[r, ids]
            out[r, ids] = torch.where(x > 0, x / rep, x * rep)
            ids, count = torch.unique(new, return_counts=True)
            out[r, ids] -= pres + freq * count.double()
        if s.bias_n:
            part = slice(int(s.bias_start[i]), int(s.bias_start[i + 1]))
            out[r, s.bias_tok[part].long()] += s.bias[part].double()
        if s.allow_n and int(s.allow_row[r]) >= 0:
            words = s.allow[int(s.allow_row[r])].cpu().numpy().view(np.uint8)
            allowed = np.unpackbits(words, bitorder="little")[:c["vocab"]].astype(bool)
            out[r, torch.from_numpy(~allowed).cuda()] = -math.inf
    return {"logits": out}


def exact(case, seed):
    if case["kind"] in ("tree", "compact", "fork"):
        return None                  # whole numbers, and rows that are moved as they are
    s = prepare(case, seed)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_logits(s)
