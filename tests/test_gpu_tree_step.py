"""A server that verifies trees of drafted tokens, over many steps: pages, ancestors, rows, attention, rules, draws, accepted paths, rows moved, pages back, and conversations that fork and end; the same
recorded into a graph; and servers on streams of their own.  Everything against the plain forms."""
import ctypes as C

import numpy as np
import pytest

from drafts import accept_ref, compact_ref, fork_ref, penalties, random_parents, rules_ref, starts_of, tree_attend_ref, tree_plan_ref
from serving import Device, plan_ref, sample_ref, within

pytestmark = pytest.mark.gpu
H, KV, HD, PAGE, BLOCKS, N_PAGES, SEQS, VOCAB, MOST, LAYERS, TEXT = 8, 2, 64, 16, 16, 130, 6, 700, 9, 3, 64
WIDTH, MAX_LEN, ROWS = KV * HD, BLOCKS * PAGE, SEQS * MOST
PENALTY = [(1.2, 0.0, 0.0, 2), (1.0, 0.5, 0.25, 0), (1.0, 0.0, 0.0, 0), (1.3, 0.1, 0.0, 5), (0.9, 0.0, 0.5, 1), (1.1, 0.2, 0.1, 0)]


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


class Server:
    """A pool of several layers, its bookkeeping and one step's buffers on the device, with the plain forms' state beside them."""

    def __init__(self, lg, dev, window=0):
        self.lg, self.dev, self.H, self.window = lg, dev, dev.H, window
        self.pools = np.zeros((LAYERS, 2, N_PAGES, PAGE, WIDTH), np.uint16)
        self.table, self.stack, self.n_free = np.full((SEQS, BLOCKS), -1, np.int32), np.arange(N_PAGES, dtype=np.int32), N_PAGES
        self.shares, self.lens, self.texts = np.zeros(N_PAGES, np.int32), [0] * SEQS, [[] for _ in range(SEQS)]
        i32 = (lambda *s: np.zeros(s, np.int32))  # noqa: E731
        self.d = {n: dev.up(a) for n, a in dict(
            pool=self.pools, table=self.table, stack=self.stack, free=np.array([N_PAGES], np.int32), shares=self.shares, old=i32(SEQS), new=i32(SEQS), start=i32(SEQS + 1), slot=i32(ROWS),
            status=i32(1), start2=i32(SEQS + 1), slot2=i32(1), parent=i32(ROWS), token=i32(ROWS), mask=np.zeros(ROWS, np.uint64), pos=i32(ROWS), seq=i32(ROWS), bad=i32(SEQS),
            x=np.zeros((LAYERS, ROWS, 2 * WIDTH), np.float32), q=np.zeros((ROWS, H * HD), np.float32), out=np.zeros((ROWS, H * HD), np.float32), logits=np.zeros((ROWS, VOCAB), np.float32),
            held=np.zeros((ROWS, VOCAB), np.float32), text=i32(SEQS, TEXT), text_len=i32(SEQS), u=np.zeros(ROWS, np.float32), next=i32(ROWS), path=i32(SEQS, MOST), count=i32(SEQS), len=i32(SEQS),
            last=i32(SEQS), src=i32(SEQS), src_old=i32(SEQS), src_new=i32(SEQS), frm=i32(SEQS), to=i32(SEQS), rows=i32(SEQS), fork_status=i32(1)).items()}
        self.d["penalty"] = dev.up(penalties(PENALTY).view(np.uint8))
        how = np.zeros(ROWS, np.dtype([("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")]))
        how[:] = (0.0, 0, 1.0, 0.0)                                    # the likeliest: tokens without numbers of their own
        self.d["how"] = dev.up(how.view(np.uint8))
        self.need = [self.H.lg_hip_paged_plan_workspace(SEQS), self.H.lg_hip_paged_tree_attention_workspace(SEQS, MOST, H, KV, HD, MAX_LEN, window), self.H.lg_hip_sample_workspace(ROWS, VOCAB),
                     self.H.lg_hip_paged_fork_workspace(SEQS, N_PAGES, BLOCKS)]
        self.work = [dev.room(n) for n in self.need]
        step, base = N_PAGES * PAGE * WIDTH * 2, self.d["pool"].value
        self.layers = (lg.hiplib.Pages * LAYERS)(*(lg.hiplib.Pages(base + 2 * i * step, base + (2 * i + 1) * step, N_PAGES, PAGE, KV, HD, WIDTH, WIDTH * PAGE) for i in range(LAYERS)))
        d = self.d
        self.rules = lg.hiplib.LogitRules(n_seq=SEQS, seq=d["seq"].value, penalty=d["penalty"].value, hist=d["text"].value, hist_len=d["text_len"].value, hist_stride=TEXT, tree_mask=d["mask"].value,
                                          tree_start=d["start"].value, tree_tok=d["token"].value)

    # ---- the calls
    def verify(self, stream=None):
        d, H_, check = self.d, self.H, self.dev.check
        check(H_.lg_hip_paged_plan(SEQS, PAGE, N_PAGES, BLOCKS, d["old"], d["new"], d["table"], d["stack"], d["free"], d["start"], d["slot"], ROWS, d["status"], self.work[0], self.need[0], stream), "plan")
        check(H_.lg_hip_tree_plan(SEQS, MOST, ROWS, d["start"], d["parent"], d["new"], d["mask"], d["pos"], d["seq"], d["bad"], stream), "tree_plan")
        for i in range(LAYERS):
            x = d["x"].value + i * ROWS * 2 * WIDTH * 4
            check(H_.lg_hip_paged_write(C.byref(self.layers[i]), C.c_void_p(x), C.c_void_p(x + 4 * WIDTH), 2 * WIDTH, d["slot"], ROWS, stream), "write")
        check(H_.lg_hip_paged_tree_attention(C.byref(self.layers[1]), d["q"], H * HD, ROWS, SEQS, MOST, H, d["table"], BLOCKS, d["new"], d["start"], d["mask"], d["pos"], MAX_LEN, self.window, 1.0, d["out"],
                                             H * HD, self.work[1], self.need[1], stream), "attention")
        check(H_.lg_hip_adjust_logits(C.byref(self.rules), d["logits"], VOCAB, ROWS, VOCAB, d["held"], VOCAB, stream), "rules")
        check(H_.lg_hip_sample(d["held"], VOCAB, ROWS, VOCAB, d["how"], d["u"], d["next"], None, None, self.work[2], self.need[2], stream), "sample")
        check(H_.lg_hip_tree_accept(SEQS, MOST, ROWS, d["start"], d["parent"], d["token"], d["next"], d["new"], d["path"], d["count"], d["len"], d["last"], stream), "accept")
        check(H_.lg_hip_paged_compact(self.layers, LAYERS, SEQS, MOST, d["table"], BLOCKS, d["new"], d["start"], d["path"], d["count"], stream), "compact")
        check(H_.lg_hip_paged_plan(SEQS, PAGE, N_PAGES, BLOCKS, d["new"], d["len"], d["table"], d["stack"], d["free"], d["start2"], None, 0, d["status"], self.work[0], self.need[0], stream), "plan back")

    def fork(self, stream=None):
        d, H_, check = self.d, self.H, self.dev.check
        check(H_.lg_hip_paged_fork(SEQS, PAGE, N_PAGES, BLOCKS, d["src"], d["src_old"], d["src_new"], d["table"], d["shares"], d["stack"], d["free"], d["frm"], d["to"], d["rows"], d["fork_status"],
                                   self.work[3], self.need[3], stream), "fork")
        check(H_.lg_hip_paged_copy(self.layers, LAYERS, SEQS, d["frm"], d["to"], d["rows"], stream), "copy")

    # ---- a step's inputs, and what it has to give
    def inputs(self, rng):
        sizes = np.array([int(rng.integers(1, MOST + 1)) if n + MOST + 3 < MAX_LEN else 0 for n in self.lens])
        start = starts_of(sizes)
        rows = int(start[-1])
        s = dict(start=start, sizes=sizes, old=np.array(self.lens), new=np.array(self.lens) + sizes, parent=np.zeros(ROWS, np.int64), token=rng.integers(0, VOCAB, ROWS))
        s["parent"][:rows] = np.concatenate([random_parents(rng, int(n), ("any", "chain")[int(rng.integers(2))]) for n in sizes if n] + [np.zeros(0, np.int64)])
        s["x"] = rng.normal(0, 1, (LAYERS, ROWS, 2 * WIDTH)).astype(np.float32)
        s["q"] = (rng.normal(0, 2, (ROWS, H * HD)) / 8).astype(np.float32)
        s["logits"] = rng.normal(0, 2, (ROWS, VOCAB)).astype(np.float32)
        for a in range(rows):                                          # two thirds of the rows are followed by a draft that hangs on them
            i = int(np.searchsorted(start[1:], a, side="right"))
            kids = [j for j in range(1, sizes[i]) if s["parent"][start[i] + j] == a - start[i]]
            if kids and rng.random() < 0.67:
                s["logits"][a, s["token"][start[i] + kids[int(rng.integers(len(kids)))]]] += 40
        text = np.zeros((SEQS, TEXT), np.int32)
        for i, t in enumerate(self.texts):
            text[i, :len(t[-TEXT:])] = t[-TEXT:]
        s["text"], s["text_len"] = text, np.array([min(len(t), TEXT) for t in self.texts])
        for n, t in (("old", np.int32), ("new", np.int32), ("parent", np.int32), ("token", np.int32), ("x", np.float32), ("q", np.float32), ("logits", np.float32), ("text", np.int32), ("text_len", np.int32)):
            self.dev.put(self.d[n], np.asarray(s[n], t))
        return s

    def plain(self, s):
        rows = int(s["start"][-1])
        start, slot, status, self.table, self.stack, self.n_free = plan_ref(PAGE, s["old"].tolist(), s["new"].tolist(), self.table, self.stack, self.n_free, ROWS)
        assert status == 0 and np.array_equal(start, s["start"])
        for r, at in enumerate(slot.tolist()):
            if at >= 0:
                for layer in range(LAYERS):
                    for which in range(2):
                        self.pools[layer, which, at // PAGE, at % PAGE] = s["x"][layer, r, which * WIDTH:(which + 1) * WIDTH].astype(np.float16).view(np.uint16)
        w = dict(start=start, slot=slot)
        w["mask"], w["pos"], w["seq"] = tree_plan_ref(start, s["parent"][:rows], s["new"])
        kv = self.pools[1].view(np.float16).reshape(2, N_PAGES, PAGE, KV, HD)
        w["out"] = tree_attend_ref(s["q"][:rows].reshape(rows, H, HD), kv[0], kv[1], self.table, s["new"], start, w["mask"], w["pos"], PAGE, N_PAGES, KV, self.window, 1.0, MAX_LEN)
        # (rows behind the last tree have no sequence of their own in d["seq"]: whatever is left there)
        w["held"] = rules_ref(s["logits"][:rows], w["seq"], PENALTY, s["text"], s["text_len"], (w["mask"], start, s["token"][:rows]), None, None, None)
        w["next"] = np.array([sample_ref(w["held"][r].astype(np.float32), 0.0, 0, 1.0, 0.0, 0.0)[0] for r in range(rows)])
        w["path"], w["count"], w["len"], w["last"] = accept_ref(start, s["parent"], s["token"], w["next"], s["new"], MOST)
        self.pools = compact_ref(self.pools, PAGE, N_PAGES, self.table, s["new"], start, w["path"], w["count"])
        _, _, status, self.table, self.stack, self.n_free = plan_ref(PAGE, s["new"].tolist(), w["len"].tolist(), self.table, self.stack, self.n_free, 0)
        assert status == 0
        self.lens = w["len"].tolist()
        for i in range(SEQS):
            self.texts[i] = (self.texts[i] + [int(s["token"][start[i] + k]) for k in w["path"][i, :w["count"][i]]])
        return w

    def compare(self, w, what):
        back, d, rows = self.dev.back, self.d, int(w["start"][-1])
        for n, t in (("start", np.int32), ("slot", np.int32), ("path", np.int32), ("count", np.int32), ("len", np.int32), ("last", np.int32)):
            assert np.array_equal(back(d[n], np.shape(w[n]), t), w[n]), (what, n)
        for n, t in (("mask", np.uint64), ("pos", np.int32), ("seq", np.int32), ("next", np.int32)):
            assert np.array_equal(back(d[n], rows, t), w[n]), (what, n)
        assert not back(d["bad"], SEQS, np.int32).any() and back(d["status"], 1, np.int32)[0] == 0
        within(back(d["out"], (ROWS, H, HD), np.float32)[:rows], *w["out"], what)
        held = back(d["held"], (ROWS, VOCAB), np.float32)[:rows]
        assert (np.abs(held - w["held"]) <= np.abs(w["held"]) * 2.0 ** -24 * (1 + 2.0 ** -20) + 1e-14).all(), what
        self.pages(what)

    def pages(self, what):
        back, d = self.dev.back, self.d
        assert np.array_equal(back(d["table"], self.table.shape, np.int32), self.table) and np.array_equal(back(d["shares"], N_PAGES, np.int32), self.shares), what
        assert np.array_equal(back(d["stack"], N_PAGES, np.int32), self.stack) and back(d["free"], 1, np.int32)[0] == self.n_free, what
        assert np.array_equal(back(d["pool"], self.pools.shape, np.uint16), self.pools), what

    def branch(self, rng, stream=None, run=True):
        """Some conversations become copies of others, at their end or a few tokens back; some end."""
        src, new = np.arange(SEQS), np.array(self.lens)
        for i in range(SEQS):
            r = rng.random()
            if r < 0.35:
                src[i] = int(rng.integers(0, SEQS))
                new[i] = max(0, self.lens[src[i]] - int(rng.integers(0, 3)) * int(rng.integers(0, 20)))
            elif r < 0.45:
                src[i], new[i] = -1, 0
        for n, a in (("src", src), ("src_old", self.lens), ("src_new", new)):
            self.dev.put(self.d[n], np.asarray(a, np.int32))
        if run:
            self.fork(stream)
        frm, to, rows, status, self.table, self.shares, self.stack, self.n_free = fork_ref(PAGE, src, self.lens, new, self.table, self.shares, self.stack, self.n_free)
        assert status == 0
        out = self.pools.copy()
        for a, b, r in zip(frm, to, rows):
            if a >= 0:
                out[:, :, b, :r] = self.pools[:, :, a, :r]
        self.pools = out
        self.texts = [self.texts[s][:int(n)] if s >= 0 else [] for s, n in zip(src, new)]
        self.lens = new.tolist()
        return frm, to, rows

    def branched(self, want, what):
        for n, x in zip(("frm", "to", "rows"), want):
            assert np.array_equal(self.dev.back(self.d[n], SEQS, np.int32), x), (what, n)
        assert self.dev.back(self.d["fork_status"], 1, np.int32)[0] == 0
        self.pages(what)


@pytest.mark.parametrize("window", [0, 24])
def test_a_server_over_many_steps(lg, dev, window):
    rng = np.random.default_rng(41)
    s = Server(lg, dev, window)
    forked = accepted = shared = 0
    for step in range(28):
        x = s.inputs(rng)
        s.verify()
        w = s.plain(x)
        s.compare(w, f"step {step}")
        accepted += int((w["count"] > 2).sum())
        if step % 3 == 2:
            want = s.branch(rng)
            s.branched(want, f"fork after step {step}")
            forked += int((want[0] >= 0).sum())
            shared += int(s.shares.any())
    assert forked > 3 and accepted > 10 and shared
    dev.free()


def test_the_same_step_recorded_into_graphs(lg, dev):
    """One graph of a step and one of a fork; between replays the host puts other inputs in place and another server runs eagerly."""
    rng, rt = np.random.default_rng(42), dev.rt
    s, other = Server(lg, dev), Server(lg, dev, 24)
    stream = C.c_void_p()
    assert rt.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    graphs = []
    for call in (s.verify, s.fork):
        print("recording", call.__name__, flush=True)
        graph, gexec = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(stream, 0) == 0
        try:
            call(stream)
        finally:
            end = rt.hipStreamEndCapture(stream, C.byref(graph))
        assert end == 0 and graph.value
        assert rt.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
        graphs.append((graph, gexec))
    for replay in range(6):
        x = s.inputs(rng)
        assert rt.hipDeviceSynchronize() == 0
        print(f"replay {replay}", flush=True)
        assert rt.hipGraphLaunch(graphs[0][1], stream) == 0 and rt.hipStreamSynchronize(stream) == 0
        s.compare(s.plain(x), f"replay {replay}")
        y = other.inputs(rng)                                          # eager work of another server in between
        other.verify()
        other.compare(other.plain(y), f"eager {replay}")
        want = s.branch(rng, run=False)
        assert rt.hipDeviceSynchronize() == 0
        assert rt.hipGraphLaunch(graphs[1][1], stream) == 0 and rt.hipStreamSynchronize(stream) == 0
        s.branched(want, f"fork {replay}")
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = rt.hipStreamDestroy.argtypes = [C.c_void_p]
    for graph, gexec in graphs:
        rt.hipGraphExecDestroy(gexec); rt.hipGraphDestroy(graph)
    rt.hipStreamDestroy(stream)
    dev.free()


def test_servers_on_streams_of_their_own(lg, dev):
    """Three servers whose steps overlap, each with its own working memory."""
    rng, rt = np.random.default_rng(43), dev.rt
    servers, streams = [Server(lg, dev, 24 * (k == 1)) for k in range(3)], [C.c_void_p() for _ in range(3)]
    for st in streams:
        assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0
    for step in range(4):
        xs = [s.inputs(rng) for s in servers]
        assert rt.hipDeviceSynchronize() == 0
        for s, st in zip(servers, streams):
            s.verify(st)
        assert rt.hipDeviceSynchronize() == 0
        for k, (s, x) in enumerate(zip(servers, xs)):
            s.compare(s.plain(x), f"step {step} server {k}")
        wants = [s.branch(rng, st) for s, st in zip(servers, streams)]
        assert rt.hipDeviceSynchronize() == 0
        for k, (s, want) in enumerate(zip(servers, wants)):
            s.branched(want, f"fork {step} server {k}")
    rt.hipStreamDestroy.argtypes = [C.c_void_p]
    for st in streams:
        rt.hipStreamDestroy(st)
    dev.free()


def test_a_verified_chain_attends_as_its_tokens_would_one_by_one(lg, dev):
    """The rows of a chain, and lg_hip_paged_attention for each of them as a sequence of its own over the same pages: the same keys."""
    rng = np.random.default_rng(44)
    s = Server(lg, dev)
    s.lens = [40, 3, 0, 100, 17, 64]
    for i in range(SEQS):
        n = -(-s.lens[i] // PAGE)
        s.table[i, :n] = s.stack[s.n_free - n:s.n_free]
        s.n_free -= n
    s.pools[:] = rng.normal(0, 1, s.pools.shape).astype(np.float16).view(np.uint16)
    for n, a in (("table", s.table), ("free", np.array([s.n_free], np.int32)), ("pool", s.pools)):
        dev.put(s.d[n], a)
    x = s.inputs(rng)
    x["parent"] = np.concatenate([np.arange(n) - 1 for n in x["sizes"]] + [np.zeros(ROWS - int(x["start"][-1]), np.int64)])
    dev.put(s.d["parent"], np.asarray(x["parent"], np.int32))
    d, H_ = s.d, s.H
    dev.check(H_.lg_hip_paged_plan(SEQS, PAGE, N_PAGES, BLOCKS, d["old"], d["new"], d["table"], d["stack"], d["free"], d["start"], d["slot"], ROWS, d["status"], s.work[0], s.need[0], None), "plan")
    dev.check(H_.lg_hip_tree_plan(SEQS, MOST, ROWS, d["start"], d["parent"], d["new"], d["mask"], d["pos"], d["seq"], d["bad"], None), "tree_plan")
    dev.check(H_.lg_hip_paged_write(C.byref(s.layers[1]), C.c_void_p(d["x"].value), C.c_void_p(d["x"].value + 4 * WIDTH), 2 * WIDTH, d["slot"], ROWS, None), "write")
    dev.check(H_.lg_hip_paged_tree_attention(C.byref(s.layers[1]), d["q"], H * HD, ROWS, SEQS, MOST, H, d["table"], BLOCKS, d["new"], d["start"], d["mask"], d["pos"], MAX_LEN, 0, 1.0, d["out"], H * HD,
                                             s.work[1], s.need[1], None), "tree attention")
    rows = int(x["start"][-1])
    got, table = dev.back(d["out"], (ROWS, H * HD), np.float32)[:rows], dev.back(d["table"], s.table.shape, np.int32)
    seq = np.repeat(np.arange(SEQS), x["sizes"])
    lens = dev.back(d["pos"], ROWS, np.int32)[:rows] + 1
    p = [dev.up(table[seq]), dev.up(lens, np.int32), dev.up(np.zeros((rows, H * HD), np.float32))]
    need = H_.lg_hip_paged_attention_workspace(rows, H, KV, HD, MAX_LEN, 0)
    dev.check(H_.lg_hip_paged_attention(C.byref(s.layers[1]), d["q"], H * HD, rows, H, p[0], BLOCKS, p[1], MAX_LEN, 0, 1.0, p[2], H * HD, dev.room(need), need, None), "attention")
    want = dev.back(p[2], (rows, H * HD), np.float32)
    dev.free()
    # both are within the bounds of their roundings of the same value: scores of a spread of 2 and 64 dimensions of unit size, at most 110 keys
    assert np.abs(got - want).max() < 2 * 4 * 1e-5
