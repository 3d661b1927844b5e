"""The operators of a batched decode step together, as a server calls them: plan, write, attend, (a product,) sample, over steps in which sequences
come, grow, lose drafts and end; the same recorded into a graph; and calls on several streams at once."""
import ctypes as C

import numpy as np
import pytest

from serving import Device, attend_ref, pages_of, plan_ref, sample_ref, within

pytestmark = pytest.mark.gpu
H, KV, HD, PAGE, BLOCKS, N_PAGES, SEQS, VOCAB = 8, 2, 64, 16, 12, 60, 6, 9000
WIDTH, MAX_LEN = KV * HD, 12 * 16
HOW = [(1.0, 20, 0.95, 0.0), (0.8, 0, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0), (0.7, 3000, 0.99, 0.0)]


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


class Server:
    """A pool, its bookkeeping and one step's buffers on the device, with the plain forms' state beside them."""

    def __init__(self, lg, dev, slots):
        self.lg, self.dev, self.slots, self.H = lg, dev, slots, dev.H
        z = np.zeros((N_PAGES, PAGE, WIDTH), np.uint16)
        self.k, self.v = np.zeros((N_PAGES, PAGE, KV, HD), np.float16), np.zeros((N_PAGES, PAGE, KV, HD), np.float16)
        self.table, self.stack, self.n_free = np.full((SEQS, BLOCKS), -1, np.int32), np.arange(N_PAGES, dtype=np.int32), N_PAGES
        self.dk, self.dv = dev.up(z), dev.up(z)
        self.d = {n: dev.up(a) for n, a in dict(
            old=np.zeros(SEQS, np.int32), new=np.zeros(SEQS, np.int32), table=self.table, stack=self.stack, free=np.array([N_PAGES], np.int32),
            start=np.zeros(SEQS + 1, np.int32), slot=np.zeros(slots, np.int32), status=np.zeros(1, np.int32), x=np.zeros((slots, 2 * WIDTH), np.float32),
            q=np.zeros((SEQS, H * HD), np.float32), out=np.zeros((SEQS, H * HD), np.float32), logits=np.zeros((SEQS, VOCAB), np.float32),
            u=np.zeros(SEQS, np.float32), tok=np.zeros(SEQS, np.int32), prob=np.zeros(SEQS, np.float32), kept=np.zeros(SEQS, np.int32)).items()}
        raw = np.zeros(SEQS, np.dtype([("t", "f4"), ("k", "i4"), ("p", "f4"), ("m", "f4")]))
        for i, x in enumerate(HOW):
            raw[i] = x
        self.d["how"] = dev.up(raw.view(np.uint8))
        self.need = [self.H.lg_hip_paged_plan_workspace(SEQS), self.H.lg_hip_paged_attention_workspace(SEQS, H, KV, HD, MAX_LEN, 0), self.H.lg_hip_sample_workspace(SEQS, VOCAB)]
        self.work = [dev.room(n) for n in self.need]
        self.pages = lg.hiplib.Pages(self.dk.value, self.dv.value, N_PAGES, PAGE, KV, HD, WIDTH, WIDTH * PAGE)

    def cache(self, stream=None):
        d, H_ = self.d, self.H
        self.dev.check(H_.lg_hip_paged_plan(SEQS, PAGE, N_PAGES, BLOCKS, d["old"], d["new"], d["table"], d["stack"], d["free"], d["start"], d["slot"], self.slots,
                                            d["status"], self.work[0], self.need[0], stream), "plan")
        self.dev.check(H_.lg_hip_paged_write(C.byref(self.pages), d["x"], C.c_void_p(d["x"].value + 4 * WIDTH), 2 * WIDTH, d["slot"], self.slots, stream), "write")
        self.dev.check(H_.lg_hip_paged_attention(C.byref(self.pages), d["q"], H * HD, SEQS, H, d["table"], BLOCKS, d["new"], MAX_LEN, 0, 1.0, d["out"], H * HD,
                                                 self.work[1], self.need[1], stream), "attention")

    def draw(self, stream=None):
        d = self.d
        self.dev.check(self.H.lg_hip_sample(d["logits"], VOCAB, SEQS, VOCAB, d["how"], d["u"], d["tok"], d["prob"], d["kept"], self.work[2], self.need[2], stream), "sample")

    def inputs(self, rng, old, new):
        x = rng.normal(0, 1, (self.slots, 2 * WIDTH)).astype(np.float32)
        q = (rng.normal(0, 2, (SEQS, H * HD)) / 8).astype(np.float32)
        for n, a in (("old", np.asarray(old, np.int32)), ("new", np.asarray(new, np.int32)), ("x", x), ("q", q)):
            self.dev.put(self.d[n], a)
        return x, q

    def plain(self, old, new, x, q):
        start, slot, status, self.table, self.stack, self.n_free = plan_ref(PAGE, list(old), list(new), self.table, self.stack, self.n_free, self.slots)
        assert status == 0
        for i, s in enumerate(slot.tolist()):
            if s >= 0:
                self.k[s // PAGE, s % PAGE] = x[i, :WIDTH].reshape(KV, HD)
                self.v[s // PAGE, s % PAGE] = x[i, WIDTH:].reshape(KV, HD)
        return start, slot, attend_ref(q.reshape(SEQS, H, HD), self.k, self.v, self.table, new, PAGE, N_PAGES, KV, 0, 1.0, MAX_LEN)

    def compare(self, new, start, slot, want, what):
        back = self.dev.back
        assert np.array_equal(back(self.d["start"], SEQS + 1, np.int32), start) and np.array_equal(back(self.d["slot"], self.slots, np.int32), slot)
        assert np.array_equal(back(self.d["table"], self.table.shape, np.int32), self.table)
        assert np.array_equal(back(self.dk, self.k.shape, np.uint16), self.k.view(np.uint16)) and np.array_equal(back(self.dv, self.v.shape, np.uint16), self.v.view(np.uint16))
        got = back(self.d["out"], (SEQS, H, HD), np.float32)
        within(got, *want, what)
        assert (got[np.asarray(new) == 0] == 0).all()
        return got

    def check_draw(self, logits, us, what):
        got = [self.dev.back(self.d[n], SEQS, t) for n, t in (("tok", np.int32), ("kept", np.int32))]
        want = [sample_ref(logits[i], *HOW[i], us[i]) for i in range(SEQS)]
        assert got[0].tolist() == [w[0] for w in want] and got[1].tolist() == [w[2] for w in want], what


def lengths(rng, old, slots):
    """The next lengths: one more token for most, a prompt for the empty ones, some drafts taken back, some at their end."""
    new = [min(n + 1, MAX_LEN) if n else int(rng.integers(0, 25)) for n in old]
    for i in range(SEQS):
        r = rng.random()
        if r < 0.15:
            new[i] = max(0, old[i] - int(rng.integers(0, 20)))
        elif r < 0.25:
            new[i] = 0
    return new


def numbers(rng, logits):
    us = rng.random(SEQS).astype(np.float32)
    for i in range(SEQS):
        while not sample_ref(logits[i], *HOW[i], us[i])[3]:
            us[i] = np.float32(rng.random())
    return us


def test_a_server_over_many_steps(lg, dev):
    rng = np.random.default_rng(31)
    s = Server(lg, dev, 128)
    head = rng.normal(0, 0.7, (H * HD, VOCAB)).astype(np.float32)
    old = [0] * SEQS
    for step in range(14):
        new = lengths(rng, old, s.slots)
        x, q = s.inputs(rng, old, new)
        s.cache()
        start, slot, want = s.plain(old, new, x, q)
        got = s.compare(new, start, slot, want, f"step {step}")
        logits = (got.reshape(SEQS, -1) @ head).astype(np.float32)
        us = numbers(rng, logits)
        dev.put(s.d["logits"], logits); dev.put(s.d["u"], us)
        s.draw()
        s.check_draw(logits, us, f"step {step}")
        old = new
    dev.free()


def test_the_same_step_recorded_into_a_graph(lg, dev):
    """One graph of plan, write, attend and sample; between its replays the host puts other lengths, rows, logits and numbers in place and runs other work; every
    replay gives what the plain forms give."""
    rng, rt = np.random.default_rng(32), dev.rt
    s, other = Server(lg, dev, 128), Server(lg, dev, 128)
    stream, graph, gexec = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert rt.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    print("recording a step", flush=True)
    assert rt.hipStreamBeginCapture(stream, 0) == 0
    try:
        s.cache(stream); s.draw(stream)
    finally:
        end = rt.hipStreamEndCapture(stream, C.byref(graph))
    assert end == 0 and graph.value
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    assert rt.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
    old, o2 = [0] * SEQS, [0] * SEQS
    for replay in range(6):
        new = lengths(rng, old, s.slots)
        x, q = s.inputs(rng, old, new)
        logits = rng.normal(0, 4, (SEQS, VOCAB)).astype(np.float32)
        us = numbers(rng, logits)
        dev.put(s.d["logits"], logits); dev.put(s.d["u"], us)
        assert rt.hipDeviceSynchronize() == 0
        print(f"replay {replay}", flush=True)
        assert rt.hipGraphLaunch(gexec, stream) == 0
        start, slot, want = s.plain(old, new, x, q)
        s.compare(new, start, slot, want, f"replay {replay}")
        s.check_draw(logits, us, f"replay {replay}")
        old = new
        n2 = lengths(rng, o2, other.slots)                  # eager work of another server in between
        x, q = other.inputs(rng, o2, n2)
        other.cache()
        other.compare(n2, *other.plain(o2, n2, x, q), f"eager {replay}")
        o2 = n2
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = rt.hipStreamDestroy.argtypes = [C.c_void_p]
    rt.hipGraphExecDestroy(gexec); rt.hipGraphDestroy(graph); rt.hipStreamDestroy(stream)
    dev.free()


def test_servers_on_streams_of_their_own(lg, dev):
    """Three servers whose steps overlap, each with its own working memory."""
    rng, rt = np.random.default_rng(33), dev.rt
    servers, streams = [Server(lg, dev, 128) for _ in range(3)], [C.c_void_p() for _ in range(3)]
    for st in streams:
        assert rt.hipStreamCreateWithFlags(C.byref(st), 1) == 0
    olds = [[0] * SEQS for _ in servers]
    for step in range(4):
        todo = []
        for s, old in zip(servers, olds):
            new = lengths(rng, old, s.slots)
            x, q = s.inputs(rng, old, new)
            logits = rng.normal(0, 4, (SEQS, VOCAB)).astype(np.float32)
            us = numbers(rng, logits)
            dev.put(s.d["logits"], logits); dev.put(s.d["u"], us)
            todo.append((new, x, q, logits, us))
        assert rt.hipDeviceSynchronize() == 0
        for s, st in zip(servers, streams):
            s.cache(st); s.draw(st)
        assert rt.hipDeviceSynchronize() == 0
        for k, (s, old, (new, x, q, logits, us)) in enumerate(zip(servers, olds, todo)):
            s.compare(new, *s.plain(old, new, x, q), f"step {step} server {k}")
            s.check_draw(logits, us, f"step {step} server {k}")
            olds[k] = new
    rt.hipStreamDestroy.argtypes = [C.c_void_p]
    for st in streams:
        rt.hipStreamDestroy(st)
    dev.free()
