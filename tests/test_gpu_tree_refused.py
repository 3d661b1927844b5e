"""Steps of which a part is refused: trees that the plan tells to be wrong, and pages that are not enough.  What is refused leaves its sequence at the committed length, and the others as they would be alone."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_tree_step as step
from drafts import accept_ref, random_parents, starts_of, tree_accept, tree_plan, tree_plan_ref
from serving import Device, plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def test_nothing_is_accepted_in_trees_that_are_refused(dev):
    """Chains whose every token is the one picked: all rows would be passed.  Refused ones keep the committed length, and no token is picked behind them."""
    n = 5
    parent = np.tile(np.arange(n) - 1, 6)
    parent[n + 2] = 3                                              # tree 1: a parent that is a later row
    parent[2 * n + 4] = -1                                         # tree 2: none, in its last row
    parent[5 * n + 1] = 64                                         # tree 5: one that no tree has; too short besides
    start, lens = np.arange(7) * n, np.array([30, 30, 30, 3, 0, 4])
    token, after = np.tile(np.arange(n), 6), np.tile(np.arange(n) + 1, 6)
    status = tree_plan(dev, start, parent, lens, 8)[3]
    assert status.tolist() == [0, 2, 2, 4, 4, 6]
    path, count, ends, last = tree_accept(dev, start, parent, token, after, lens, 8)
    assert count.tolist() == [5, 1, 1, 0, 0, 0]
    assert path[:3].tolist() == [[0, 1, 2, 3, 4, -1, -1, -1], [0] + [-1] * 7, [0] + [-1] * 7] and (path[3:] == -1).all()
    assert ends.tolist() == [30, 25, 25, 3, 0, 4]
    assert last.tolist() == [5, -1, -1, -1, -1, -1]


@pytest.mark.parametrize("n, most", [(3, 1), (7, 64), (300, 9)])
def test_the_closing_plan_takes_the_lengths_of_refused_trees(dev, n, most):
    """A batch in which a third of the trees have a parent that is no earlier row and a third a length below their rows: lengths stay what a plan takes, and the sound trees' are what they are alone."""
    rng = np.random.default_rng(n * 100 + most)
    sizes = rng.integers(1, most + 1, n)
    start = starts_of(sizes)
    parent = np.concatenate([random_parents(rng, int(x)) for x in sizes])
    lens = sizes + rng.integers(0, 50, n)
    kind = np.arange(n) % 3
    for i in range(n):
        if kind[i] == 1 and sizes[i] > 1:
            parent[start[i] + int(rng.integers(1, sizes[i]))] = int(rng.choice([-1, 64, sizes[i] - 1 if sizes[i] > 1 else 5]))
        if kind[i] == 2:
            lens[i] = int(rng.integers(0, sizes[i]))
    token, after = rng.integers(0, 3, parent.size), rng.integers(-1, 3, parent.size)
    status = tree_plan(dev, start, parent, lens, most)[3]
    path, count, ends, last = tree_accept(dev, start, parent, token, after, lens, most)
    ways = accept_ref(start, np.where(parent < 0, -1, parent), token, after, lens, most)
    for i in range(n):
        if status[i] == 0:
            assert path[i].tolist() == ways[0][i].tolist() and (count[i], ends[i], last[i]) == tuple(int(x[i]) for x in ways[1:])
        elif status[i] & 4:
            assert (path[i] == -1).all() and (count[i], ends[i], last[i]) == (0, lens[i], -1)
        else:
            assert path[i].tolist() == [0] + [-1] * (most - 1) and (count[i], ends[i], last[i]) == (1, lens[i] - sizes[i], -1)
    assert (status != 0).any() and (status == 0).any()
    # back from the grown lengths to those, in pages that hold the grown ones
    page, blocks = 16, int(-(-lens.max() // 16)) + 1
    held = -(-lens // page)
    table, at = np.full((n, blocks), -1, np.int32), 0
    for i, m in enumerate(held):
        table[i, :m] = np.arange(at, at + m)
        at += int(m)
    got = plan(dev, page, lens.tolist(), ends.tolist(), table, np.zeros(at + 1, np.int32), 0, 0)
    assert got[2] == 0 and got[5] == int((held - -(-ends // page)).sum())


# ---- a growth plan that is refused
class Careful(step.Server):
    """The step as it is documented: lengths behind the plan come from what the plan has given, and each plan has a status word of its own."""

    def __init__(self, lg, dev, window=0):
        super().__init__(lg, dev, window)
        self.d["grown"], self.d["back"] = dev.up(np.full(step.SEQS, 77, np.int32)), dev.up(np.full(1, 77, np.int32))

    def verify(self, stream=None):
        d, H_, check, S = self.d, self.H, self.dev.check, step
        size = (S.SEQS, S.PAGE, S.N_PAGES, S.BLOCKS)
        check(H_.lg_hip_paged_plan(*size, d["old"], d["new"], d["table"], d["stack"], d["free"], d["start"], d["slot"], S.ROWS, d["status"], self.work[0], self.need[0], stream), "plan")
        check(H_.lg_hip_tree_plan_from(S.SEQS, S.MOST, S.ROWS, d["start"], d["parent"], d["old"], d["grown"], d["mask"], d["pos"], d["seq"], d["bad"], stream), "tree_plan_from")
        for i in range(S.LAYERS):
            x = d["x"].value + i * S.ROWS * 2 * S.WIDTH * 4
            check(H_.lg_hip_paged_write(C.byref(self.layers[i]), C.c_void_p(x), C.c_void_p(x + 4 * S.WIDTH), 2 * S.WIDTH, d["slot"], S.ROWS, stream), "write")
        check(H_.lg_hip_paged_tree_attention(C.byref(self.layers[1]), d["q"], S.H * S.HD, S.ROWS, S.SEQS, S.MOST, S.H, d["table"], S.BLOCKS, d["grown"], d["start"], d["mask"], d["pos"], S.MAX_LEN,
                                             self.window, 1.0, d["out"], S.H * S.HD, self.work[1], self.need[1], stream), "attention")
        check(H_.lg_hip_adjust_logits(C.byref(self.rules), d["logits"], S.VOCAB, S.ROWS, S.VOCAB, d["held"], S.VOCAB, stream), "rules")
        check(H_.lg_hip_sample(d["held"], S.VOCAB, S.ROWS, S.VOCAB, d["how"], d["u"], d["next"], None, None, self.work[2], self.need[2], stream), "sample")
        check(H_.lg_hip_tree_accept(S.SEQS, S.MOST, S.ROWS, d["start"], d["parent"], d["token"], d["next"], d["grown"], d["path"], d["count"], d["len"], d["last"], stream), "accept")
        check(H_.lg_hip_paged_compact(self.layers, S.LAYERS, S.SEQS, S.MOST, d["table"], S.BLOCKS, d["grown"], d["start"], d["path"], d["count"], stream), "compact")
        check(H_.lg_hip_paged_plan(*size, d["grown"], d["len"], d["table"], d["stack"], d["free"], d["start2"], None, 0, d["back"], self.work[0], self.need[0], stream), "plan back")

    def nothing_happened(self, x, bit, what):
        """The first plan told, lengths are the committed ones, and pages, table and stack are as they were."""
        back, d, n = self.dev.back, self.d, step.SEQS
        assert back(d["status"], 1, np.int32)[0] == bit and back(d["back"], 1, np.int32)[0] == 0, what
        assert (back(d["start"], n + 1, np.int32) == 0).all() and (back(d["slot"], step.ROWS, np.int32) == -1).all(), what
        for name in ("grown", "len"):
            assert np.array_equal(back(d[name], n, np.int32), x["old"]), (what, name)
        assert (back(d["count"], n, np.int32) == 0).all() and (back(d["path"], (n, step.MOST), np.int32) == -1).all() and (back(d["last"], n, np.int32) == -1).all(), what
        assert not back(d["bad"], n, np.int32).any(), what
        assert (back(d["out"], (step.ROWS, step.H * step.HD), np.float32) == 77).all(), what
        self.pages(what)

    def happened(self, x, what):
        w = self.plain(x)
        assert np.array_equal(self.dev.back(self.d["grown"], step.SEQS, np.int32), x["new"]) and self.dev.back(self.d["back"], 1, np.int32)[0] == 0, what
        self.compare(w, what)


def steps_of_which_some_are_refused(s, rng, run):
    """Every third step finds too few free pages, or has more rows than the lengths have room for; then the same step again with what it needs."""
    dev, refused = s.dev, 0
    for k in range(9):
        x = s.inputs(rng)
        grows = (-(-x["new"] // step.PAGE) + x["old"] // -step.PAGE).sum()
        dev.put(s.d["out"], np.full((step.ROWS, step.H * step.HD), 77, np.float32))
        # (what lies in table entries that no sequence holds does not matter)
        if k % 3 == 1 and grows:
            kept, s.n_free = s.n_free, int(grows) - 1
            dev.put(s.d["free"], np.array([s.n_free], np.int32))
            run(f"step {k}, {s.n_free} pages for {grows}")
            s.nothing_happened(x, 2, f"step {k}")
            s.n_free = kept
            dev.put(s.d["free"], np.array([kept], np.int32))
            refused += 1
        if k % 3 == 2:
            new = x["new"].copy()
            new[k % step.SEQS] = step.MAX_LEN + 1
            dev.put(s.d["new"], new.astype(np.int32))
            run(f"step {k}, a length above the room")
            s.nothing_happened(x, 1, f"step {k}")
            dev.put(s.d["new"], x["new"].astype(np.int32))
            refused += 1
        run(f"step {k}")
        s.happened(x, f"step {k}")
    assert refused > 4


@pytest.mark.parametrize("window", [0, 24])
def test_a_refused_growth_plan_leaves_the_step_without_effect(lg, dev, window):
    s = Careful(lg, dev, window)

    def run(what):
        s.verify()
    steps_of_which_some_are_refused(s, np.random.default_rng(51), run)
    dev.free()


def test_a_refused_growth_plan_in_a_recorded_step(lg, dev):
    """One graph for steps that are taken and steps that are refused, with another server's eager steps in between."""
    rng, rt = np.random.default_rng(52), dev.rt
    s, other = Careful(lg, dev), Careful(lg, dev, 24)
    stream, graph, gexec = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert rt.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    assert rt.hipDeviceSynchronize() == 0 and rt.hipStreamBeginCapture(stream, 0) == 0
    try:
        s.verify(stream)
    finally:
        end = rt.hipStreamEndCapture(stream, C.byref(graph))
    assert end == 0 and rt.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0

    def run(what):
        print(what, flush=True)
        y = other.inputs(rng)
        assert rt.hipDeviceSynchronize() == 0
        assert rt.hipGraphLaunch(gexec, stream) == 0 and rt.hipStreamSynchronize(stream) == 0
        other.verify()
        other.happened(y, what)
    steps_of_which_some_are_refused(s, rng, run)
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = rt.hipStreamDestroy.argtypes = [C.c_void_p]
    rt.hipGraphExecDestroy(gexec), rt.hipGraphDestroy(graph), rt.hipStreamDestroy(stream)
    dev.free()


def test_lengths_behind_a_plan(dev):
    """Those ahead of it and the rows it has given: also of trees that are refused, and none where no plan can have given them."""
    n_rows, most = 18, 4
    start = np.array([0, 3, 9, 10, 12, 12, 14, 13, 30])
    parent = np.array([-1, 0, 1, -1, 0, 0, 0, 0, 0, -1, -1, 5, -1, 0, 0, 0, 0, 0])
    before = np.array([7, 20, 0, 38, 9, -2, 50, 61])
    n = len(before)
    p = [dev.up(x, t) for x, t in ((start, np.int32), (parent, np.int32), (before, np.int32), (np.full(n, 77), np.int32), (np.full(n_rows, 77), np.uint64), (np.full(n_rows, 77), np.int32),
                                   (np.full(n_rows, 77), np.int32), (np.full(n, 77), np.int32))]
    dev.check(dev.H.lg_hip_tree_plan_from(n, most, n_rows, *p, None), "tree_plan_from")
    grown, status = dev.back(p[3], n, np.int32), dev.back(p[7], n, np.int32)
    mask, pos, seq = dev.back(p[4], n_rows, np.uint64), dev.back(p[5], n_rows, np.int32), dev.back(p[6], n_rows, np.int32)
    dev.free()
    assert grown.tolist() == [10, 26, 1, 40, 9, 0, 50, 78] and status.tolist() == [0, 1, 0, 2, 0, 4, 1, 1]
    assert mask[[0, 1, 2, 9, 10, 12]].tolist() == [1, 3, 7, 1, 0, 0]
    assert pos[[0, 1, 2, 9, 10, 12]].tolist() == [7, 8, 9, 0, -1, -1] and seq[[0, 9, 12]].tolist() == [0, 2, 5]


def test_a_step_without_rows_has_the_lengths_ahead_of_it(dev):
    p = [dev.up(x, np.int32) for x in ([0, 0, 0, 0], [5, 0, 70], [77] * 3, [77] * 3)]
    dev.check(dev.H.lg_hip_tree_plan_from(3, 4, 0, p[0], None, p[1], p[2], None, None, None, p[3], None), "tree_plan_from")
    assert dev.back(p[2], 3, np.int32).tolist() == [5, 0, 70] and dev.back(p[3], 3, np.int32).tolist() == [0, 0, 0]
    dev.free()


@pytest.mark.parametrize("n, most", [(1, 64), (257, 9)])
def test_both_forms_of_the_tree_plan_agree(dev, n, most):
    rng = np.random.default_rng(n)
    sizes, before = rng.integers(0, most + 1, n), rng.integers(0, 1000, n)
    sizes[0] = most
    start, parent = starts_of(sizes), np.concatenate([random_parents(rng, int(x)) for x in sizes])
    p = [dev.up(x, t) for x, t in ((start, np.int32), (parent, np.int32), (before, np.int32), (np.zeros(n), np.int32), (np.zeros(parent.size), np.uint64), (np.zeros(parent.size), np.int32),
                                   (np.zeros(parent.size), np.int32), (np.full(n, 77), np.int32))]
    dev.check(dev.H.lg_hip_tree_plan_from(n, most, parent.size, *p, None), "tree_plan_from")
    got = dev.back(p[4], parent.size, np.uint64), dev.back(p[5], parent.size, np.int32), dev.back(p[6], parent.size, np.int32)
    assert np.array_equal(dev.back(p[3], n, np.int32), before + sizes) and np.array_equal(dev.back(p[2], n, np.int32), before)
    dev.free()
    for x, w in zip(got, tree_plan_ref(start, parent, before + sizes)):
        assert np.array_equal(x, w)
