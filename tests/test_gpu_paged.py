"""Pages of a shared KV cache through the C ABI against plain forms in 64 bits: the plan of a step, the rows of new tokens, attention of one new
token per sequence."""
import ctypes as C

import numpy as np
import pytest

from serving import Device, attend_ref, pages_of, plan, plan_ref, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def pool_of(rng, lens, page, n_pages, blocks):
    """Distinct random pages for the lengths; (table, stack, n_free)."""
    ids = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((len(lens), blocks), -1, np.int32), 0
    for i, n in enumerate(pages_of(lens, page)):
        table[i, :n] = ids[at:at + n]
        at += n
    stack = np.full(n_pages, -7, np.int32)
    stack[:n_pages - at] = ids[at:]
    return table, stack, n_pages - at


def same(got, want):
    for name, g, w in zip(("start", "slots", "status", "table", "stack", "height"), got, want):
        assert np.array_equal(g, w), (name, g, w)


# ---- plan
@pytest.mark.parametrize("n, page, most, grow, shrink", [
    (1, 16, 1, 1, 0), (1, 256, 3000, 5, 0), (7, 16, 40, 1, 0), (64, 32, 2000, 1, 0), (65, 64, 500, 700, 0), (130, 16, 300, 3, 40), (1000, 16, 100, 17, 100),
    (1025, 128, 400, 1, 1), (4096, 16, 33, 2, 3), (3, 16, 100, 20000, 0), (256, 16, 700, 1, 3), (257, 16, 64, 1, 0), (9, 16, 2000, 2000, 2000), (40, 64, 3, 60, 3)])
def test_plan_of_a_step_and_its_undoing(dev, n, page, most, grow, shrink):
    rng = np.random.default_rng(n * 1000 + page)
    old = rng.integers(0, most + 1, n)
    new = old + (rng.integers(0, grow + 1, n) if grow > 1 else 1)
    if shrink:
        back = rng.random(n) < 0.4
        new[back] = np.maximum(0, old[back] - rng.integers(0, shrink + 1, back.sum()))
    blocks = int(pages_of(max(old.max(), new.max()), page)) + 1
    n_pages = int(pages_of(np.maximum(old, new), page).sum()) + 3
    table, stack, nf = pool_of(rng, old, page, n_pages, blocks)
    n_slots = max(int(np.maximum(0, new - old).sum()), int(np.maximum(0, old - new).sum())) + 2
    print(f"plan n={n} page={page} most={most} grow={grow} shrink={shrink} slots={n_slots}", flush=True)
    want = plan_ref(page, old.tolist(), new.tolist(), table, stack, nf, n_slots)
    assert want[2] == 0
    got = plan(dev, page, old, new, table, stack, nf, n_slots)
    same(got, want)
    used = got[1][got[1] >= 0]
    assert len(set(used.tolist())) == used.size
    # exchanged, it restores table and stack
    again = plan(dev, page, new, old, got[3], got[4], got[5], n_slots)
    same(again, plan_ref(page, new.tolist(), old.tolist(), want[3], want[4], want[5], n_slots))
    assert np.array_equal(again[3], table) and again[5] == nf and np.array_equal(again[4][:nf], stack[:nf])


def test_plan_of_no_sequence_and_of_exact_room(dev):
    stack = np.arange(4, dtype=np.int32)
    start, slots, status, _, s2, nf = plan(dev, 16, [], [], np.zeros((0, 3), np.int32), stack, 2, 5)
    assert status == 0 and start.tolist() == [0] and (slots == -1).all() and nf == 2 and np.array_equal(s2, stack)
    # the last free page, the last slot, a table filled to its end; and steps in which nothing changes
    table = np.array([[3, -1], [2, 1]], np.int32)
    for old, new, nf, n_slots in (([16, 32], [17, 32], 1, 1), ([16, 32], [16, 32], 1, 0), ([0, 0], [0, 0], 4, 1), ([16, 32], [0, 0], 1, 0)):
        got = plan(dev, 16, old, new, table, stack, nf, n_slots)
        same(got, plan_ref(16, old, new, table, stack, nf, n_slots))
        assert got[2] == 0


@pytest.mark.parametrize("old, new, nf, n_slots, change, status", [
    ([5, 40], [-1, 41], 9, 9, {}, 1), ([5, 40], [5, 65], 9, 99, {}, 1), ([5, 65], [5, 40], 9, 99, {}, 1), ([-2**31, 40], [5, 40], 9, 9, {}, 1),
    ([5, 40], [40, 64], 2, 99, {}, 2), ([5, 40], [6, 42], 9, 2, {}, 4), ([5, 40], [40, 64], 2, 9, {}, 6), ([5, 40], [6, 41], -1, 9, {}, 8),
    ([5, 40], [6, 41], 13, 9, {}, 8), ([5, 40], [0, 0], 9, 9, {}, 8), ([5, 40], [6, 41], 8, 9, {(0, 0): 12}, 16), ([5, 40], [6, 41], 8, 9, {(1, 2): -1}, 16),
    ([5, 40], [0, 41], 8, 9, {(0, 0): 1 << 30}, 16), ([5, 48], [5, 49], 8, 9, {"stack": 12}, 16), ([5, 48], [5, 49], 8, 9, {"stack": -1}, 16)])
def test_plan_reports_and_leaves_everything_as_it_was(dev, old, new, nf, n_slots, change, status):
    table = np.array([[3, -1, -1, -1], [2, 1, 0, -1]], np.int32)
    stack = np.array([4, 5, 6, 7, 8, 9, 10, 11, 11, 11, 11, 11], np.int32)
    for at, v in change.items():
        if at == "stack":
            stack[nf - 1] = v
        else:
            table[at] = v
    start, slots, st, t2, s2, nf2 = plan(dev, 16, old, new, table, stack, nf, n_slots)
    assert st == status and (start == 0).all() and (slots == -1).all()
    assert np.array_equal(t2, table) and np.array_equal(s2, stack) and nf2 == nf


@pytest.mark.parametrize("n, grow", [(200, 1), (900, 1), (300, 40)])
def test_plan_of_many_sequences_refuses_one_bad_page(dev, n, grow):
    """Whichever wavefront finds it, all of them refuse: a page outside the cache in the first, the last and another sequence, and on the stack."""
    rng = np.random.default_rng(n)
    old = rng.integers(1, 120, n)
    old[[0, n // 2, n - 1]] = 21                             # (a page that is written into; and one that is taken)
    old[1] = 32
    new = old + grow
    n_pages = int(pages_of(new, 16).sum()) + 2
    table, stack, nf = pool_of(rng, old, 16, n_pages, 12)
    n_slots = n * grow
    for i in (0, n // 2, n - 1, None):
        t, s = table.copy(), stack.copy()
        if i is None:
            s[nf - 1] = n_pages
        else:
            t[i, pages_of(old[i], 16) - 1] = -5
        want = plan_ref(16, old.tolist(), new.tolist(), t, s, nf, n_slots)
        assert want[2] == 16
        for _ in range(5):
            same(plan(dev, 16, old, new, t, s, nf, n_slots), want)


def test_plan_through_many_steps_keeps_every_page_once(dev):
    rng = np.random.default_rng(5)
    page, n, n_pages, blocks = 16, 23, 150, 12
    lens = np.zeros(n, np.int64)
    table, stack, nf = pool_of(rng, lens, page, n_pages, blocks)
    for step in range(12):
        new = np.clip(lens + rng.integers(-30, 45, n), 0, blocks * page)
        new[rng.random(n) < 0.1] = 0
        want = plan_ref(page, lens.tolist(), new.tolist(), table, stack, nf, 2000)
        got = plan(dev, page, lens, new, table, stack, nf, 2000)
        same(got, want)
        if got[2] == 0:
            lens, table, stack, nf = new, got[3], got[4], got[5]
        held = [int(x) for i in range(n) for x in table[i, :pages_of(lens[i], page)]]
        assert sorted(held + stack[:nf].tolist()) == list(range(n_pages))


# ---- write
@pytest.mark.parametrize("n_tok, kv, hd, page, pad, fused", [(1, 2, 64, 16, 0, 0), (3, 1, 512, 256, 8, 1), (64, 2, 256, 16, 0, 8), (333, 8, 256, 64, 24, 0), (29, 3, 128, 32, 8, 5)])
def test_write_rounds_into_the_slots(lg, dev, n_tok, kv, hd, page, pad, fused):
    rng = np.random.default_rng(n_tok)
    width, n_pages = kv * hd, -(-n_tok // page) + 2
    row, stride = width + pad, (fused + 2 * kv) * hd
    page_stride = row * page + 3 * pad
    x = (rng.normal(0, 1, (n_tok, stride)) * 2.0 ** rng.integers(-28, 18, (n_tok, stride))).astype(np.float32)
    x[0, fused * hd:fused * hd + 8] = [65504.0, 65519.9, 65520.0, -np.inf, np.nan, -0.0, 2.0 ** -25, 3 * 2.0 ** -25]
    slots = rng.permutation(n_pages * page)[:n_tok].astype(np.int32)
    for at, s in ((1, -1), (2, n_pages * page), (5, 2**31 - 1), (7, -2**31)):
        if at < n_tok:
            slots[at] = s
    before = rng.integers(0, 2**16, (2, n_pages, page_stride)).astype(np.uint16)
    dk, dv = dev.up(before[0]), dev.up(before[1])
    dx, ds = dev.up(x), dev.up(slots)
    p = lg.hiplib.Pages(dk.value, dv.value, n_pages, page, kv, hd, row, page_stride)
    k0 = C.c_void_p(dx.value + 4 * fused * hd)
    v0 = C.c_void_p(dx.value + 4 * (fused + kv) * hd)
    print(f"write {n_tok} x {kv} x {hd}", flush=True)
    dev.check(dev.H.lg_hip_paged_write(C.byref(p), k0, v0, stride, ds, n_tok, None), "paged_write")
    want = before.copy()
    with np.errstate(over="ignore"):
        h = x.astype(np.float16).view(np.uint16)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < n_pages * page:
            for which in (0, 1):
                at = (s % page) * row
                want[which, s // page, at:at + width] = h[i, (fused + which * kv) * hd:(fused + which * kv + kv) * hd]
    for which, d in ((0, dk), (1, dv)):
        got = dev.back(d, before[which].shape, np.uint16)
        nan = np.isnan(want[which].view(np.float16))
        assert np.array_equal(got[~nan], want[which][~nan]) and np.isnan(got.view(np.float16)[nan]).all()
    dev.free()


# ---- attend
def attend(lg, dev, q, k, v, table, lens, page, kv, window, scale, max_len, pad=0, qpad=0, opad=0, poison=True, stream=None, work=None):
    """q [n][H][hd], k / v [n_pages][page][kv][hd] binary16; rows and pages `pad` values apart, what lies between them poisoned."""
    n, H, hd = q.shape
    n_pages, width = k.shape[0], kv * hd
    row, page_stride = width + pad, (width + pad) * page + 2 * pad
    mem = []
    for x in (k, v):
        wide = np.full((n_pages, page_stride), 0x7E00 if poison else 0, np.uint16)               # NaN
        for r in range(page):
            wide[:, r * row:r * row + width] = x.view(np.uint16)[:, r].reshape(n_pages, width)
        mem.append(dev.up(wide))
    qs, os_ = H * hd + qpad, H * hd + opad
    qw = np.full((n, qs), np.nan, np.float32)
    qw[:, :H * hd] = q.reshape(n, -1)
    out = np.full((n + 1, os_), 7.5, np.float32)                                                  # a row behind the last sequence too
    dq, dt, dl, do = dev.up(qw), dev.up(table, np.int32), dev.up(lens, np.int32), dev.up(out)
    need = dev.H.lg_hip_paged_attention_workspace(n, H, kv, hd, max_len, window)
    p = lg.hiplib.Pages(mem[0].value, mem[1].value, n_pages, page, kv, hd, row, page_stride)
    dev.check(dev.H.lg_hip_paged_attention(C.byref(p), dq, qs, n, H, dt, table.shape[1], dl, max_len, window, scale, do, os_, work or dev.room(need), need, stream), "paged_attention")
    got = dev.back(do, out.shape, np.float32)
    dev.free()
    assert (got[n] == 7.5).all() and (got[:, H * hd:] == 7.5).all()
    return got[:n, :H * hd].reshape(n, H, hd)


def case(rng, H, kv, hd, page, lens, spread=2.0, extra=2):
    n_pages = int(pages_of(lens, page).sum()) + extra
    blocks = int(pages_of(max(lens), page)) + 1
    table, _, _ = pool_of(rng, lens, page, n_pages, blocks)
    k, v = (rng.normal(0, 1, (n_pages, page, kv, hd)).astype(np.float16) for _ in range(2))
    q = (rng.normal(0, spread, (len(lens), H, hd)) / np.sqrt(hd)).astype(np.float32)
    # places that no sequence holds: infinities and NaN
    held = np.zeros((n_pages, page), bool)
    for i, n in enumerate(lens):
        pos = np.arange(n)
        held[table[i, pos // page], pos % page] = True
    for x, bad in ((k, np.float16(np.nan)), (v, np.float16(np.inf))):
        x[~held] = bad
    return q, k, v, table


SHAPES = [
    (8, 2, 64, 16, 0, [0, 1, 15, 16, 17, 31, 32, 33, 100, 127, 128, 129]),
    (8, 2, 256, 32, 0, [1, 129, 1000, 0, 257, 2049]),
    (8, 2, 256, 16, 512, [1, 511, 512, 513, 544, 0, 2000]),
    (16, 8, 256, 64, 1024, [1023, 1024, 1025, 3000, 5]),
    (8, 1, 512, 128, 0, [1, 700, 64]),
    (5, 1, 64, 16, 333, [333, 334, 1, 800, 365]),
    (8, 8, 128, 256, 0, [511, 512, 513, 1]),
    (12, 4, 256, 32, 1, [1, 2, 33, 64]),
    (8, 2, 128, 16, 31, [64, 63, 65, 40]),
    (3, 3, 64, 16, 0, [5000]),
]


@pytest.mark.parametrize("H, kv, hd, page, window, lens", SHAPES)
@pytest.mark.parametrize("pad", [0, 8])
def test_attention_of_one_token_per_sequence(lg, dev, H, kv, hd, page, window, lens, pad):
    rng = np.random.default_rng(H * 100 + hd + page + window)
    q, k, v, table = case(rng, H, kv, hd, page, lens)
    max_len = max(lens) + (pad and 500)
    print(f"attend H={H} kv={kv} hd={hd} page={page} window={window} lens={lens} pad={pad}", flush=True)
    want, bound = attend_ref(q, k, v, table, lens, page, k.shape[0], kv, window, 1.0, max_len)
    got = attend(lg, dev, q, k, v, table, lens, page, kv, window, 1.0, max_len, pad=pad, qpad=4 * pad, opad=pad)
    within(got, want, bound)
    empty = np.array(lens) == 0
    assert (got[empty] == 0).all()


@pytest.mark.parametrize("n, H, kv, hd, window", [(63, 2, 2, 64, 0), (64, 2, 1, 64, 40), (65, 2, 2, 64, 0), (300, 4, 2, 64, 0), (1025, 1, 1, 64, 33), (4096, 1, 1, 64, 0)])
def test_attention_of_many_sequences(lg, dev, n, H, kv, hd, window):
    """A lane, a thread or several of one for the lengths; sequences of one split beside such of many; most free places of a batch."""
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 40, n)
    lens[rng.integers(0, n, 3)] = 1500
    lens[rng.random(n) < 0.3] = 0
    q, k, v, table = case(rng, H, kv, hd, 16, lens)
    print(f"attend {n} sequences", flush=True)
    want, bound = attend_ref(q, k, v, table, lens, 16, k.shape[0], kv, window, 1.0, 1500)
    within(attend(lg, dev, q, k, v, table, lens, 16, kv, window, 1.0, 1500), want, bound)


@pytest.mark.parametrize("n, H, kv, hd, window, longest", [(65, 8, 2, 64, 0, 2500), (66, 1, 1, 64, 0, 20011), (300, 4, 2, 128, 0, 3000), (70, 8, 2, 256, 2100, 2500),
                                                           (67, 8, 1, 512, 0, 1500), (1025, 2, 1, 64, 0, 3001), (4096, 1, 1, 64, 0, 2500)])
def test_attention_of_many_sequences_in_splits(lg, dev, n, H, kv, hd, window, longest):
    """More sequences than a wavefront has lanes, one of them long and a few of middle length: cut by the launch ahead; more splits of one sequence than a
    wavefront joins at a time; one length that a captured call would bring later."""
    rng = np.random.default_rng(n + hd)
    lens = rng.integers(0, 50, n)
    lens[rng.integers(0, n, 4)] = 700
    lens[rng.random(n) < 0.2] = 0
    lens[n // 3] = longest
    q, k, v, table = case(rng, H, kv, hd, 16, lens)
    print(f"attend {n} sequences of up to {longest}, hd={hd}", flush=True)
    for told in (lens, np.minimum(lens, 40), np.zeros_like(lens)):
        want, bound = attend_ref(q, k, v, table, told, 16, k.shape[0], kv, window, 1.0, longest)
        within(attend(lg, dev, q, k, v, table, told, 16, kv, window, 1.0, longest), want, bound)


@pytest.mark.parametrize("lens", [[0], [0, 0, 0], [1, 0, 31]])
def test_split_attention_of_more_key_heads_than_workgroups_at_a_time(lg, dev, lens):
    """A cut of next to nothing among 300 heads of 512, all sequences empty or nearly."""
    rng = np.random.default_rng(len(lens))
    q, k, v, table = case(rng, 300, 300, 512, 16, lens)
    want, bound = attend_ref(q, k, v, table, lens, 16, k.shape[0], 300, 0, 1.0, 1000)
    within(attend(lg, dev, q, k, v, table, lens, 16, 300, 0, 1.0, 1000), want, bound)


@pytest.mark.parametrize("n, H, kv, hd, longest", [(3, 8, 2, 256, 3000), (64, 4, 1, 64, 2500), (70, 8, 2, 128, 2500)])
def test_split_attention_in_two_graphs_at_once(lg, dev, n, H, kv, hd, longest):
    """Joined splits recorded into two graphs, each with working memory of its own that holds rubbish; between the replays, which overlap, the lengths change
    and eager calls run.  Every replay gives to the bit what the call by itself gives, and that is near the plain form."""
    rng, rt = np.random.default_rng(n), dev.rt
    most = np.where(np.arange(n) % 7 == 0, longest, 90)
    q, k, v, table = case(rng, H, kv, hd, 32, most)
    mem = [dev.up(x.view(np.uint16)) for x in (k, v)]
    dq, dt, dl, out = dev.up(q), dev.up(table, np.int32), dev.up(most, np.int32), [dev.up(np.zeros((n, H, hd), np.float32)) for _ in range(3)]
    p = lg.hiplib.Pages(mem[0].value, mem[1].value, k.shape[0], 32, kv, hd, kv * hd, 32 * kv * hd)
    need = dev.H.lg_hip_paged_attention_workspace(n, H, kv, hd, longest, 0)
    assert need > 0
    work = [dev.up(np.full(need, 0xFF, np.uint8)) for _ in range(3)]

    def call(i, stream=None):
        dev.check(dev.H.lg_hip_paged_attention(C.byref(p), dq, H * hd, n, H, dt, table.shape[1], dl, longest, 0, 1.0, out[i], H * hd, work[i], need, stream), "paged_attention")

    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = rt.hipStreamDestroy.argtypes = [C.c_void_p]
    streams, graphs, execs = [[C.c_void_p() for _ in range(2)] for _ in range(3)]
    for i in range(2):
        assert rt.hipStreamCreateWithFlags(C.byref(streams[i]), 1) == 0
        assert rt.hipStreamBeginCapture(streams[i], 0) == 0
        try:
            call(i, streams[i])
        finally:
            end = rt.hipStreamEndCapture(streams[i], C.byref(graphs[i]))
        assert end == 0 and rt.hipGraphInstantiate(C.byref(execs[i]), graphs[i], None, None, 0) == 0
    for replay in range(4):
        lens = most if replay == 0 else np.where(rng.random(n) < 0.2, 0, rng.integers(1, most + 1))
        dev.put(dl, lens.astype(np.int32))
        assert rt.hipDeviceSynchronize() == 0
        print(f"replay {replay}", flush=True)
        for i in range(2):
            assert rt.hipGraphLaunch(execs[i], streams[i]) == 0
        call(2)
        assert rt.hipDeviceSynchronize() == 0
        got = [dev.back(o, (n, H, hd), np.float32) for o in out]
        assert np.array_equal(got[0], got[2]) and np.array_equal(got[1], got[2])
        within(got[2], *attend_ref(q, k, v, table, lens, 32, k.shape[0], kv, 0, 1.0, longest), f"replay {replay}")
    for i in range(2):
        rt.hipGraphExecDestroy(execs[i]); rt.hipGraphDestroy(graphs[i]); rt.hipStreamDestroy(streams[i])
    dev.free()


def test_attention_of_large_and_tiny_queries_and_scales(lg, dev):
    """Scores from almost equal to one key far above the rest, queries near the ends of f32's range, a negative scale, rows of zeros."""
    rng = np.random.default_rng(3)
    lens = [700, 45, 300, 33, 64, 1]
    q, k, v, table = case(rng, 4, 2, 128, 16, lens)
    for spread, scale in ((2.0 ** -60, 2.0 ** 61), (2.0 ** 50, 2.0 ** -49), (12.0, 1.0), (3.0, -0.5), (0.0, 1.0), (1e-38, 1.0), (2.0, 0.0), (2.0 ** -100, 2.0 ** 101)):
        qs = (q * np.float32(0.5) * np.float32(spread)).astype(np.float32)
        want, bound = attend_ref(qs, k, v, table, lens, 16, k.shape[0], 2, 0, float(np.float32(scale)), 700)
        got = attend(lg, dev, qs, k, v, table, lens, 16, 2, 0, scale, 700)
        within(got, want, bound, (spread, scale))


def test_attention_clamps_lengths_and_leaves_out_bad_pages(lg, dev):
    """Lengths beyond max_len and the table count as these; negative ones as 0; positions of pages outside the pool are left out, whole sequences too."""
    rng = np.random.default_rng(11)
    lens = [200, 90, 160, 64, 48]
    q, k, v, table = case(rng, 8, 2, 64, 16, lens)
    k, v = np.nan_to_num(k, nan=0.5), np.nan_to_num(v, posinf=0.25)
    table[0, 3] = -1; table[0, 5] = k.shape[0]; table[1, :] = 2**31 - 1; table[2, 0] = -2**31; table[3, 3] = k.shape[0] + 5
    for max_len, told in ((4096, [200, 90, 160, 64, 48]), (150, [200, 90, 2**31 - 1, 64, -5]), (1, [200, 1, 0, 64, -2**31]), (0, lens)):
        want, bound = attend_ref(q, k, v, table, told, 16, k.shape[0], 2, 0, 1.0, max_len)
        got = attend(lg, dev, q, k, v, table, np.array(told), 16, 2, 0, 1.0, max_len)
        within(got, want, bound, max_len)


def test_rows_of_a_verify_block_are_sequences_that_share_pages(lg, dev):
    """Five rows of one sequence: the same table row, lengths one apart."""
    rng = np.random.default_rng(12)
    _, k, v, table = case(rng, 8, 2, 256, 32, [1003])
    q = (rng.normal(0, 2, (5, 8, 256)) / 16).astype(np.float32)
    lens = np.arange(999, 1004)
    got = attend(lg, dev, q, k, v, np.repeat(table, 5, 0), lens, 32, 2, 0, 1.0, 1003)
    want, bound = attend_ref(q, k, v, np.repeat(table, 5, 0), lens, 32, k.shape[0], 2, 0, 1.0, 1003)
    within(got, want, bound)


def test_attention_beyond_32_bits_of_offset(lg, dev):
    """Pages 2^27 values apart, 20 of them: value offsets pass 2^31 and byte offsets 2^32.  Only the pages in use are written."""
    rng = np.random.default_rng(13)
    H, kv, hd, page, stride, n_pages = 4, 2, 64, 16, 1 << 27, 20
    lens = np.array([45, 16])
    table = np.array([[19, 17, 0], [18, -1, -1]], np.int32)
    k, v = (rng.normal(0, 1, (n_pages, page, kv, hd)).astype(np.float16) for _ in range(2))
    q = (rng.normal(0, 2, (2, H, hd)) / 8).astype(np.float32)
    big = dev.room(n_pages * stride * 2)
    for p in (0, 17, 18, 19):
        dev.put(C.c_void_p(big.value + 2 * p * stride), k[p])
        dev.put(C.c_void_p(big.value + 2 * (p * stride + stride // 2)), v[p])
    new = rng.normal(0, 1, (1, 2 * kv * hd)).astype(np.float32)
    dn, ds = dev.up(new), dev.up([19 * page + 3], np.int32)
    p = lg.hiplib.Pages(big.value, big.value + stride, n_pages, page, kv, hd, kv * hd, stride)
    dev.check(dev.H.lg_hip_paged_write(C.byref(p), dn, C.c_void_p(dn.value + 4 * kv * hd), 2 * kv * hd, ds, 1, None), "paged_write")
    k[19, 3], v[19, 3] = new[0, :kv * hd].reshape(kv, hd), new[0, kv * hd:].reshape(kv, hd)
    dq, dt, dl, do = dev.up(q), dev.up(table), dev.up(lens, np.int32), dev.room(q.nbytes)
    need = dev.H.lg_hip_paged_attention_workspace(2, H, kv, hd, 48, 0)
    dev.check(dev.H.lg_hip_paged_attention(C.byref(p), dq, H * hd, 2, H, dt, 3, dl, 48, 0, 1.0, do, H * hd, dev.room(need), need, None), "paged_attention")
    got = dev.back(do, q.shape, np.float32)
    dev.free()
    want, bound = attend_ref(q, k, v, table, lens, page, n_pages, kv, 0, 1.0, 48)
    within(got, want, bound)


def test_infinities_and_nan_stay_with_the_sequences_that_see_them(lg, dev):
    rng = np.random.default_rng(14)
    lens = [100, 70]
    q, k, v, table = case(rng, 8, 2, 64, 16, lens)
    clean = attend(lg, dev, q, k, v, table, lens, 16, 2, 0, 1.0, 100)
    for x, at, bad in ((v, 50, np.inf), (k, 20, np.nan), (v, 99, np.nan), (k, 0, np.inf)):
        y = x.copy()
        y[table[0, at // 16], at % 16, 1] = bad                        # sequence 0, key head 1
        args = (q, y if x is k else k, y if x is v else v)
        got = attend(lg, dev, *args, table, lens, 16, 2, 0, 1.0, 100)
        assert np.array_equal(got[1], clean[1]) and np.array_equal(got[0, :4], clean[0, :4])
        assert not np.isfinite(got[0, 4:]).any()
        # and out of the window they are out of sight
        if at < 50:
            assert np.isfinite(attend(lg, dev, *args, table, lens, 16, 2, 50, 1.0, 100)).all()
