"""Pages that sequences share, rows moved and pages copied in every layer, through the C ABI against plain forms in whole numbers."""
import ctypes as C

import numpy as np
import pytest

from drafts import compact_ref, fork, fork_ref, layers_of, starts_of
from serving import Device, pages_of, plan, plan_ref

pytestmark = pytest.mark.gpu
NAMES = ("from", "to", "rows", "status", "table", "shares", "stack", "height")


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def pool_of(rng, lens, page, n_pages, blocks):
    """Distinct random pages for the lengths; (table, shares, stack, n_free)."""
    ids = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((len(lens), blocks), -1, np.int32), 0
    for i, n in enumerate(pages_of(lens, page)):
        table[i, :n] = ids[at:at + n]
        at += n
    stack = np.full(n_pages, -7, np.int32)
    stack[:n_pages - at] = ids[at:][::-1]
    return table, np.zeros(n_pages, np.int32), stack, n_pages - at


def same(got, want, what=""):
    for name, g, w in zip(NAMES, got, want):
        assert np.array_equal(g, w), (what, name, g, w)


def sound(page, lens, table, shares, stack, n_free):
    """Every page is free or held as often as its shares say; a last page that is not full is held once."""
    held = np.zeros(stack.size, np.int64)
    for i, n in enumerate(pages_of(lens, page)):
        assert (table[i, n:] == -1).all()
        np.add.at(held, table[i, :n], 1)
        if lens[i] % page:
            assert shares[table[i, n - 1]] == 0, (i, lens[i])
    free = stack[:n_free]
    assert len(set(free.tolist())) == n_free and (held[free] == 0).all() and n_free + (held > 0).sum() == stack.size
    assert np.array_equal(shares, np.maximum(held - 1, 0))


# ---- fork
@pytest.mark.parametrize("n, page, most, steps", [(1, 16, 40, 4), (2, 16, 100, 8), (9, 16, 70, 8), (64, 32, 500, 6), (130, 64, 300, 5), (1000, 16, 60, 4), (4096, 16, 40, 2), (7, 256, 2000, 6)])
def test_forks_cuts_swaps_and_ends(dev, n, page, most, steps):
    """Any sources and lengths, several steps on one table, and growth by the plan in between."""
    rng = np.random.default_rng(n + page)
    lens = rng.integers(0, most + 1, n)
    blocks = int(pages_of(most, page)) + 2
    state = pool_of(rng, lens, page, int(n * blocks) + 5, blocks)
    for step in range(steps):
        src = np.arange(n)
        change = rng.random(n) < (0.6 if step % 2 else 0.2)
        src[change] = rng.integers(-1, n, change.sum())
        new = np.where(src >= 0, lens[src], 0)
        cut = rng.random(n) < 0.4
        new[cut] = np.floor(new[cut] * rng.random(cut.sum()))
        want = fork_ref(page, src, lens, new, *state)
        assert want[3] == 0
        same(fork(dev, page, src, lens, new, *state), want, f"step {step}")
        state, lens = want[4:], new
        sound(page, lens, *state)
        grown = np.minimum(lens + rng.integers(0, page + 3, n), blocks * page)
        got = plan(dev, page, lens, grown, state[0], state[2], state[3], int((grown - lens).sum()))
        ref = plan_ref(page, lens, grown, state[0], state[2], state[3], int((grown - lens).sum()))
        assert ref[2] == 0 and all(np.array_equal(g, w) for g, w in zip(got, ref))
        state, lens = (ref[3], state[1], ref[4], ref[5]), grown
        sound(page, lens, *state)


def test_forks_of_a_prompt_and_their_end(dev):
    """Four answers to one prompt: its whole pages are shared, the last one copied; when they have ended, the pool is as it was."""
    rng = np.random.default_rng(1)
    lens = np.array([100, 0, 0, 0])
    state = pool_of(rng, lens, 16, 20, 8)
    got = fork(dev, 16, [0, 0, 0, 0], lens, [100, 100, 100, 99], *state)
    same(got, fork_ref(16, [0, 0, 0, 0], lens, [100, 100, 100, 99], *state))
    assert got[0].tolist() == [-1] + [state[0][0, 6]] * 3 and got[2].tolist() == [0, 4, 4, 3] and got[5][state[0][0, :7]].tolist() == [3] * 6 + [0]
    back = fork(dev, 16, [0, -1, -1, -1], [100, 100, 100, 99], [100, 0, 0, 0], *got[4:])
    assert back[3] == 0
    for g, w in zip(back[4:], state):
        assert np.array_equal(g, w)


def test_beams_that_trade_places(dev):
    rng = np.random.default_rng(2)
    lens = np.array([33, 40, 47, 48])
    state = pool_of(rng, lens, 16, 30, 4)
    src, new = np.array([1, 0, 2, 2]), np.array([40, 33, 47, 47])
    got = fork(dev, 16, src, lens, new, *state)
    same(got, fork_ref(16, src, lens, new, *state))
    assert got[0].tolist() == [-1, -1, -1, state[0][2, 2]]           # a place that is traded is no copy; row 2 keeps its page
    sound(16, new, *got[4:])


@pytest.mark.parametrize("change, status", [
    (dict(old=[20, -1, 0]), 1), (dict(old=[20, 65, 0]), 1), (dict(new=[20, 20, 21]), 1), (dict(new=[20, 20, -1]), 1), (dict(src=[0, -1, 0]), 1), (dict(src=[0, 3, 0]), 4), (dict(src=[0, -2, 0]), 4),
    (dict(n_free=-1), 8), (dict(n_free=9), 8), (dict(page0=(0, 0, -1)), 16), (dict(page0=(0, 1, 8)), 16), (dict(shares=-1), 32), (dict(shares=5000), 32), (dict(n_free=0), 2),
    (dict(stack=-7), 16)])
def test_what_is_wrong_is_told_and_nothing_is_done(dev, change, status):
    rng = np.random.default_rng(3)
    src, old, new = np.array([0, 1, 0]), np.array([20, 20, 0]), np.array([20, 20, 20])
    table, shares, stack, n_free = pool_of(rng, old, 16, 8, 4)
    src, old, new = (np.array(change.get(k, v)) for k, v in (("src", src), ("old", old), ("new", new)))
    n_free = change.get("n_free", n_free)
    if "page0" in change:
        i, b, p = change["page0"]
        table[i, b] = p
    if "shares" in change:
        shares[table[0, 0]] = change["shares"]
    if "stack" in change:
        stack[:] = change["stack"]
    got = fork(dev, 16, src, old, new, table, shares, stack, n_free)
    same(got, fork_ref(16, src, old, new, table, shares, stack, n_free))
    assert got[3] == status


def test_shares_that_are_too_few(dev):
    """A page that two rows hold and whose shares say one: both let it go."""
    rng = np.random.default_rng(4)
    table, shares, stack, n_free = pool_of(rng, np.array([16, 0]), 16, 8, 4)
    table[1, 0] = table[0, 0]
    args = 16, [-1, -1], np.array([16, 16]), np.array([0, 0]), table, shares, stack, n_free
    got = fork(dev, *args)
    same(got, fork_ref(*args))
    assert got[3] == 32


def test_no_sequence(dev):
    got = fork(dev, 16, [], [], [], np.zeros((0, 4), np.int32), np.zeros(8, np.int32), np.arange(8, dtype=np.int32), 8)
    assert got[3] == 0 and got[7] == 8


# ---- rows and pages in every layer
def paths(rng, sizes, most):
    path, count = np.full((len(sizes), most), -1, np.int32), np.zeros(len(sizes), np.int32)
    for i, n in enumerate(sizes):
        count[i] = rng.integers(0, n + 1)
        rows = np.sort(rng.choice(n, count[i], replace=False)) if count[i] else []
        if count[i] and rng.random() < 0.8:
            rows[0] = 0
        path[i, :count[i]] = rows
    return path, count


@pytest.mark.parametrize("layers, n, most, kv, hd, page", [(1, 1, 2, 1, 64, 16), (3, 7, 64, 2, 64, 16), (2, 5, 17, 1, 512, 32), (65, 3, 9, 1, 64, 16), (130, 2, 33, 2, 64, 16), (4, 70, 20, 2, 128, 64),
                                                           (2, 3, 64, 8, 256, 16), (1, 2, 30, 3, 128, 256)])
def test_rows_of_paths(lg, dev, layers, n, most, kv, hd, page):
    rng = np.random.default_rng(layers * 100 + n)
    sizes = rng.integers(1, most + 1, n)
    sizes[0] = most
    lens = sizes + rng.integers(0, 50, n)
    held = pages_of(lens, page)
    n_pages, blocks = int(held.sum()) + 2, int(held.max()) + 1
    table, _, _, _ = pool_of(rng, lens, page, n_pages, blocks)
    start = starts_of(sizes)
    path, count = paths(rng, sizes, most)
    pools = rng.integers(0, 1 << 16, (layers, 2, n_pages, page, kv * hd)).astype(np.uint16)
    ls, pool = layers_of(lg, pools, kv, hd, dev)
    p = [dev.up(x, np.int32) for x in (table, lens, start, path, count)]
    dev.check(dev.H.lg_hip_paged_compact(ls, layers, n, most, p[0], blocks, *p[1:], None), "paged_compact")
    got = dev.back(pool, pools.shape, np.uint16)
    dev.free()
    assert np.array_equal(got, compact_ref(pools, page, n_pages, table, lens, start, path, count))
    assert n * most == 2 or not np.array_equal(got, pools)           # (the smallest tree may have nothing to move)


def test_paths_that_do_not_rise_and_rows_without_a_place(lg, dev):
    rng = np.random.default_rng(5)
    sizes = np.array([6, 6, 6, 6, 6, 6])
    lens = np.array([20, 20, 20, 5, 40, 20])
    table, _, _, _ = pool_of(rng, np.full(6, 20), 16, 14, 2)
    table[5, 1], table[2, 0] = 99, -3
    path = np.array([[0, 3, 2, 5], [0, 2, 6, 7], [0, 2, 3, 5], [0, 2, 3, 4], [0, 2, 3, 4], [1, 2, 4, 5]], np.int32)
    count = np.array([4, 4, 9, 4, 4, 4])
    pools = rng.integers(0, 1 << 16, (2, 2, 14, 16, 64)).astype(np.uint16)
    ls, pool = layers_of(lg, pools, 1, 64, dev)
    p = [dev.up(x, np.int32) for x in (table, lens, starts_of(sizes), path, count)]
    dev.check(dev.H.lg_hip_paged_compact(ls, 2, 6, 4, p[0], 2, *p[1:], None), "paged_compact")
    got = dev.back(pool, pools.shape, np.uint16)
    want = compact_ref(pools, 16, 14, table, lens, starts_of(sizes), path, count)
    # (trees of more than max_tree rows are left alone: all of them here)
    assert np.array_equal(got, pools) and np.array_equal(want, pools)
    path6 = np.pad(path, ((0, 0), (0, 2)), constant_values=-1)
    p[3] = dev.up(path6)
    dev.check(dev.H.lg_hip_paged_compact(ls, 2, 6, 6, p[0], 2, *p[1:], None), "paged_compact")
    got = dev.back(pool, pools.shape, np.uint16)
    want = compact_ref(pools, 16, 14, table, lens, starts_of(sizes), path6, count)
    dev.free()
    assert np.array_equal(got, want) and not np.array_equal(got, pools)


def test_layers_of_different_heads(lg, dev):
    """One table, layers whose rows are not alike in width and whose strides leave room."""
    rng = np.random.default_rng(6)
    n_pages, page = 6, 16
    shapes = [(2, 64, 128 + 8, 17), (1, 512, 512, 16), (3, 128, 400, 20)]                   # key heads, size, row stride, rows of a page
    hosts = [[rng.integers(0, 1 << 16, (n_pages, rows, stride)).astype(np.uint16) for _ in range(2)] for _, _, stride, rows in shapes]
    devs = [[dev.up(x) for x in h] for h in hosts]
    ls = (lg.hiplib.Pages * 3)(*(lg.hiplib.Pages(d[0].value, d[1].value, n_pages, page, kv, hd, stride, stride * rows) for d, (kv, hd, stride, rows) in zip(devs, shapes)))
    table, lens, start = np.array([[4, 1], [0, 5]], np.int32), np.array([20, 31]), np.array([0, 8, 20])
    path, count = np.full((2, 12), -1, np.int32), np.array([3, 4])
    path[0, :3], path[1, :4] = [0, 2, 7], [1, 5, 6, 11]
    p = [dev.up(x, np.int32) for x in (table, lens, start, path, count)]
    dev.check(dev.H.lg_hip_paged_compact(ls, 3, 2, 12, p[0], 2, *p[1:], None), "paged_compact")
    q = [dev.up(x, np.int32) for x in ([2, -1, 5, 3, 1], [3, 2, 0, 99, 1], [16, 4, 7, 3, 9])]
    for h, d, (kv, hd, _, _) in zip(hosts, devs, shapes):
        for x, y in zip(h, d):
            want = x.copy()
            w = kv * hd
            want[:, :page, :w] = compact_ref(x[None, None, :, :page, :w], page, n_pages, table, lens, start, path, count)[0, 0]
            assert np.array_equal(dev.back(y, x.shape, np.uint16), want)
            x[:] = want
    dev.check(dev.H.lg_hip_paged_copy(ls, 3, 5, *q, None), "paged_copy")
    for h, d, (kv, hd, _, _) in zip(hosts, devs, shapes):
        for x, y in zip(h, d):
            want, w = x.copy(), kv * hd
            want[3, :16, :w], want[0, :7, :w] = x[2, :16, :w], x[5, :7, :w]
            assert np.array_equal(dev.back(y, x.shape, np.uint16), want)
    dev.free()


@pytest.mark.parametrize("layers, n, kv, hd, page", [(1, 1, 1, 64, 16), (3, 9, 2, 128, 32), (70, 2, 1, 64, 16), (2, 300, 1, 64, 16), (1, 3, 8, 256, 256), (2, 5, 3, 64, 64)])
def test_pages_are_copied(lg, dev, layers, n, kv, hd, page):
    rng = np.random.default_rng(layers + n)
    n_pages = 2 * n + 1
    ids = rng.permutation(n_pages)
    frm, to, rows = ids[:n].copy(), ids[n:2 * n].copy(), rng.integers(0, page + 3, n)
    rows[0] = page
    if n > 2:
        frm[1], to[2] = -1, n_pages
    pools = rng.integers(0, 1 << 16, (layers, 2, n_pages, page, kv * hd)).astype(np.uint16)
    ls, pool = layers_of(lg, pools, kv, hd, dev)
    p = [dev.up(x, np.int32) for x in (frm, to, rows)]
    dev.check(dev.H.lg_hip_paged_copy(ls, layers, n, *p, None), "paged_copy")
    got = dev.back(pool, pools.shape, np.uint16)
    dev.free()
    want = pools.copy()
    for a, b, r in zip(frm, to, rows):
        if 0 <= a < n_pages and 0 <= b < n_pages:
            want[:, :, b, :r] = pools[:, :, a, :r]
    assert np.array_equal(got, want)


def test_nothing_to_move(lg, dev):
    H = dev.H
    assert H.lg_hip_paged_compact(None, 0, 3, 4, None, 2, None, None, None, None, None) == 0
    assert H.lg_hip_paged_copy(None, 0, 3, None, None, None, None) == 0
    g = lg.hiplib.Pages(1 << 20, 1 << 20, 8, 16, 1, 64, 64, 1024)
    assert H.lg_hip_paged_compact(C.byref(g), 1, 0, 4, None, 2, None, None, None, None, None) == 0
    assert H.lg_hip_paged_copy(C.byref(g), 1, 0, None, None, None, None) == 0
