"""Trees of drafted tokens through the C ABI against plain forms: ancestors, positions and accepted paths in whole numbers, attention in 64 bits."""
import numpy as np
import pytest

from drafts import accept_ref, bits, random_parents, starts_of, tree_accept, tree_attend, tree_attend_ref, tree_plan, tree_plan_ref
from serving import Device, pages_of, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def forest(rng, sizes, kind="any"):
    return np.concatenate([random_parents(rng, int(n), kind) for n in sizes] + [np.zeros(0, np.int64)]).astype(np.int64)


# ---- plan and accept
@pytest.mark.parametrize("n, most, kind", [(1, 1, "any"), (1, 8, "any"), (1, 64, "chain"), (3, 64, "star"), (5, 17, "any"), (64, 33, "any"), (257, 64, "any"), (4096, 5, "any"), (9, 64, "chain")])
def test_ancestors_positions_and_paths(dev, n, most, kind):
    rng = np.random.default_rng(n * 100 + most)
    sizes = rng.integers(0, most + 1, n)
    sizes[0] = most
    start, parent = starts_of(sizes), forest(rng, sizes, kind)
    lens = sizes + rng.integers(0, 100, n)
    mask, pos, seq, status = tree_plan(dev, start, parent, lens, most)
    want = tree_plan_ref(start, parent, lens)
    assert not status.any()
    assert np.array_equal(mask, want[0]) and np.array_equal(pos, want[1]) and np.array_equal(seq, want[2])
    token = rng.integers(0, 9, parent.size)                          # few different ones, so that several rows fit
    after = rng.integers(-1, 9, parent.size)
    for got, ref in zip(tree_accept(dev, start, parent, token, after, lens, most), accept_ref(start, parent, token, after, lens, most)):
        assert np.array_equal(got, ref)


def test_a_whole_chain_is_accepted(dev):
    parent = np.arange(64) - 1
    token, after = np.arange(64) + 5, np.arange(64) + 6
    path, count, ends, last = tree_accept(dev, [0, 64], parent, token, after, [1000], 64)
    assert path[0].tolist() == list(range(64)) and count[0] == 64 and ends[0] == 1000 and last[0] == 69


def test_trees_that_do_not_fit_are_told(dev):
    """A tree with too many rows, a falling start, rows outside the step, a parent that is not an earlier row, a length below the rows: the others are as they would be alone."""
    # rows:        0..2   3..3+5 (too many)  8 (fine) ...
    start = np.array([0, 3, 9, 10, 12, 14, 13, 30])
    parent = np.array([-1, 0, 1, -1, 0, 0, 0, 0, 0, -1, -1, 5, -1, 0, 0, 0, 0, 0])
    lens = np.array([10, 20, 30, 40, 1, 50, 60])
    mask, pos, seq, status = tree_plan(dev, start, parent, lens, 4, n_rows=18)
    assert status.tolist() == [0, 1, 0, 2, 4, 1, 1]
    assert mask[:3].tolist() == [1, 3, 7] and pos[:3].tolist() == [7, 8, 9] and seq[:3].tolist() == [0, 0, 0]
    assert mask[9] == 1 and pos[9] == 29 and mask[10:14].tolist() == [0, 0, 0, 0] and pos[10:14].tolist() == [-1] * 4
    untouched = [3, 4, 5, 6, 7, 8, 14, 15, 16, 17]
    assert (mask[untouched] == 77).all() and (pos[untouched] == 77).all() and (seq[untouched] == 77).all()
    path, count, ends, last = tree_accept(dev, start, parent, np.zeros(18), np.zeros(18), lens, 4, n_rows=18)
    assert count.tolist()[:4] == [3, 0, 1, 1] and count[5:].tolist() == [0, 0]
    assert ends[1] == 20 and last[1] == -1 and (path[1] == -1).all() and ends[6] == 60


def test_no_sequence_and_no_rows(dev):
    assert dev.H.lg_hip_tree_plan(0, 4, 0, *[None] * 7, None) == 0
    mask, pos, seq, status = tree_plan(dev, [0, 0, 0], np.zeros(0, np.int64), [5, 0], 4)
    assert status.tolist() == [0, 0]
    path, count, ends, last = tree_accept(dev, [0, 0, 0], np.zeros(0, np.int64), [], [], [5, 0], 4)
    assert (path == -1).all() and count.tolist() == [0, 0] and ends.tolist() == [5, 0] and last.tolist() == [-1, -1]


# ---- attention
def scene(rng, committed, sizes, heads, kv, hd, page, kind="any", spare=3, blocks=None):
    committed, sizes = np.asarray(committed), np.asarray(sizes)
    lens = committed + sizes
    held = pages_of(lens, page)
    n_pages = int(held.sum()) + spare
    blocks = blocks or int(max(1, held.max())) + 1
    ids = rng.permutation(n_pages)
    table, at = np.full((len(lens), blocks), -1, np.int32), 0
    for i, m in enumerate(held):
        table[i, :m] = ids[at:at + m]
        at += m
    k, v = (rng.normal(0, 1, (n_pages, page, kv, hd)).astype(np.float16) for _ in range(2))
    start, parent = starts_of(sizes), forest(rng, sizes, kind)
    mask, pos, _ = tree_plan_ref(start, parent, lens)
    q = (rng.normal(0, 2, (parent.size, heads, hd)) / hd ** 0.5).astype(np.float32)
    return dict(q=q, k=k, v=v, table=table, lens=lens, start=start, mask=mask, pos=pos)


def check(lg, dev, s, kv, window=0, scale=1.0, most=None, max_len=None, pad=0, what=""):
    page, n_pages = s["k"].shape[1], s["k"].shape[0]
    most = most or int(max(1, np.diff(s["start"]).max()))
    max_len = max_len if max_len is not None else int(s["lens"].max())
    got = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=window, scale=scale, max_len=max_len, pad=pad)
    want, bound = tree_attend_ref(**s, page=page, n_pages=n_pages, n_head_kv=kv, window=window, scale=scale, max_len=max_len)
    within(got, want, bound, what)
    return got


@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 64), (5, 1, 64), (8, 8, 64), (8, 2, 128), (3, 3, 128), (8, 1, 128), (8, 2, 256), (16, 8, 256), (8, 1, 256), (8, 1, 512), (2, 2, 512), (4, 1, 512)])
@pytest.mark.parametrize("most", [1, 5, 16, 23, 64])
def test_trees_of_all_sizes_over_all_heads(lg, dev, heads, kv, hd, most):
    rng = np.random.default_rng(heads * 1000 + kv * 100 + hd + most)
    committed = [0, 1, 15, 16, 33, 200]
    sizes = [most, max(1, most - 1), 1, most, (most + 1) // 2, most]
    check(lg, dev, scene(rng, committed, sizes, heads, kv, hd, 16), kv, what="whole")


@pytest.mark.parametrize("heads, kv, hd, most, page", [(8, 2, 64, 5, 16), (8, 2, 64, 64, 32), (8, 2, 128, 16, 64), (8, 4, 128, 64, 16), (8, 2, 256, 4, 128), (8, 2, 256, 16, 16), (8, 2, 256, 37, 256), (8, 1, 512, 2, 16),
                                                       (8, 1, 512, 9, 32)])
def test_long_sequences_in_splits(lg, dev, heads, kv, hd, most, page):
    rng = np.random.default_rng(hd + most)
    check(lg, dev, scene(rng, [2500, 1, 3000, 700], [most, most, max(1, most // 2), 1], heads, kv, hd, page), kv)


@pytest.mark.parametrize("window", [1, 2, 7, 31, 32, 33, 100, 512])
@pytest.mark.parametrize("kind", ["chain", "any"])
def test_windows_end_in_the_tree_and_before_it(lg, dev, window, kind):
    rng = np.random.default_rng(window)
    check(lg, dev, scene(rng, [0, 5, 40, 64, 300, 1500], [40, 3, 64, 17, 33, 20], 8, 2, 64, 16, kind), 2, window=window)
    check(lg, dev, scene(rng, [0, 31, 1500], [40, 3, 20], 8, 2, 256, 32, kind), 2, window=window)


@pytest.mark.parametrize("n, hd, window", [(65, 64, 0), (200, 128, 0), (70, 256, 300), (130, 512, 0)])
def test_many_sequences(lg, dev, n, hd, window):
    rng = np.random.default_rng(n)
    committed = (1200 * rng.random(n) ** 3).astype(np.int64)
    committed[:2] = 1200, 0
    check(lg, dev, scene(rng, committed, rng.integers(1, 7, n), 4, 1, hd, 32), 1, window=window)


@pytest.mark.parametrize("scale, size", [(1.0, 30.0), (0.0625, 1.0), (-1.0, 1.0), (0.0, 1.0), (1.0, 1e-30), (1e-20, 1e22)])
def test_scales_and_sizes_of_queries(lg, dev, scale, size):
    rng = np.random.default_rng(5)
    s = scene(rng, [100, 0, 700], [9, 4, 16], 8, 2, 128, 16)
    s["q"] *= np.float32(size)
    check(lg, dev, s, 2, scale=scale)


def test_rows_that_are_not_aligned(lg, dev):
    rng = np.random.default_rng(6)
    check(lg, dev, scene(rng, [100, 700], [9, 16], 8, 2, 64, 16), 2, pad=4)
    check(lg, dev, scene(rng, [100, 2700], [9, 16], 8, 2, 256, 16), 2, pad=12)


def test_more_room_than_is_used(lg, dev):
    """max_tree, max_len and the table as a captured step has them."""
    rng = np.random.default_rng(7)
    check(lg, dev, scene(rng, [100, 700, 3], [9, 16, 1], 8, 2, 64, 16, blocks=300), 2, most=64, max_len=4800)
    check(lg, dev, scene(rng, [100, 700, 3], [9, 16, 1], 8, 2, 256, 16, blocks=300), 2, most=33, max_len=4800, window=512)


def test_sets_of_the_callers_own(lg, dev):
    """No row, later rows, rows that are not above each other; rows that the tree does not have are not seen."""
    rng = np.random.default_rng(8)
    s = scene(rng, [0, 50, 33], [12, 12, 30], 8, 2, 64, 16)
    s["mask"] = rng.integers(0, 1 << 62, s["mask"].size).astype(np.uint64)
    s["mask"][[0, 13]] = 0
    got = check(lg, dev, s, 2)
    assert (got[0] == 0).all()                                       # nothing committed and no row of the tree
    check(lg, dev, s, 2, window=9)


def test_rows_without_a_position_see_nothing(lg, dev):
    rng = np.random.default_rng(9)
    s = scene(rng, [40, 50, 2000], [6, 20, 5], 8, 2, 64, 16)
    s["pos"] = s["pos"].copy()
    s["pos"][[1, 7, 8, 27]] = [-1, 49, -5, 1999]
    for window in (0, 10):
        got = check(lg, dev, s, 2, window=window)
        assert (got[[1, 7, 8, 27]] == 0).all() and (np.abs(got).sum((1, 2)) > 0).sum() == 27


def test_sequences_that_do_not_fit(lg, dev):
    """Lengths below the rows or above the room: zeros.  Trees with too many rows or outside the step, and rows of no tree: as they were."""
    rng = np.random.default_rng(10)
    s = scene(rng, [40, 50, 60, 70, 80], [6, 9, 5, 4, 3], 8, 2, 64, 16)
    s["lens"] = s["lens"].copy()
    s["lens"][0] = 5
    s["lens"][2] = 1 << 30
    got = tree_attend(lg, dev, **s, most=6, n_head_kv=2, window=0, scale=1.0, max_len=120, n_rows=26)
    want, bound = tree_attend_ref(**s, page=16, n_pages=s["k"].shape[0], n_head_kv=2, window=0, scale=1.0, max_len=120)
    assert (got[:6] == 0).all() and (got[6:15] == 77).all() and (got[15:20] == 0).all()
    within(got[20:24], want[20:24], bound[20:24])
    assert (got[24:] == 77).all()                                    # rows 24..26 reach beyond the step's 26
    s["start"] = np.array([0, 6, 3, 3, 7, 10])                       # falling; the third has none
    s["lens"][:] = 60
    got = tree_attend(lg, dev, **s, most=64, n_head_kv=2, window=0, scale=1.0, max_len=120)
    assert (got[10:] == 77).all() and not (got[:3] == 77).any()


def test_pages_that_are_not_there_are_left_out(lg, dev):
    rng = np.random.default_rng(11)
    s = scene(rng, [100, 300, 20], [9, 16, 12], 8, 2, 64, 16)
    s["table"] = s["table"].copy()
    s["table"][0, [0, 3]], s["table"][1, [2, 19]], s["table"][2] = -1, 1 << 30, -7
    got = check(lg, dev, s, 2)
    assert (got[25:] == 0).all()
    check(lg, dev, s, 2, window=40)


@pytest.mark.parametrize("heads, kv, hd, most", [(8, 2, 64, 12), (8, 2, 256, 5), (8, 2, 256, 40), (8, 1, 512, 7), (8, 8, 128, 20)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_what_a_row_does_not_see_does_not_reach_it(lg, dev, heads, kv, hd, most, bad):
    """Rows behind the length and in pages of nobody, positions in front of a window, and rows of the tree that another row sees."""
    rng = np.random.default_rng(hd + most)
    s = scene(rng, [90, 0, 333], [most, most, most], heads, kv, hd, 16)
    page, table = 16, s["table"]
    window = 50
    good = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=window, scale=1.0, max_len=500)
    want, bound = tree_attend_ref(**s, page=page, n_pages=s["k"].shape[0], n_head_kv=kv, window=window, scale=1.0, max_len=500)
    within(good, want, bound)
    spoiled = 2                                                      # a row of each tree whose keys and values are bad
    rows_that_see = np.zeros(s["q"].shape[0], bool)
    s["k"], s["v"] = s["k"].copy(), s["v"].copy()
    held = set(table[table >= 0].tolist())
    for p in range(s["k"].shape[0]):
        if p not in held:
            s["k"][p] = s["v"][p] = bad
    for i in range(3):
        L = int(s["lens"][i])
        done = L - most
        for t in [*range(L, int(pages_of(L, page)) * page), *range(0, max(0, done - window + 1)), done + spoiled]:
            s["k"][table[i, t // page], t % page] = bad
            s["v"][table[i, t // page], t % page] = bad
        a = int(s["start"][i])
        for j in range(most):
            rows_that_see[a + j] = int(s["mask"][a + j]) >> spoiled & 1 and s["pos"][a + spoiled] > s["pos"][a + j] - window
    got = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=window, scale=1.0, max_len=500)
    assert rows_that_see.any() and not rows_that_see.all()
    assert np.array_equal(got[~rows_that_see], good[~rows_that_see])
    assert not np.isfinite(got[rows_that_see]).any()


def test_a_bad_value_alone_spoils_its_dimension(lg, dev):
    """Values of one key head that are not finite where the keys are: the dimensions of the heads that read them, in rows that see them."""
    rng = np.random.default_rng(12)
    s = scene(rng, [20], [8], 8, 2, 64, 16, "chain")
    t = 20 + 5
    s["v"] = s["v"].copy()
    s["v"][s["table"][0, t // 16], t % 16, 1, [3, 40]] = [np.inf, np.nan]
    got = tree_attend(lg, dev, **s, most=8, n_head_kv=2, window=0, scale=1.0, max_len=28)
    bad = np.zeros(got.shape, bool)
    for d in (3, 40):
        bad[5:, 4:, d] = True
    assert not np.isfinite(got[bad]).any() and np.isfinite(got[~bad]).all()


def test_a_bad_query_spoils_its_row(lg, dev):
    rng = np.random.default_rng(13)
    s = scene(rng, [70, 30], [8, 5], 8, 2, 64, 16)
    good = check(lg, dev, s, 2)
    s["q"] = s["q"].copy()
    s["q"][3, 2, 7] = np.nan
    s["q"][9, 5, 0] = np.inf
    got = tree_attend(lg, dev, **s, most=8, n_head_kv=2, window=0, scale=1.0, max_len=78)
    same = np.ones(got.shape[:2], bool)
    same[3, 2] = same[9, 5] = False
    assert np.array_equal(got[same], good[same]) and not np.isfinite(got[~same]).any()


def test_a_tree_of_one_row_is_a_new_token(lg, dev):
    """The same as lg_hip_paged_attention's sum, by a kernel of its own."""
    from serving import attend_ref
    rng = np.random.default_rng(14)
    s = scene(rng, [70, 0, 900], [1, 1, 1], 8, 2, 128, 32)
    got = check(lg, dev, s, 2, window=200)
    want, bound = attend_ref(s["q"], s["k"], s["v"], s["table"], s["lens"], 32, s["k"].shape[0], 2, 200, 1.0, 901)
    within(got, want, 2 * bound)


def test_a_long_cache_passes_32_bits(lg, dev):
    """Values further than 2^32 bytes into a pool: the last of its pages."""
    rng = np.random.default_rng(15)
    s = scene(rng, [40], [9], 8, 8, 256, 16)
    page, width = 16, 8 * 256
    n_pages = (1 << 32) // (page * width * 2) + 40
    import ctypes as C
    pools = [dev.room(n_pages * page * width * 2) for _ in range(2)]
    far = np.arange(4) + n_pages - 4
    for pool, x in zip(pools, (s["k"], s["v"])):
        for b, p in zip(s["table"][0, :4], far):
            dev.put(C.c_void_p(pool.value + int(p) * page * width * 2), x[b])
    table = s["table"].copy()
    table[0, :4] = far
    p = {n: dev.up(x) for n, x in dict(q=s["q"], table=table, lens=s["lens"].astype(np.int32), start=s["start"].astype(np.int32), mask=s["mask"], pos=s["pos"].astype(np.int32),
                                       out=np.zeros(s["q"].shape, np.float32)).items()}
    g = lg.hiplib.Pages(pools[0].value, pools[1].value, n_pages, page, 8, 256, width, width * page)
    need = dev.H.lg_hip_paged_tree_attention_workspace(1, 9, 8, 8, 256, 49, 0)
    dev.check(dev.H.lg_hip_paged_tree_attention(C.byref(g), p["q"], 2048, 9, 1, 9, 8, p["table"], table.shape[1], p["lens"], p["start"], p["mask"], p["pos"], 49, 0, 1.0, p["out"], 2048,
                                                dev.room(need), need, None), "paged_tree_attention")
    got = dev.back(p["out"], s["q"].shape, np.float32)
    dev.free()
    want, bound = tree_attend_ref(**s, page=16, n_pages=s["k"].shape[0], n_head_kv=8, window=0, scale=1.0, max_len=49)
    within(got, want, bound)
    assert bits([0, 2]) == 5
