"""Attention of trees in each of its forms, which go by the room that a call is given (sequences, max_len) and not by the lengths it finds: small trees as a captured call over a large cache takes them."""
import ctypes as C

import numpy as np
import pytest

from drafts import tree_attend, tree_attend_ref
from serving import pages_of, within
from test_gpu_trees import check, dev, scene  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


def tiles_for(form, pairs, hd):
    """Tiles of a call's room, of all sequences and key heads, with which trees of so many pairs go to workgroups of 16, 32 or 64."""
    sixteens, sixties = -(-pairs // 16), -(-pairs // 64)
    few = (9216 if hd == 64 else 4608) // sixteens
    return {16: 1, 32: few + few // 20 + 8, 64: max(few, 2560 // sixties) + 3000}[form]


FORMS = [(16, 8, 2, 64, 64), (16, 8, 1, 512, 9), (16, 8, 2, 256, 64), (32, 8, 2, 64, 30), (32, 8, 2, 64, 8), (32, 8, 4, 128, 64), (32, 5, 1, 128, 5), (32, 8, 2, 256, 16), (32, 16, 8, 256, 16), (32, 8, 2, 256, 61),
         (32, 8, 1, 512, 4), (32, 2, 2, 512, 23), (64, 8, 2, 64, 64), (64, 8, 2, 64, 11), (64, 8, 2, 128, 23), (64, 8, 1, 128, 5), (64, 8, 2, 256, 16), (64, 8, 1, 256, 37), (64, 8, 1, 512, 64), (64, 2, 2, 512, 40)]


def room_of(form, n, heads, kv, hd, most):
    return 32 * -(-tiles_for(form, most * (heads // kv), hd) // (n * kv))


def with_empty(x, n):
    """A list of counts with sequences of nothing behind it, up to n of them."""
    return list(x) + [0] * (n - len(x))


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS)
def test_in_splits(lg, dev, form, heads, kv, hd, most):
    rng = np.random.default_rng(form + hd + most)
    committed, sizes = [0, 1, 15, 33, 1200, 500], [most, max(1, most - 1), 1, most, (most + 1) // 2, most]
    s = scene(rng, committed, sizes, heads, kv, hd, 16)
    check(lg, dev, s, kv, most=most, max_len=max(int(s["lens"].max()), room_of(form, 6, heads, kv, hd, most)), pad=4 if most & 1 else 0)


@pytest.mark.parametrize("form, heads, kv, hd, most", [x for x in FORMS if x[0] > 16])
def test_whole(lg, dev, form, heads, kv, hd, most):
    """Many sequences, most of them empty, so short that none is split."""
    rng = np.random.default_rng(form + hd + most)
    n = -(-tiles_for(form, most * (heads // kv), hd) // (8 * kv))
    check(lg, dev, scene(rng, with_empty([0, 1, 15, 33, 120, 190], n), with_empty([most, 1, max(1, most - 1), most, (most + 1) // 2, most], n), heads, kv, hd, 32), kv, most=most, max_len=256)


@pytest.mark.parametrize("form, heads, kv, hd, most", [x for x in FORMS if x[0] > 16])
@pytest.mark.parametrize("window", [1, 30, 100])
def test_windows(lg, dev, form, heads, kv, hd, most, window):
    rng = np.random.default_rng(form + hd + most)
    n = -(-tiles_for(form, most * (heads // kv), hd) // ((window + most + 32 + 31) // 32 * kv))
    n = min(n, 4096)
    s = scene(rng, with_empty([0, 5, 40, 300, 1500], n), with_empty([most, max(1, most // 2), most, 1, most], n), heads, kv, hd, 16, "any" if most & 1 else "chain")
    check(lg, dev, s, kv, most=most, window=window)


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS)
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_what_is_not_seen(lg, dev, form, heads, kv, hd, most, bad):
    """Bad keys and values behind the lengths, in pages of nobody and in one row of each tree: rows that do not see that one come out as before, to the bit."""
    rng = np.random.default_rng(form + hd + most)
    page, spoiled = 16, 2
    s = scene(rng, [90, 0, 433], [most] * 3, heads, kv, hd, page)
    room = max(433 + most, room_of(form, 3, heads, kv, hd, most))
    good = check(lg, dev, s, kv, most=most, max_len=room)
    s["k"], s["v"] = s["k"].copy(), s["v"].copy()
    held = set(s["table"][s["table"] >= 0].tolist())
    for p in set(range(s["k"].shape[0])) - held:
        s["k"][p] = s["v"][p] = bad
    sees = np.zeros(s["q"].shape[0], bool)
    for i in range(3):
        L, a = int(s["lens"][i]), int(s["start"][i])
        for t in [*range(L, int(pages_of(L, page)) * page), L - most + spoiled]:
            s["k"][s["table"][i, t // page], t % page] = s["v"][s["table"][i, t // page], t % page] = bad
        sees[a:a + most] = s["mask"][a:a + most].astype(np.uint64) >> np.uint64(spoiled) & np.uint64(1) == 1
    got = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=0, scale=1.0, max_len=room)
    assert sees.any() and not sees.all()
    assert np.array_equal(got[~sees], good[~sees]) and not np.isfinite(got[sees]).any()


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS)
def test_pages_and_positions_that_are_not_there(lg, dev, form, heads, kv, hd, most):
    rng = np.random.default_rng(form + hd + most)
    s = scene(rng, [100, 300, 20, 640], [most, 1, most, most], heads, kv, hd, 16)
    s["table"], s["pos"], s["mask"] = s["table"].copy(), s["pos"].copy(), s["mask"].copy()
    s["table"][0, [0, 3]], s["table"][1, [2, 18]], s["table"][2], s["table"][3, [7, 31]] = -1, 1 << 30, -7, -1
    s["pos"][1] = -1                                                 # a row without a position, and one that names rows of which its tree has some
    s["mask"][-1] = (1 << 64) - 1
    room = max(700, room_of(form, 4, heads, kv, hd, most))
    got = check(lg, dev, s, kv, most=most, max_len=room)
    assert (got[1] == 0).all() and (got[most + 1:2 * most + 1] == 0).all()
    # sequences that do not fit: zeros
    s["lens"] = s["lens"].copy()
    s["lens"][0], s["lens"][3] = most - 1, 1 << 30
    got = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=0, scale=1.0, max_len=room)
    want, bound = tree_attend_ref(**s, page=16, n_pages=s["k"].shape[0], n_head_kv=kv, window=0, scale=1.0, max_len=room)
    within(got, want, bound)
    assert (got[:most] == 0).all() and (got[-most:] == 0).all()


def put_scene(dev, s, H, hd, pad=0):
    """Its arrays on the device, those of a call in their types; outputs of 77."""
    out = np.full((s["q"].shape[0], H * hd + pad), 77, np.float32)
    return {n: dev.up(x) for n, x in dict(q=s["q"], table=s["table"].astype(np.int32), lens=np.asarray(s["lens"], np.int32), start=np.asarray(s["start"], np.int32), mask=np.asarray(s["mask"], np.uint64),
                                          pos=np.asarray(s["pos"], np.int32), out=out).items()}


def call(dev, g, p, s, heads, most, max_len, window, work, need, stream=None):
    n, rows, qd = len(s["lens"]), s["q"].shape[0], heads * g.head_dim
    return dev.H.lg_hip_paged_tree_attention(C.byref(g), p["q"], qd, rows, n, most, heads, p["table"], s["table"].shape[1], p["lens"], p["start"], p["mask"], p["pos"], max_len, window, 1.0,
                                             p["out"], qd, work, need, stream)


@pytest.mark.parametrize("form, heads, kv, hd, most", [x for x in FORMS if x[4] < 64])
def test_keys_and_values_in_turn_in_one_array(lg, dev, form, heads, kv, hd, most):
    """Rows of K and V next to each other, and room between rows and between pages."""
    rng = np.random.default_rng(form + hd + most)
    page, width = 32, kv * hd
    s = scene(rng, [77, 0, 500], [most, most, 1], heads, kv, hd, page)
    n_pages, row = s["k"].shape[0], 2 * width + 24
    pool = rng.integers(0, 1 << 16, (n_pages, page + 3, row)).astype(np.uint16)          # NaN and infinities among them
    pool[:, :page, :width], pool[:, :page, width:2 * width] = s["k"].reshape(n_pages, page, -1).view(np.uint16), s["v"].reshape(n_pages, page, -1).view(np.uint16)
    kv_at, p = dev.up(pool), put_scene(dev, s, heads, hd)
    g = lg.hiplib.Pages(kv_at.value, kv_at.value + 2 * width, n_pages, page, kv, hd, row, row * (page + 3))
    room = max(501 + most, room_of(form, 3, heads, kv, hd, most))
    need = dev.H.lg_hip_paged_tree_attention_workspace(3, most, heads, kv, hd, room, 0)
    dev.check(call(dev, g, p, s, heads, most, room, 0, dev.room(need), need), "paged_tree_attention")
    got = dev.back(p["out"], s["q"].shape, np.float32)
    dev.free()
    want, bound = tree_attend_ref(**s, page=page, n_pages=n_pages, n_head_kv=kv, window=0, scale=1.0, max_len=room)
    within(got, want, bound)


@pytest.mark.parametrize("form, heads, kv, hd, most", [(16, 8, 2, 64, 4), (32, 8, 2, 256, 16), (64, 8, 2, 64, 20), (64, 8, 1, 512, 9)])
def test_rows_as_far_apart_as_they_may_be(lg, dev, form, heads, kv, hd, most):
    """2^27 values between rows, so that a page's last row begins 4 GiB behind its first (K and V share the array)."""
    rng = np.random.default_rng(form + hd)
    page, width, row = 16, kv * hd, 1 << 27
    s = scene(rng, [11], [most], heads, kv, hd, page, spare=0)
    n_pages = s["k"].shape[0]
    length = int(s["lens"][0])
    pool = dev.room((n_pages * page - 1) * row * 2 + 4 * width)
    for t in range(length):
        b = int(s["table"][0, t // page])
        for at, x in ((0, s["k"]), (2 * width, s["v"])):
            dev.put(C.c_void_p(pool.value + (b * page + t % page) * row * 2 + at), x[b, t % page])
    p, room = put_scene(dev, s, heads, hd), max(length, room_of(form, 1, heads, kv, hd, most))
    g = lg.hiplib.Pages(pool.value, pool.value + 2 * width, n_pages, page, kv, hd, row, row * page)
    need = dev.H.lg_hip_paged_tree_attention_workspace(1, most, heads, kv, hd, room, 0)
    dev.check(call(dev, g, p, s, heads, most, room, 0, dev.room(need), need), "paged_tree_attention")
    got = dev.back(p["out"], s["q"].shape, np.float32)
    dev.free()
    want, bound = tree_attend_ref(**s, page=page, n_pages=n_pages, n_head_kv=kv, window=0, scale=1.0, max_len=room)
    within(got, want, bound)


@pytest.mark.parametrize("n", [5, 90])
@pytest.mark.parametrize("form, heads, kv, hd, most", [(16, 8, 2, 64, 9), (32, 8, 2, 256, 16), (64, 8, 2, 128, 23)])
def test_one_recorded_call_for_all_lengths(lg, dev, form, heads, kv, hd, most, n):
    """Recorded once, with room for rows behind the last tree; between replays other trees, lengths, pages and queries are put in place, and an eager call with memory of its own runs."""
    rt, page = dev.rt, 16
    rng = np.random.default_rng(form + n)

    def draw():
        sizes = rng.integers(0, most + 1, n)
        sizes[0] = most
        return scene(rng, (700 * rng.random(n) ** 4).astype(np.int64), sizes, heads, kv, hd, page, blocks=50)
    scenes = [draw() for _ in range(4)]
    rows, n_pages = max(x["q"].shape[0] for x in scenes), max(x["k"].shape[0] for x in scenes)
    room = max(720 + most, room_of(form, n, heads, kv, hd, most))
    need = dev.H.lg_hip_paged_tree_attention_workspace(n, most, heads, kv, hd, room, 0)
    wide = lambda x, m: np.concatenate([x, np.zeros((m - x.shape[0],) + x.shape[1:], x.dtype)])          # noqa: E731
    for x in scenes:
        x.update(q=wide(x["q"], rows), mask=wide(np.asarray(x["mask"], np.uint64), rows), pos=wide(np.asarray(x["pos"], np.int32), rows), k=wide(x["k"], n_pages), v=wide(x["v"], n_pages))
    k, v = dev.up(scenes[0]["k"]), dev.up(scenes[0]["v"])
    p = put_scene(dev, scenes[0], heads, hd)
    g = lg.hiplib.Pages(k.value, v.value, n_pages, page, kv, hd, kv * hd, kv * hd * page)
    work, own = dev.room(need), dev.room(need)
    stream, graph, gexec = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert rt.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    rt.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    rt.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    assert rt.hipDeviceSynchronize() == 0 and rt.hipStreamBeginCapture(stream, 0) == 0
    try:
        rc = call(dev, g, p, scenes[0], heads, most, room, 0, work, need, stream)
    finally:
        end = rt.hipStreamEndCapture(stream, C.byref(graph))
    assert rc == 0 and end == 0 and rt.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
    for replay, s in enumerate(scenes + scenes[:1]):
        for name in ("q", "table", "lens", "start", "mask", "pos"):
            dev.put(p[name], np.asarray(s[name], dict(q=np.float32, mask=np.uint64).get(name, np.int32)))
        dev.put(k, s["k"]), dev.put(v, s["v"]), dev.put(p["out"], np.full((rows, heads * hd), 77, np.float32))
        assert rt.hipDeviceSynchronize() == 0
        print(f"replay {replay}", flush=True)
        assert rt.hipGraphLaunch(gexec, stream) == 0 and rt.hipStreamSynchronize(stream) == 0
        got = dev.back(p["out"], s["q"].shape, np.float32)
        dev.put(p["out"], np.full((rows, heads * hd), 77, np.float32))
        dev.check(call(dev, g, p, s, heads, most, room, 0, own, need), "paged_tree_attention")
        assert np.array_equal(got, dev.back(p["out"], s["q"].shape, np.float32))
        last = int(s["start"][-1])
        want, bound = tree_attend_ref(**s, page=page, n_pages=n_pages, n_head_kv=kv, window=0, scale=1.0, max_len=room)
        within(got[:last], want[:last], bound[:last], f"replay {replay}")
        assert (got[last:] == 77).all()
    rt.hipGraphExecDestroy.argtypes = rt.hipGraphDestroy.argtypes = rt.hipStreamDestroy.argtypes = [C.c_void_p]
    rt.hipGraphExecDestroy(gexec), rt.hipGraphDestroy(graph), rt.hipStreamDestroy(stream)
    dev.free()


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS)
def test_scores_that_rise_all_the_way(lg, dev, form, heads, kv, hd, most):
    """A new maximum in nearly every tile, in some rows only."""
    rng = np.random.default_rng(form + hd + most)
    page = 16
    s = scene(rng, [700, 0, 300], [most, most, 1], heads, kv, hd, page)
    s["k"], s["q"] = s["k"].astype(np.float32), np.abs(s["q"])
    s["q"][::3] *= -1
    for i in range(3):
        for b in range(int(pages_of(s["lens"][i], page))):
            s["k"][s["table"][i, b]] = np.abs(s["k"][s["table"][i, b]]) * (0.02 + 0.05 * b)
    s["k"] = s["k"].astype(np.float16)
    check(lg, dev, s, kv, most=most, max_len=max(700 + most, room_of(form, 3, heads, kv, hd, most)))
    check(lg, dev, s, kv, most=most, max_len=max(700 + most, room_of(form, 3, heads, kv, hd, most)), scale=-1.0)
