"""Attention of trees in each of its forms, which go by the room that a call is given (sequences, max_len) and not by the lengths it finds: small trees as a captured call over a large cache takes them."""
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
