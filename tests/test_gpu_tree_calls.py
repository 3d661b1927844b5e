"""Calls of tree attention that stand apart from the others: the largest batches, scores far from one another, and the same rows by lg_hip_paged_attention."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_tree_forms as forms
from drafts import tolerance, tree_attend, tree_attend_ref
from serving import attend_ref, within
from test_gpu_tree_forms import FORMS, room_of, with_empty
from test_gpu_trees import check, dev, scene  # noqa: F401  (dev: the fixture)
from tree_errors import relative_rms, rms_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 256])
def test_the_most_sequences_of_the_largest_trees_that_are_left_whole(lg, dev, hd):
    """4096 sequences with room for trees of 64 rows of 64 heads, most of them empty: nothing is joined, so that no joining launch has to hold all their rows."""
    rng = np.random.default_rng(hd)
    s = scene(rng, with_empty([0, 1, 12, 17], 4096), with_empty([20, 1, 20, 15], 4096), 64, 8, hd, 16)
    assert dev.H.lg_hip_paged_tree_attention_workspace(4096, 64, 64, 8, hd, 32, 0) == 0
    check(lg, dev, s, 8, most=64, max_len=32)


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS)
def test_scores_that_f32_holds_in_steps_of_sixteen(lg, dev, form, heads, kv, hd, most):
    """Scores of 2^25 to 2^30, of either sign, in whole steps of a row's own that no rounding bridges: the keys of the largest one share the row evenly.  Their scores are equal to the bit, so of the
    tolerance only what does not go by the scores' size is left."""
    rng = np.random.default_rng(form + hd + most)
    s = scene(rng, [90, 0, 433], [most, most, 1], heads, kv, hd, 16)
    sign = rng.choice([-1.0, 1.0], hd)
    s["k"] = (rng.integers(1, 5, s["k"].shape[:3] + (1,)) * sign).astype(np.float16)
    step = 2.0 ** rng.uniform(23, 28, s["q"].shape[:2]) * rng.choice([-1, 1], s["q"].shape[:2])
    s["q"] = np.float32(step / hd)[..., None] * sign.astype(np.float32)
    room = max(433 + most, room_of(form, 3, heads, kv, hd, most))
    got = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=0, scale=1.0, max_len=room)
    want, _ = tree_attend_ref(**s, page=16, n_pages=s["k"].shape[0], n_head_kv=kv, window=0, scale=1.0, max_len=room)
    within(got, want, tolerance(0.0, hd, 433 + most) * float(np.abs(s["v"]).max()))


def attend(lg, dev, s, kv, window, max_len):
    """lg_hip_paged_attention of the same rows, a sequence each."""
    n, H, hd = s["q"].shape
    n_pages, page = s["k"].shape[:2]
    p = {x: dev.up(s[x]) for x in ("q", "k", "v")}
    table, lens, out = dev.up(s["table"], np.int32), dev.up(s["lens"], np.int32), dev.up(np.full(s["q"].shape, np.nan, np.float32))
    g = lg.hiplib.Pages(p["k"].value, p["v"].value, n_pages, page, kv, hd, kv * hd, kv * hd * page)
    need = dev.H.lg_hip_paged_attention_workspace(n, H, kv, hd, max_len, window)
    dev.check(dev.H.lg_hip_paged_attention(C.byref(g), p["q"], H * hd, n, H, table, s["table"].shape[1], lens, max_len, window, 1.0, out, H * hd, dev.room(need), need, None), "paged_attention")
    got = dev.back(out, s["q"].shape, np.float32)
    dev.free()
    return got


@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 64), (8, 2, 128), (8, 2, 256), (16, 8, 256), (8, 1, 512)])
@pytest.mark.parametrize("window", [0, 1, 200])
def test_a_tree_of_one_row_gives_what_a_new_token_gives(lg, dev, heads, kv, hd, window):
    """By lg_hip_paged_tree_attention and by lg_hip_paged_attention, over the same pages: each within its own bound of the same value, and as a whole within both."""
    rng = np.random.default_rng(hd + window)
    s = scene(rng, [70, 0, 900, 31, 1999], [1] * 5, heads, kv, hd, 32)
    tree, token = check(lg, dev, s, kv, window=window), attend(lg, dev, s, kv, window, 2000)
    want, bound = attend_ref(s["q"], s["k"], s["v"], s["table"], s["lens"], 32, s["k"].shape[0], kv, window, 1.0, 2000)
    within(token, want, bound)
    within(tree, token, 3 * bound)
    assert relative_rms(tree, token) <= 2 * rms_tolerance(2.0, hd, 2000)


def test_rows_of_sound_trees_beside_starts_that_fall(lg, dev):
    """The first and the last trees are as they are alone; rows that two trees claim belong to neither."""
    rng = np.random.default_rng(10)
    s = scene(rng, [40, 50, 60, 70, 80], [6, 9, 5, 4, 3], 8, 2, 64, 16)
    s["start"], s["lens"] = np.array([0, 6, 3, 3, 7, 10]), np.array([46, 59, 65, 74, 40])
    got = tree_attend(lg, dev, **s, most=64, n_head_kv=2, window=0, scale=1.0, max_len=120)
    want, bound = tree_attend_ref(**s, page=16, n_pages=s["k"].shape[0], n_head_kv=2, window=0, scale=1.0, max_len=120)
    for rows in (slice(0, 3), slice(7, 10)):
        within(got[rows], want[rows], bound[rows])
        assert (np.abs(want[rows]).max((1, 2)) > 0).all()
    assert (got[10:] == 77).all()


@pytest.mark.parametrize("heads, kv, hd, most", [(8, 2, 256, 64), (8, 2, 64, 33), (8, 2, 128, 20)])
def test_many_pairs_in_workgroups_of_sixteen(lg, dev, heads, kv, hd, most):
    """Trees of more than 16 pairs where there is little to read, in splits."""
    rng = np.random.default_rng(hd + most)
    assert dev.H.lg_hip_paged_tree_attention_pairs(3, most, heads, kv, hd, 680, 0) == 16 and dev.H.lg_hip_paged_tree_attention_workspace(3, most, heads, kv, hd, 680, 0)
    check(lg, dev, scene(rng, [600, 0, 333], [most, max(1, most - 1), most], heads, kv, hd, 16), kv, most=most, max_len=680)


@pytest.mark.parametrize("form, heads, kv, hd, most", [(16, 8, 2, 64, 4), (16, 8, 2, 256, 3), (32, 8, 2, 256, 8), (32, 8, 2, 64, 7)])
def test_one_recorded_call_of_many_sequences_and_few_pairs(lg, dev, form, heads, kv, hd, most):
    """90 sequences, recorded and replayed with others, in workgroups of 16 and 32 pairs."""
    assert dev.H.lg_hip_paged_tree_attention_pairs(90, most, heads, kv, hd, max(720 + most, room_of(form, 90, heads, kv, hd, most)), 0) == form
    forms.test_one_recorded_call_for_all_lengths(lg, dev, form, heads, kv, hd, most, 90)
