"""Which kernel a call of tree attention takes, without a GPU: the tests of its forms call the forms that they name."""
import pytest

from test_gpu_tree_forms import FORMS, room_of, tiles_for

# calls of tests/test_gpu_tree_forms.py whose floor under max_len takes another form than their name says: tests/test_gpu_tree_calls.py has calls of the form itself
OTHERS = {(16, 8, 2, 256, 64, 6): 32, (16, 8, 2, 64, 9, 90): 64, (32, 8, 2, 256, 16, 90): 64}
RECORDED = [(16, 8, 2, 64, 9), (32, 8, 2, 256, 16), (64, 8, 2, 128, 23)]
FAR_APART = [(16, 8, 2, 64, 4), (32, 8, 2, 256, 16), (64, 8, 2, 64, 20), (64, 8, 1, 512, 9)]


def pairs(lg, n, most, heads, kv, hd, max_len, window=0):
    return lg.hiplib.load_hip().lg_hip_paged_tree_attention_pairs(n, most, heads, kv, hd, max_len, window)


def named(lg, form, heads, kv, hd, most, n, least):
    got = pairs(lg, n, most, heads, kv, hd, max(least, room_of(form, n, heads, kv, hd, most)))
    assert got == OTHERS.get((form, heads, kv, hd, most, n), form), (n, least, got)


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS)
def test_calls_in_splits(lg, form, heads, kv, hd, most):
    for n, least in ((6, 1200 + (most + 1) // 2), (3, 433 + most), (4, 700), (3, 501 + most), (3, 700 + most)):
        named(lg, form, heads, kv, hd, most, n, least)


def test_recorded_calls_and_rows_far_apart(lg):
    for x in RECORDED:
        named(lg, *x, 5, 720 + x[4])
        named(lg, *x, 90, 720 + x[4])
    for x in FAR_APART:
        named(lg, *x, 1, 11 + x[4])


@pytest.mark.parametrize("form, heads, kv, hd, most", [x for x in FORMS if x[0] > 16])
def test_calls_left_whole(lg, form, heads, kv, hd, most):
    tiles = tiles_for(form, most * (heads // kv), hd)
    assert pairs(lg, -(-tiles // (8 * kv)), most, heads, kv, hd, 256) == form
    for window in (1, 30, 100):
        n = min(4096, -(-tiles // ((window + most + 63) // 32 * kv)))
        assert pairs(lg, n, most, heads, kv, hd, 1500 + most, window) == form, window


@pytest.mark.parametrize("args", [(-1, 4, 8, 2, 64, 100, 0), (3, 0, 8, 2, 64, 100, 0), (3, 65, 8, 2, 64, 100, 0), (3, 4, 7, 2, 64, 100, 0), (3, 4, 8, 2, 65, 100, 0), (3, 4, 8, 2, 64, -1, 0), (3, 4, 8, 2, 64, 100, -1)])
def test_calls_that_are_refused_take_none(lg, args):
    assert lg.hiplib.load_hip().lg_hip_paged_tree_attention_pairs(*args) == 0
