"""Errors of tree attention as a whole, for every head size and all three sizes of workgroups: the second binary16 parts of queries and probabilities are there."""
import numpy as np
import pytest

from drafts import tree_attend, tree_attend_ref
from test_gpu_tree_forms import FORMS, room_of, tiles_for, with_empty
from test_gpu_trees import dev, scene  # noqa: F401  (dev: the fixture)
from tree_errors import relative_rms, rms_tolerance

pytestmark = pytest.mark.gpu


def small(lg, dev, s, kv, most, max_len, window=0):
    got = tree_attend(lg, dev, **s, most=most, n_head_kv=kv, window=window, scale=1.0, max_len=max_len)
    want, _ = tree_attend_ref(**s, page=s["k"].shape[1], n_pages=s["k"].shape[0], n_head_kv=kv, window=window, scale=1.0, max_len=max_len)
    off, bound = relative_rms(got, want), rms_tolerance(2.0, s["q"].shape[2], int(s["lens"].max()))
    print(f"relative error {off:.3g}, {off / bound:.3g} of the bound", flush=True)
    assert off <= bound


@pytest.mark.parametrize("form, heads, kv, hd, most", FORMS + [(16, 8, 2, 128, 7)])
def test_in_splits(lg, dev, form, heads, kv, hd, most):
    rng = np.random.default_rng(form + hd + most)
    s = scene(rng, [100, 0, 600 if form == 16 else 1200, 33, 500], [most, max(1, most - 1), most, 1, most], heads, kv, hd, 16)
    room = max(int(s["lens"].max()), room_of(form, 5, heads, kv, hd, most))
    assert dev.H.lg_hip_paged_tree_attention_pairs(5, most, heads, kv, hd, room, 0) == form
    small(lg, dev, s, kv, most, room)


@pytest.mark.parametrize("form, heads, kv, hd, most", [x for x in FORMS if x[0] > 16])
@pytest.mark.parametrize("window", [0, 100])
def test_whole(lg, dev, form, heads, kv, hd, most, window):
    rng = np.random.default_rng(form + hd + most)
    n = min(4096, -(-tiles_for(form, most * (heads // kv), hd) // ((window + most + 63) // 32 * kv if window else 8 * kv)))
    s = scene(rng, with_empty([0, 40, 120, 190 if not window else 1500], n), with_empty([most, most, 1, most], n), heads, kv, hd, 16)
    room = int(s["lens"].max()) if window else 256
    assert dev.H.lg_hip_paged_tree_attention_pairs(n, most, heads, kv, hd, room, window) == form
    small(lg, dev, s, kv, most, room, window)
