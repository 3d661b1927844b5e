"""Calls of tree attention that stand apart from the others: the largest batches, scores far from one another, and the same rows by lg_hip_paged_attention."""
import numpy as np
import pytest

from drafts import tolerance, tree_attend, tree_attend_ref
from serving import within
from test_gpu_tree_forms import FORMS, room_of, with_empty
from test_gpu_trees import check, dev, scene  # noqa: F401  (dev: the fixture)

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
