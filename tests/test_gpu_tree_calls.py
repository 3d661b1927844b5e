"""Calls of tree attention that stand apart from the others: the largest batches, scores far from one another, and the same rows by lg_hip_paged_attention."""
import numpy as np
import pytest

from test_gpu_tree_forms import with_empty
from test_gpu_trees import check, dev, scene  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 256])
def test_the_most_sequences_of_the_largest_trees_that_are_left_whole(lg, dev, hd):
    """4096 sequences with room for trees of 64 rows of 64 heads, most of them empty: nothing is joined, so that no joining launch has to hold all their rows."""
    rng = np.random.default_rng(hd)
    s = scene(rng, with_empty([0, 1, 12, 17], 4096), with_empty([20, 1, 20, 15], 4096), 64, 8, hd, 16)
    assert dev.H.lg_hip_paged_tree_attention_workspace(4096, 64, 64, 8, hd, 32, 0) == 0
    check(lg, dev, s, 8, most=64, max_len=32)
