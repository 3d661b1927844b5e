"""The bound of tree attention's errors as a whole, without a GPU: the documented arithmetic keeps it by half, and arithmetic that has lost the second binary16 part of queries or probabilities passes it five times over."""
import numpy as np
import pytest

from drafts import tree_attend_ref
from test_gpu_trees import scene
from tree_errors import emulate, relative_rms, rms_tolerance


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [0, 60])
def test_what_the_bound_sees(hd, window):
    rng = np.random.default_rng(hd + window)
    s = scene(rng, [100, 0, 700], [9, 16, 5], 4, 1, hd, 16)
    want, _ = tree_attend_ref(**s, page=16, n_pages=s["k"].shape[0], n_head_kv=1, window=window, scale=1.0, max_len=1000)
    bound = rms_tolerance(2.0, hd, 705)
    off = {parts: relative_rms(emulate(s, 1, window, *parts), want) / bound for parts in ((2, 2), (1, 2), (2, 1), (1, 1))}
    assert off[2, 2] < 0.5, off
    assert min(off[1, 2], off[2, 1], off[1, 1]) > 5, off
