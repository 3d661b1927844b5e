"""What calls of trees refuse before anything is launched, without a GPU."""
import ctypes as C

import pytest

from test_draft_refusals import RULES
from test_serving_refusals import P16, pages, refused

P32 = C.c_void_p(1 << 22)


@pytest.mark.parametrize("change, code, words", [
    (dict(n_seq=-1), -2, "-1 sequences"), (dict(n_seq=4097), -2, "4097 sequences"), (dict(most=0), -2, "up to 0 rows"), (dict(most=65), -2, "up to 65 rows"), (dict(rows=-1), -2, "-1 rows"),
    *((dict(null=k), -1, "tree_plan_from: null") for k in range(8)), (dict(grown=P16), -2, "in one place"), (dict(mask=C.c_void_p((1 << 20) + 4)), -2, "aligned")])
def test_tree_plans_from_earlier_lengths_refuse(lg, change, code, words):
    a = dict(n_seq=3, most=4, rows=9, null=None, grown=P32, mask=P16)
    a.update(change)
    p = [P16, P16, P16, a["grown"], a["mask"], P16, P16, P16]
    H = lg.hiplib.load_hip()
    refused(lg, H.lg_hip_tree_plan_from(a["n_seq"], a["most"], a["rows"], *(None if a["null"] == k else x for k, x in enumerate(p)), None), code, words)
    assert H.lg_hip_tree_plan_from(0, 4, 9, *[None] * 8, None) == 0


def attend(H, lg, seqs, heads, kv, most, max_len, hd=64):
    p = pages(lg, dict(n_head_kv=kv, head_dim=hd, row_stride=kv * hd, page_stride=kv * hd * 16))
    return H.lg_hip_paged_tree_attention(C.byref(p), P16, hd * heads, 9, seqs, most, heads, P16, 1 << 26, P16, P16, P16, P16, max_len, 0, 1.0, P16, hd * heads, P16, 1 << 62, None)


@pytest.mark.parametrize("below", [1, 20, 63])
def test_launches_are_counted_as_they_are_made(lg, below):
    """A call of 2^24 - below workgroups is launched in whole sixty-fours: 2^24, whose threads pass 32 bits.  Splits of 127 tiles in rounds of 768 workgroups, 2^24 - 256 of them, and one more for each sequence."""
    seqs = 256 - below
    tiles = (2 ** 24 - 256) * 127 // seqs
    assert tiles * seqs < 1 << 31
    refused(lg, attend(lg.hiplib.load_hip(), lg, seqs, 1, 1, 1, tiles * 32), -2, "in one call")


@pytest.mark.parametrize("seqs, heads, kv, most", [(3813, 4400, 550, 64), (2713, 6184, 773, 64)])
def test_launches_of_whole_trees_are_counted_as_they_are_made(lg, seqs, heads, kv, most):
    """2^24 - 16 and 2^24 - 24 workgroups of 64 pairs, and no joining launch."""
    refused(lg, attend(lg.hiplib.load_hip(), lg, seqs, heads, kv, most, 32), -2, "in one call")


@pytest.mark.parametrize("n", [(1 << 30) + 1, (1 << 31) - 1])
def test_more_biases_than_a_workgroup_counts_are_refused(lg, n):
    """Its threads count on behind the last one: near 2^31 past what 32 bits hold."""
    r = lg.hiplib.LogitRules(**{**RULES, "n_bias": n})
    refused(lg, lg.hiplib.load_hip().lg_hip_adjust_logits(C.byref(r), P16, 100, 3, 100, P32, 100, None), -2, "biases")
