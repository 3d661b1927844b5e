"""What calls of trees refuse before anything is launched, without a GPU."""
import ctypes as C

import pytest

from test_serving_refusals import P16, refused

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
