"""What the operators around trees, shared pages and rules refuse before anything is launched: no GPU is needed (a call that got past its checks would fail otherwise on a machine without one)."""
import ctypes as C

import pytest

from test_serving_refusals import BAD_PAGES, P16, pages, refused


def tree_args(**change):
    a = dict(n_seq=3, most=4, rows=9, start=P16, parent=P16, len=P16, a=P16, b=P16, c=P16, d=P16, e=P16, f=P16)
    a.update(change)
    return a


@pytest.mark.parametrize("change, code, words", [
    (dict(n_seq=-1), -2, "-1 sequences"), (dict(n_seq=4097), -2, "4097 sequences"), (dict(most=0), -2, "up to 0 rows"), (dict(most=65), -2, "up to 65 rows"), (dict(rows=-1), -2, "-1 rows"),
    (dict(start=None), -1, "null"), (dict(parent=None), -1, "null"), (dict(len=None), -1, "null"), (dict(a=None), -1, "null"), (dict(b=None), -1, "null"), (dict(c=None), -1, "null"), (dict(d=None), -1, "null")])
def test_tree_calls_refuse(lg, change, code, words):
    H, a = lg.hiplib.load_hip(), tree_args(**change)
    refused(lg, H.lg_hip_tree_plan(a["n_seq"], a["most"], a["rows"], a["start"], a["parent"], a["len"], a["a"], a["b"], a["c"], a["d"], None), code, "tree_plan" if code == -1 else words)
    refused(lg, H.lg_hip_tree_accept(a["n_seq"], a["most"], a["rows"], a["start"], a["parent"], a["a"], a["b"], a["len"], a["c"], a["d"], a["e"], a["f"], None), code, words)


def test_tree_plan_refuses_sets_that_are_not_aligned(lg):
    H = lg.hiplib.load_hip()
    refused(lg, H.lg_hip_tree_plan(3, 4, 9, P16, P16, P16, C.c_void_p((1 << 20) + 4), P16, P16, P16, None), -2, "aligned")
    for bad in range(2):
        outs = [P16] * 4
        outs[2 + bad] = None
        refused(lg, H.lg_hip_tree_accept(3, 4, 9, P16, P16, P16, P16, P16, *outs, None), -1, "null")


def attend(H, p, **change):
    a = dict(q=P16, q_stride=512, rows=9, n_seq=3, most=16, heads=8, table=P16, blocks=1024, lens=P16, start=P16, mask=P16, pos=P16, max_len=8192, window=0, out=P16, out_stride=512, work=P16, short=0)
    a.update(change)
    need = H.lg_hip_paged_tree_attention_workspace(3, 16, 8, 2, 64, 8192, 0)
    assert need > 0
    return H.lg_hip_paged_tree_attention(C.byref(p), a["q"], a["q_stride"], a["rows"], a["n_seq"], a["most"], a["heads"], a["table"], a["blocks"], a["lens"], a["start"], a["mask"], a["pos"],
                                         a["max_len"], a["window"], 1.0, a["out"], a["out_stride"], a["work"], need - a["short"], None)


@pytest.mark.parametrize("change, code, words", [
    (dict(n_seq=-1), -2, "-1 sequences"), (dict(n_seq=4097), -2, "4097 sequences"), (dict(most=0), -2, "up to 0 rows"), (dict(most=65), -2, "up to 65 rows"), (dict(rows=-1), -2, "-1 rows"),
    (dict(heads=7), -2, "7 query heads"), (dict(heads=18), -2, "18 query heads"), (dict(heads=0), -2, "0 query heads"), (dict(max_len=-1), -2, "lengths up to -1"),
    (dict(max_len=(1 << 30) + 1), -2, "lengths up to"), (dict(blocks=0), -2, "0 blocks"), (dict(blocks=1 << 27), -2, "blocks"), (dict(window=-5), -2, "window"), (dict(q=None), -1, "null"),
    (dict(table=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(start=None), -1, "null"), (dict(mask=None), -1, "null"), (dict(pos=None), -1, "null"), (dict(out=None), -1, "null"),
    (dict(q_stride=508), -2, "508 apart"), (dict(q_stride=513), -2, "513 apart"), (dict(out_stride=511), -2, "511 apart"), (dict(q=C.c_void_p((1 << 20) + 8)), -2, "aligned"),
    (dict(out=C.c_void_p((1 << 20) + 2)), -2, "output rows"), (dict(mask=C.c_void_p((1 << 20) + 4)), -2, "sets"), (dict(work=None), -2, "working memory"), (dict(short=1), -2, "working memory"),
    (dict(work=C.c_void_p((1 << 20) + 16)), -2, "working memory")])
def test_tree_attention_refuses(lg, change, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, {})
    refused(lg, attend(H, p, **change), code, words)
    assert attend(H, p, n_seq=0) == 0 and attend(H, p, rows=0) == 0


@pytest.mark.parametrize("change, code, words", BAD_PAGES)
def test_bad_pages_are_refused(lg, change, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, change)
    refused(lg, attend(H, p), code, words)
    two = (lg.hiplib.Pages * 2)(pages(lg, {}), p)
    refused(lg, H.lg_hip_paged_compact(two, 2, 3, 4, P16, 4, P16, P16, P16, P16, None), code, words)
    refused(lg, H.lg_hip_paged_copy(two, 2, 3, P16, P16, P16, None), code, words)


def test_rows_too_far_apart_for_tree_attention_are_refused(lg):
    H, far = lg.hiplib.load_hip(), (1 << 27) + 8
    refused(lg, attend(H, pages(lg, dict(row_stride=far, page_stride=far * 16))), -2, "at most 2^27")
    assert attend(H, pages(lg, dict(row_stride=1 << 27, page_stride=1 << 31)), rows=0) == 0


def test_calls_beyond_what_a_launch_holds_are_refused(lg):
    H = lg.hiplib.load_hip()
    for seqs, heads, kv, most in ((4096, 2, 1, 1), (128, 2, 1, 64), (4096, 1024, 128, 64)):
        p = pages(lg, dict(n_head_kv=kv, row_stride=kv * 64, page_stride=kv * 1024))
        rc = H.lg_hip_paged_tree_attention(C.byref(p), P16, 64 * heads, 9, seqs, most, heads, P16, 1 << 26, P16, P16, P16, P16, 1 << 30, 0, 1.0, P16, 64 * heads, P16, 1 << 62, None)
        refused(lg, rc, -2, "in one call")


@pytest.mark.parametrize("args", [(-1, 4, 8, 2, 64, 100, 0), (3, 0, 8, 2, 64, 100, 0), (3, 65, 8, 2, 64, 100, 0), (3, 4, 7, 2, 64, 100, 0), (3, 4, 8, 2, 65, 100, 0), (3, 4, 8, 2, 64, -1, 0), (3, 4, 8, 2, 64, 100, -1)])
def test_workspaces_of_calls_that_are_refused_are_nothing(lg, args):
    assert lg.hiplib.load_hip().lg_hip_paged_tree_attention_workspace(*args) == 0


@pytest.mark.parametrize("layers, n_seq, most, blocks, null, code, words", [
    (-1, 3, 4, 4, None, -2, "-1 layers"), (1, -1, 4, 4, None, -2, "-1 sequences"), (1, 4097, 4, 4, None, -2, "4097 sequences"), (1, 3, 0, 4, None, -2, "up to 0 rows"), (1, 3, 65, 4, None, -2, "up to 65"),
    (1, 3, 4, 0, None, -2, "0 blocks"), (1, 3, 4, 1 << 27, None, -2, "blocks"), *((1, 3, 4, 4, k, -1, "null") for k in range(5))])
def test_compact_refuses(lg, layers, n_seq, most, blocks, null, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, {})
    a = [None if null == k else P16 for k in range(5)]
    refused(lg, H.lg_hip_paged_compact(C.byref(p), layers, n_seq, most, a[0], blocks, *a[1:], None), code, words)
    refused(lg, H.lg_hip_paged_compact(None, 1, 3, 4, P16, 4, P16, P16, P16, P16, None), -1, "null")


def test_layers_of_one_table_are_alike_in_pages(lg):
    H = lg.hiplib.load_hip()
    for change in (dict(n_pages=9), dict(page_size=32, page_stride=4096)):
        two = (lg.hiplib.Pages * 2)(pages(lg, {}), pages(lg, change))
        refused(lg, H.lg_hip_paged_compact(two, 2, 3, 4, P16, 4, P16, P16, P16, P16, None), -2, "layer 1")
        refused(lg, H.lg_hip_paged_copy(two, 2, 3, P16, P16, P16, None), -2, "layer 1")


@pytest.mark.parametrize("layers, n, null, code, words", [(-1, 3, None, -2, "-1 layers"), (1, -1, None, -2, "-1 pages"), (1, 65536, None, -2, "65536 pages"), *((1, 3, k, -1, "null") for k in range(3))])
def test_copy_refuses(lg, layers, n, null, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, {})
    refused(lg, H.lg_hip_paged_copy(C.byref(p), layers, n, *(None if null == k else P16 for k in range(3)), None), code, words)


@pytest.mark.parametrize("change, code, words", [
    (dict(n_seq=-1), -2, "sequences"), (dict(n_seq=4097), -2, "sequences"), (dict(page=8), -2, "pages of 8"), (dict(page=48), -2, "pages of 48"), (dict(page=512), -2, "pages of 512"),
    (dict(n_pages=0), -2, "0 pages"), (dict(n_pages=1 << 27), -2, "31 bits"), (dict(blocks=0), -2, "0 blocks"), (dict(blocks=1 << 27), -2, "31 bits"), (dict(n_seq=4096, blocks=1 << 19), -2, "31 bits"),
    *((dict(null=k), -1, "null") for k in range(11)), (dict(work=None), -2, "working memory"), (dict(short=1), -2, "working memory"), (dict(work=C.c_void_p((1 << 20) + 16)), -2, "working memory")])
def test_fork_refuses(lg, change, code, words):
    H = lg.hiplib.load_hip()
    a = dict(n_seq=3, page=16, n_pages=8, blocks=4, null=None, work=P16, short=0)
    a.update(change)
    p = [None if a["null"] == k else P16 for k in range(11)]
    need = H.lg_hip_paged_fork_workspace(3, 8, 4)
    assert need > 0
    refused(lg, H.lg_hip_paged_fork(a["n_seq"], a["page"], a["n_pages"], a["blocks"], *p, a["work"], (1 << 40 if a["n_seq"] != 3 else need) - a["short"], None), code, words)


RULES = dict(n_seq=3, hist=1 << 20, hist_len=1 << 20, hist_stride=50, penalty=1 << 20, n_bias=4, bias_start=1 << 20, bias_tok=1 << 20, bias=1 << 20, n_allow=2, allow=1 << 20, allow_stride=4,
             tree_mask=1 << 20, tree_start=1 << 20, tree_tok=1 << 20)


@pytest.mark.parametrize("change, call, code, words", [
    ({}, dict(rows=-1), -2, "-1 rows"), ({}, dict(rows=65536), -2, "65536 rows"), ({}, dict(vocab=0), -2, "vocabulary of 0"), ({}, dict(vocab=524289), -2, "vocabulary"), ({}, dict(stride=99), -2, "99 and 100 apart"),
    ({}, dict(out_stride=99), -2, "100 and 99 apart"), (dict(n_seq=-1), {}, -2, "-1 sequences"), (dict(n_bias=-1), {}, -2, "-1 biases"), (dict(n_allow=-1), {}, -2, "-1 grammars"), (dict(hist_stride=0), {}, -2, "texts 0"),
    (dict(hist_stride=(1 << 30) + 1), {}, -2, "texts"), (dict(allow_stride=3), {}, -2, "3 words"), (dict(hist_len=None), {}, -1, "null"), (dict(penalty=None), {}, -1, "null"), (dict(bias_start=None), {}, -1, "null"),
    (dict(bias_tok=None), {}, -1, "null"), (dict(bias=None), {}, -1, "null"), (dict(allow=None), {}, -1, "null"), (dict(tree_start=None), {}, -1, "null"), (dict(tree_tok=None), {}, -1, "null"),
    (dict(hist=None, penalty=None), {}, -1, "null"), ({}, dict(logits=None), -1, "null"), ({}, dict(out=None), -1, "null"), ({}, dict(logits=C.c_void_p((1 << 20) + 2)), -2, "aligned"),
    (dict(hist=(1 << 20) + 2), {}, -2, "aligned"), (dict(tree_mask=(1 << 20) + 4), {}, -2, "aligned"), ({}, dict(out=P16, out_stride=104), -2, "in place")])
def test_rules_refuse(lg, change, call, code, words):
    H = lg.hiplib.load_hip()
    a = dict(rows=3, vocab=100, stride=100, out_stride=100, logits=P16, out=C.c_void_p(1 << 22))
    a.update(call)
    r = lg.hiplib.LogitRules(**{**RULES, **change})
    refused(lg, H.lg_hip_adjust_logits(C.byref(r), a["logits"], a["stride"], a["rows"], a["vocab"], a["out"], a["out_stride"], None), code, words)
    refused(lg, H.lg_hip_adjust_logits(None, P16, 100, 3, 100, P16, 100, None), -1, "null")
    assert H.lg_hip_adjust_logits(C.byref(lg.hiplib.LogitRules()), P16, 100, 0, 100, P16, 100, None) == 0
