"""What the operators of a batched decode step refuse before anything is launched, with the codes and messages of the C ABI: no GPU is needed
(a call that got past its checks would fail otherwise on a machine without one)."""
import ctypes as C

import pytest

P16 = C.c_void_p(1 << 20)          # a pointer that nothing reads: every call below is refused


def refused(lg, rc, code, words):
    msg = lg.hiplib.load_hip().lg_hip_last_error().decode()
    assert rc == code and words in msg, (rc, msg)


@pytest.mark.parametrize("change, code, words", [
    (dict(n_seq=-1), -2, "sequences"), (dict(n_seq=4097), -2, "sequences"), (dict(page=8), -2, "pages of 8"), (dict(page=48), -2, "pages of 48"),
    (dict(page=512), -2, "pages of 512"), (dict(n_pages=0), -2, "0 pages"), (dict(n_pages=1 << 27), -2, "31 bits"), (dict(blocks=0), -2, "0 blocks"),
    (dict(blocks=1 << 27), -2, "31 bits"), (dict(n_slots=-1), -2, "slots"), (dict(old=None), -1, "null"), (dict(free=None), -1, "null"),
    (dict(status=None), -1, "null"), (dict(slots=None), -1, "null"), (dict(start=None), -1, "null")])
def test_plan_refuses(lg, change, code, words):
    H = lg.hiplib.load_hip()
    a = dict(n_seq=3, page=16, n_pages=8, blocks=4, old=P16, new=P16, table=P16, free=P16, n_free=P16, start=P16, slots=P16, n_slots=5, status=P16)
    a.update(change)
    rc = H.lg_hip_paged_plan(a["n_seq"], a["page"], a["n_pages"], a["blocks"], a["old"], a["new"], a["table"], a["free"], a["n_free"], a["start"],
                             a["slots"], a["n_slots"], a["status"], None, 0, None)
    refused(lg, rc, code, words)


PAGES = dict(k=1 << 20, v=1 << 21, n_pages=8, page_size=16, n_head_kv=2, head_dim=64, row_stride=128, page_stride=2048)
BAD_PAGES = [
    (dict(k=0), -1, "null"), (dict(v=0), -1, "null"), (dict(page_size=24), -2, "pages of 24"), (dict(n_pages=0), -2, "0 pages"),
    (dict(n_pages=1 << 27), -2, "31 bits"), (dict(head_dim=96), -2, "heads of 96"), (dict(head_dim=0), -2, "heads of"), (dict(n_head_kv=0), -2, "0 key heads"),
    (dict(row_stride=120), -2, "strides"), (dict(row_stride=132), -2, "strides"), (dict(page_stride=2040), -2, "strides"), (dict(page_stride=2052), -2, "strides"),
    (dict(page_stride=1 << 62), -2, "strides"), (dict(row_stride=1 << 62), -2, "strides"), (dict(k=(1 << 20) + 8), -2, "aligned")]


def pages(lg, change):
    return lg.hiplib.Pages(**{**PAGES, **change})


@pytest.mark.parametrize("change, code, words", BAD_PAGES)
def test_bad_pages_are_refused(lg, change, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, change)
    refused(lg, H.lg_hip_paged_write(C.byref(p), P16, P16, 128, P16, 3, None), code, words)
    refused(lg, H.lg_hip_paged_attention(C.byref(p), P16, 512, 3, 8, P16, 4, P16, 64, 0, 1.0, P16, 512, P16, 1 << 30, None), code, words)


@pytest.mark.parametrize("k, v, stride, slots, n, code, words", [
    (None, P16, 128, P16, 3, -1, "null"), (P16, None, 128, P16, 3, -1, "null"), (P16, P16, 128, None, 3, -1, "null"), (P16, P16, 128, P16, -1, -2, "-1 tokens"),
    (P16, P16, 124, P16, 3, -2, "124 apart"), (P16, P16, 130, P16, 3, -2, "130 apart"), (C.c_void_p((1 << 20) + 4), P16, 128, P16, 3, -2, "aligned")])
def test_write_refuses(lg, k, v, stride, slots, n, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, {})
    refused(lg, H.lg_hip_paged_write(C.byref(p), k, v, stride, slots, n, None), code, words)
    assert H.lg_hip_paged_write(C.byref(p), k, v, stride, slots, 0, None) == 0                    # nothing to write


def test_calls_beyond_what_a_launch_holds_are_refused(lg):
    H, p = lg.hiplib.load_hip(), pages(lg, {})
    refused(lg, H.lg_hip_paged_write(C.byref(p), P16, P16, 128, P16, 1 << 27, None), -2, "tokens of 128 values in one call")
    for seqs, heads, kv in ((4096, 2, 1), (128, 2, 1), (4096, 16, 2)):           # tiles of all sequences, splits of all heads
        q = pages(lg, dict(n_head_kv=kv))
        refused(lg, H.lg_hip_paged_attention(C.byref(q), P16, 64 * heads, seqs, heads, P16, 1 << 26, P16, 1 << 30, 0, 1.0, P16, 64 * heads, P16, 1 << 62, None), -2, "in one call")


@pytest.mark.parametrize("change, code, words", [
    (dict(n_seq=-1), -2, "-1 sequences"), (dict(n_seq=4097), -2, "4097 sequences"), (dict(heads=7), -2, "7 query heads"), (dict(heads=18), -2, "18 query heads"), (dict(heads=0), -2, "0 query heads"),
    (dict(max_len=-1), -2, "lengths up to -1"), (dict(max_len=(1 << 30) + 1), -2, "lengths up to"), (dict(blocks=0), -2, "0 blocks"), (dict(blocks=1 << 27), -2, "blocks"),
    (dict(window=-5), -2, "window"), (dict(q=None), -1, "null"), (dict(table=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(out=None), -1, "null"),
    (dict(q_stride=508), -2, "508 apart"), (dict(q_stride=513), -2, "513 apart"), (dict(out_stride=511), -2, "511 apart"),
    (dict(q=C.c_void_p((1 << 20) + 8)), -2, "aligned"), (dict(out=C.c_void_p((1 << 20) + 2)), -2, "output rows"),
    (dict(work=None), -2, "working memory"), (dict(short=1), -2, "working memory"), (dict(work=C.c_void_p((1 << 20) + 16)), -2, "working memory")])
def test_attention_refuses(lg, change, code, words):
    H, p = lg.hiplib.load_hip(), pages(lg, {})
    a = dict(n_seq=3, heads=8, q=P16, q_stride=512, table=P16, blocks=1024, lens=P16, max_len=8192, window=0, out=P16, out_stride=512, work=P16, short=0)
    a.update(change)
    need = H.lg_hip_paged_attention_workspace(3, 8, 2, 64, 8192, 0)
    assert need > 0
    rc = H.lg_hip_paged_attention(C.byref(p), a["q"], a["q_stride"], a["n_seq"], a["heads"], a["table"], a["blocks"], a["lens"], a["max_len"], a["window"], 1.0,
                                  a["out"], a["out_stride"], a["work"], need - a["short"], None)
    refused(lg, rc, code, words)
    assert H.lg_hip_paged_attention(C.byref(p), P16, 512, 0, 8, P16, 4, P16, 64, 0, 1.0, P16, 512, None, 0, None) == 0      # no sequence


@pytest.mark.parametrize("change, code, words", [
    (dict(rows=-1), -2, "-1 rows"), (dict(rows=65536), -2, "rows"), (dict(vocab=0), -2, "vocabulary of 0"), (dict(vocab=524289), -2, "vocabulary"),
    (dict(stride=99), -2, "99 apart"), (dict(logits=None), -1, "null"), (dict(params=None), -1, "null"), (dict(u=None), -1, "null"), (dict(tok=None), -1, "null"),
    (dict(logits=C.c_void_p((1 << 20) + 2)), -2, "aligned"), (dict(vocab=8193, work=None), -2, "working memory"), (dict(vocab=8193, short=1), -2, "working memory"),
    (dict(vocab=8193, work=C.c_void_p((1 << 20) + 16)), -2, "working memory")])
def test_sample_refuses(lg, change, code, words):
    H = lg.hiplib.load_hip()
    a = dict(logits=P16, stride=524289, rows=3, vocab=100, params=P16, u=P16, tok=P16, work=P16, short=0)
    a.update(change)
    need = H.lg_hip_sample_workspace(3, a["vocab"]) - a["short"] if a["short"] else 1 << 30
    rc = H.lg_hip_sample(a["logits"], a["stride"], a["rows"], a["vocab"], a["params"], a["u"], a["tok"], None, None, a["work"], need, None)
    refused(lg, rc, code, words)
    assert H.lg_hip_sample(P16, 100, 0, 100, P16, P16, P16, None, None, P16, 1 << 30, None) == 0      # no row
