"""Rules for logits through the C ABI against the plain form in 64 bits: every logit within half a step of f32."""
import numpy as np
import pytest

from drafts import adjust, bits, rules_ref
from serving import Device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def close(got, want):
    """One rounding to f32: 2^-24 of the value, and of the intermediate results in 64 bits 2^-52 of the largest (within 2^-20 of the f32 step here)."""
    plain = np.isfinite(want) & np.isfinite(got)
    assert np.array_equal(got[~plain].astype(np.float64), want[~plain], equal_nan=True)
    off = np.abs(got.astype(np.float64)[plain] - want[plain])
    assert (off <= np.abs(want[plain]) * 2.0 ** -24 * (1 + 2.0 ** -20) + 1e-14).all(), float(off.max())


def some(rng, rows, V):
    return (rng.normal(0, 5, (rows, V))).astype(np.float32)


def sets(rng, n, V, share=0.1, room=0):
    words = (V + 31) // 32 + room
    return (np.packbits(rng.random((n, words * 32)) < share, axis=1, bitorder="little")).view(np.uint32).reshape(n, words)


@pytest.mark.parametrize("rows, V, text", [(1, 1, 3), (2, 31, 100), (5, 8191, 50), (3, 8192, 1000), (4, 8193, 333), (1, 262144, 3001), (3, 32003, 20000), (2, 524288, 1), (70, 300, 17)])
@pytest.mark.parametrize("pad", [0, 1, 4])
def test_all_rules_at_once(lg, dev, rows, V, text, pad):
    rng = np.random.default_rng(rows * 1000 + V)
    n_seq = max(1, rows // 2)
    seq = rng.integers(0, n_seq, rows)
    penalty = [(rng.choice([0.8, 1.0, 1.2]), rng.choice([0.0, 0.5]), rng.choice([0.0, 0.125, -0.3]), int(rng.integers(0, text + 1))) for _ in range(n_seq)]
    hist = np.floor(V * rng.random((n_seq, text)) ** 3).astype(np.int32)
    hist_len = rng.integers(0, text + 1, n_seq)
    hist_len[0] = text
    per = min(V, 40)
    bias = (np.arange(n_seq + 1) * per, np.concatenate([rng.choice(V, per, replace=False) for _ in range(n_seq)]), rng.normal(0, 3, n_seq * per).astype(np.float32))
    allow, allow_row = sets(rng, 3, V, 0.3, pad), rng.integers(-1, 4, rows)
    x = some(rng, rows, V)
    args = dict(seq=seq, penalty=penalty, hist=hist, hist_len=hist_len, bias=bias, allow=allow, allow_row=allow_row)
    want = rules_ref(x, seq, penalty, hist, hist_len, None, bias, allow, allow_row)
    got = adjust(lg, dev, x, **args, pad=pad)
    close(got, want)
    assert np.array_equal(adjust(lg, dev, x, **args, pad=pad, in_place=True), got, equal_nan=True)


@pytest.mark.parametrize("which", ["penalty", "bias", "allow", "none", "frequency", "tree"])
@pytest.mark.parametrize("in_place", [False, True])
def test_each_rule_alone(lg, dev, which, in_place):
    rng = np.random.default_rng(3)
    rows, V = 4, 20000
    x = some(rng, rows, V)
    hist, hist_len = rng.integers(0, V, (rows, 500)).astype(np.int32), np.array([500, 0, 33, 1])
    a = dict(penalty=None, hist=None, hist_len=None, tree=None, bias=None, allow=None, allow_row=None)
    if which == "penalty":
        a.update(penalty=[(1.3, 0, 0, 0)] * rows, hist=hist, hist_len=hist_len)
    elif which == "frequency":
        a.update(penalty=[(1.0, 0, 0.25, 100)] * rows, hist=hist, hist_len=hist_len)
    elif which == "bias":
        a.update(bias=(np.array([0, 3, 3, 700, 701]), rng.integers(0, V, 701), rng.normal(0, 1, 701).astype(np.float32)))
    elif which == "allow":
        a.update(allow=sets(rng, rows, V))
    elif which == "tree":
        a.update(penalty=[(1.1, 0.5, 0.25, 0)] * 2, tree=(np.array([1, 3, 1, 3], np.uint64), np.array([0, 2, 4]), rng.integers(0, V, rows)))
    seq = np.array([0, 0, 1, 1]) if which == "tree" else None
    got = adjust(lg, dev, x, seq=seq, in_place=in_place, **a)
    close(got, rules_ref(x, seq, **{k: a[k] for k in ("penalty", "hist", "hist_len", "tree", "bias", "allow", "allow_row")}))
    if which == "none":
        assert np.array_equal(got, x)


def test_the_way_to_a_row_of_a_tree_counts(lg, dev):
    """Two trees: the tokens of a row's set are generated ones; rows outside the step do not count, nor do sets of rows without a sequence."""
    rng = np.random.default_rng(4)
    V, start = 500, np.array([0, 5, 12])
    rows = 12
    tok = rng.integers(0, 20, rows)
    mask = np.array([bits(rng.choice(64, 3)) | np.uint64(1) for _ in range(rows)], np.uint64)
    mask[3] = np.uint64(0xFFFFFFFFFFFFFFFF)
    seq = np.array([0] * 5 + [1] * 6 + [-1])
    hist = rng.integers(0, 30, (2, 64)).astype(np.int32)
    penalty, hist_len = [(1.2, 0.5, 0.25, 60), (1.0, 0.0, 1.0, 0)], np.array([64, 7])
    x = some(rng, rows, V)
    got = adjust(lg, dev, x, seq=seq, penalty=penalty, hist=hist, hist_len=hist_len, tree=(mask, start, tok))
    close(got, rules_ref(x, seq, penalty, hist, hist_len, (mask, start, tok), None, None, None))
    assert np.array_equal(got[11], x[11])


def test_values_at_the_ends(lg, dev):
    """Infinite and NaN logits, parameters that are off, tokens outside the vocabulary, a bias named twice, lengths below 0 and above the room."""
    V = 100
    x = np.tile(np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1e-38, -3e38, 3e38, 1e-45, 7.0], np.float32), (6, 10))
    hist = np.tile(np.arange(-5, 105, dtype=np.int32), (6, 1))
    penalty = [(np.nan, np.nan, np.nan, 0), (0.0, 0.0, 0.0, 0), (-1.0, 1.0, 0.0, -5), (2.0, 0.0, 0.0, 1 << 30), (np.inf, 0.0, 0.0, 0), (0.5, 3e38, 0.0, 0)]
    hist_len = np.array([110, 110, 110, 1 << 30, 110, -3])
    bias = (np.array([0, 2, 5, 5, 9, 9, 11]), np.array([3, 3, -1, 100, 99, 2, 2, 2, 3, 0, 1]), np.array([1, 2, 3, 4, 5, 6, -np.inf, 1, np.inf, np.nan, -0.0], np.float32))
    got = adjust(lg, dev, x, penalty=penalty, hist=hist, hist_len=hist_len, bias=bias)
    want = rules_ref(x, None, penalty, hist, hist_len, None, bias, None, None)
    with np.errstate(over="ignore"):
        f = want.astype(np.float32)
    assert np.array_equal(got, f, equal_nan=True)
    assert got[0, 3] == -np.inf and (got[0] == x[0])[[0, 1, 5, 6, 7, 8, 9]].all()


def test_bias_starts_outside_the_list(lg, dev):
    rng = np.random.default_rng(6)
    x = some(rng, 4, 50)
    bias = (np.array([-3, 2, 100, 1, 0]), np.array([4, 5, 6]), np.array([1.0, 2.0, 4.0], np.float32))
    close(adjust(lg, dev, x, bias=bias), rules_ref(x, None, None, None, None, None, bias, None, None))


def test_a_set_without_a_token_leaves_nothing(lg, dev):
    rng = np.random.default_rng(7)
    x = some(rng, 2, 9000)
    got = adjust(lg, dev, x, allow=np.zeros((1, 282), np.uint32))
    assert (got[0] == -np.inf).all() and np.array_equal(got[1], x[1])            # row 1 has no set


def test_texts_that_do_not_start_at_16_bytes(lg, dev):
    rng = np.random.default_rng(8)
    for room in (1, 2, 3, 5, 1001):
        x = some(rng, 5, 3000)
        hist = rng.integers(0, 3000, (5, room)).astype(np.int32)
        penalty, lens = [(1.5, 1.0, 0.5, room // 2)] * 5, np.minimum(room, [room, 0, 1, 2, 4])
        close(adjust(lg, dev, x, penalty=penalty, hist=hist, hist_len=lens), rules_ref(x, None, penalty, hist, lens, None, None, None, None))


def test_no_row(dev, lg):
    r = lg.hiplib.LogitRules()
    import ctypes as C
    assert dev.H.lg_hip_adjust_logits(C.byref(r), None, 10, 0, 10, None, 10, None) == 0
