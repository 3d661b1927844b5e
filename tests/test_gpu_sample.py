"""Tokens drawn from logits rows through the C ABI against the definition in whole numbers (serving.sample_ref)."""
import numpy as np
import pytest

from serving import Device, sample, sample_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def clear_of_borders(l, p, u):
    """u, moved on until the last bits of weights do not decide the draw."""
    for _ in range(100):
        ref = sample_ref(l, *p, u)
        if ref[3]:
            return np.float32(u), ref
        u = np.float32((u * 0.9 + 0.07) % 1.0)
    raise AssertionError("a border of top-p or min-p is too near for this row")


def check(dev, logits, params, us, stride=None):
    pairs = [clear_of_borders(l, p, np.float32(u)) for l, p, u in zip(logits, params, us)]
    tok, prob, kept = sample(dev, logits, params, np.array([u for u, _ in pairs], np.float32), stride)
    want = [r for _, r in pairs]
    assert tok.tolist() == [r[0] for r in want]
    assert kept.tolist() == [r[2] for r in want]
    # one rounding of the quotient to f32; a weight may be one unit of 2^-44 of the largest off
    exact = np.array([r[1] for r in want])
    assert (np.abs(prob - exact) <= exact * 2.0 ** -23 + 2.0 ** -43).all()
    return tok


SETTINGS = [(1.0, 64, 0.95, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.5, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 5000, 0.98, 0.0),
            (0.6, 1, 1.0, 0.0), (2.0, 200, 0.5, 0.02), (1.0, 0, 0.0, 0.0), (1.0, 0, 1e-9, 0.0), (1.0, -3, 2.0, -1.0), (0.05, 0, 0.999, 0.0), (30.0, 0, 0.97, 0.0),
            (1.0, 3, 0.5, 0.9), (1.0, 0, 1.0, 1.0), (1.0, 300, 0.9, 0.001), (5.0, 100000, 0.6, 0.0)]


def rows_like_logits(rng, rows, V, spread=3.0):
    z = rng.normal(0, spread, (rows, V)) + (rng.random((rows, V)) < 8 / V) * rng.uniform(0, 14, (rows, 1))
    return (30.0 * np.tanh(z / 30.0)).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 255, 1000, 4097, 8192, 50001])
def test_every_setting_on_rows_of_every_size(dev, V):
    rng = np.random.default_rng(V)
    l = rows_like_logits(rng, len(SETTINGS), V)
    print(f"sample V={V}", flush=True)
    check(dev, l, SETTINGS, rng.random(len(SETTINGS)))
    check(dev, l, SETTINGS, rng.random(len(SETTINGS)), stride=V + 5)


@pytest.mark.parametrize("rows", [1, 5, 18])
def test_the_largest_vocabulary_in_use(dev, rows):
    rng = np.random.default_rng(rows)
    l = rows_like_logits(rng, rows, 262144)
    params = [SETTINGS[i % len(SETTINGS)] for i in range(rows)]
    check(dev, l, params, rng.random(rows))


def test_the_largest_vocabulary(dev):
    rng = np.random.default_rng(9)
    l = np.concatenate([np.zeros((1, 524288), np.float32), rows_like_logits(rng, 2, 524288)])
    check(dev, l, [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (1.0, 70000, 0.9, 0.0)], [0.999, 0.3, 0.7])


@pytest.mark.parametrize("kind", ["equal", "two", "coarse", "masked", "one", "far", "steep", "flat"])
def test_ties_masks_and_odd_distributions(dev, kind):
    rng = np.random.default_rng(len(kind))
    V, n = 10007, len(SETTINGS)
    l = rows_like_logits(rng, n, V)
    if kind == "equal":
        l[:] = np.float32(2.5)
    elif kind == "two":
        l = np.where(rng.random(l.shape) < 0.3, np.float32(1.0), np.float32(0.25))
    elif kind == "coarse":                                  # a head that answers in bfloat16, and zeros of either sign
        l = (l.view(np.uint32) & 0xFFFF0000).view(np.float32)
        l[:, ::7] = 0.0; l[:, 1::7] = -0.0
    elif kind == "masked":
        l[rng.random(l.shape) < 0.95] = -np.inf
        l[:, ::13] = np.nan
    elif kind == "one":
        x = l[:, 77].copy()
        l[:] = -np.inf
        l[:, 77] = x
    elif kind == "far":                                     # one logit far above the rest, one far below
        l[:, 5000] = 900.0; l[:, 1] = -1e30
    elif kind == "steep":
        l = -np.sort(rng.exponential(40.0, l.shape).astype(np.float32), 1)[:, rng.permutation(V)]
    else:
        l *= np.float32(1e-4)
    check(dev, l.astype(np.float32), SETTINGS, rng.random(n))


@pytest.mark.parametrize("kind", ["crowded", "equal", "outliers", "tiny temperature", "clustered", "two borders", "coarse"])
def test_long_rows_whose_border_is_hard_to_bracket(dev, kind):
    """More tokens in one bin than candidates are kept, a temperature whose inverse is no f32, all the likely tokens in a few groups, and
    top-k and top-p borders far from each other and in one place."""
    rng = np.random.default_rng(len(kind) + 50)
    V = 60000
    l = rows_like_logits(rng, 6, V)
    params = [(1.0, 0, 0.9, 0.0), (1.0, 20000, 0.9, 0.0), (1.0, 20000, 1.0, 0.0), (1.0, 100, 0.95, 0.0), (1.0, 600, 0.999, 0.01), (1.0, 0, 1.0, 0.0)]
    if kind == "crowded":                       # 50000 logits within a bin's width
        l[:, :50000] = np.float32(3.0) + rng.normal(0, 1e-4, (6, 50000)).astype(np.float32)
    elif kind == "equal":
        l[:] = np.float32(-4.0)
    elif kind == "outliers":
        l *= np.float32(0.01)
        l[:, 7] = -25.0; l[:, 59999] = 5.0
    elif kind == "tiny temperature":
        l = np.where(rng.random(l.shape) < 0.2, np.float32(1e-30), np.float32(0)).astype(np.float32)
        params = [(1e-30, *x[1:]) for x in params[:3]] + [(1e-42, *x[1:]) for x in params[3:]]
    elif kind == "clustered":
        l[:, 1024:3000] += 12.0
    elif kind == "two borders":
        params = [(1.0, k, p, 0.0) for k, p in ((600, 0.05), (5000, 0.5), (59999, 0.3), (60000, 0.99), (513, 0.9999), (30000, 0.9999999))]
    else:
        l = (l.view(np.uint32) & 0xFFFF0000).view(np.float32)
    check(dev, l, params, rng.random(6))


def test_random_numbers_at_the_ends_and_beyond(dev):
    rng = np.random.default_rng(21)
    us = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, 7.0, -0.5, np.nan, 2.0 ** -30, np.inf, -np.inf], np.float32)
    l = np.repeat(rows_like_logits(rng, 1, 300), len(us), 0)
    for p in ((1.0, 0, 1.0, 0.0), (1.0, 20, 0.9, 0.0)):
        tok, _, _ = sample(dev, l, [p] * len(us), us)
        ends = [sample_ref(l[0], *p, u)[0] for u in (0.0, 1.0)]
        assert [int(t) for t in tok] == [ends[0], sample_ref(l[0], *p, us[1])[0], ends[1], ends[1], ends[0], ends[0], sample_ref(l[0], *p, us[6])[0], ends[1], ends[0]]


def test_rows_without_a_token_and_with_infinities(dev):
    V = 1500
    l = np.zeros((6, V), np.float32)
    l[0] = -np.inf; l[1] = np.nan; l[2, 700] = np.inf; l[3, 3] = l[3, 1200] = np.inf; l[4, :] = -np.inf; l[4, 9] = -3e38; l[5] = np.nan; l[5, 1499] = -5.0
    for p in ((1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.01), (0.0, 0, 1.0, 0.0), (np.inf, 0, 1.0, 0.0), (np.nan, 0, np.nan, np.nan), (1e-40, 0, 0.9, 0.0)):
        tok, prob, kept = sample(dev, l, [p] * 6, np.full(6, 0.75, np.float32))
        greedy = not p[0] > 0
        assert tok.tolist() == [-1, -1, 700, 3 if greedy else 1200, 9, 1499], p
        assert prob.tolist() == [0, 0, 1, 1 if greedy else 0.5, 1, 1] and kept.tolist() == [0, 0, 1, 1 if greedy else 2, 1, 1]


def test_temperature_of_infinity_is_uniform(dev):
    l = rows_like_logits(np.random.default_rng(4), 3, 1000)
    l[:, 500:] = -np.inf
    tok, prob, kept = sample(dev, l, [(np.inf, 0, 1.0, 0.0)] * 3, np.array([0.0, 0.5, 0.999], np.float32))
    assert tok.tolist() == [0, 250, 499] and kept.tolist() == [500] * 3 and np.allclose(prob, 1 / 500, rtol=2.0 ** -23)


def test_the_share_of_each_token_is_its_probability(dev):
    """Evenly spread numbers: every token comes as often as its probability says, to one draw either side."""
    V, n = 40, 4000
    l = np.repeat(rows_like_logits(np.random.default_rng(8), 1, V, 1.0), n, 0)
    us = (np.arange(n) + 0.5) / n
    tok, prob, _ = sample(dev, l, [(1.0, 0, 1.0, 0.0)] * n, us.astype(np.float32))
    p = np.exp(l[0].astype(np.float64)); p /= p.sum()
    assert np.abs(np.bincount(tok, minlength=V) - n * p).max() <= 1.0
    assert np.allclose(prob, p[tok], rtol=1e-6)


def test_the_same_row_gives_the_same_token_wherever_it_stands(dev):
    rng = np.random.default_rng(10)
    one = rows_like_logits(rng, 1, 262144)
    p = [(1.0, 0, 0.93, 0.0), (1.0, 64, 0.95, 0.0), (1.0, 0, 1.0, 0.0)]
    alone = [sample(dev, one, [x], np.array([0.37], np.float32)) for x in p]
    many = sample(dev, np.repeat(one, 12, 0), p * 4, np.full(12, 0.37, np.float32))
    for i in range(12):
        assert [int(many[j][i]) for j in (0, 2)] == [int(alone[i % 3][j][0]) for j in (0, 2)] and many[1][i] == alone[i % 3][1][0]


@pytest.mark.parametrize("V, k", [(8193, 64), (8193, 65), (8321, 65), (33001, 257), (131072, 512), (131073, 256), (131073, 257), (262144, 513), (200003, 128)])
def test_a_small_top_k_and_the_next_larger_one(dev, V, k):
    """Rows by their groups' maxima up to a top-k of half as many as there are groups: of any distribution, of few tokens, of many equal ones, of likely ones
    that lie together, of tiny weights."""
    rng = np.random.default_rng(V + k)
    l = rows_like_logits(rng, 7, V)
    few = rng.choice(V, 30, replace=False)
    l[1] = np.where(np.isin(np.arange(V), few), l[1], -np.inf)
    l[2] = np.round(l[2] * 2) / 2                            # hundreds of equal ones at the border
    l[3, V - 700:] += np.float32(9.0)
    l[4] = np.float32(1.0); l[4, V // 2:V // 2 + 300] = np.float32(1.25)
    l[5] *= np.float32(30.0)
    print(f"sample V={V} k={k}", flush=True)
    for rest in ((0.95, 0.0), (1.0, 0.0), (0.3, 0.02)):
        check(dev, l, [(1.0, k, *rest)] * 6 + [(0.4, k - 7, *rest)], rng.random(7))
