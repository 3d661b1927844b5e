"""Rows of logits at the ends of what f32 holds, and filters at theirs, through the C ABI against the definition in whole numbers."""
import numpy as np
import pytest

from test_gpu_sample import check, dev, rows_like_logits  # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [8192, 8193, 60000])
def test_logits_whose_distance_is_beyond_f32(dev, V):
    """Logits up to 6e38 apart, at temperatures at which such a distance still leaves weight: rows of one launch, and the shortest and a usual one of four.
    (At 2e37 the far tokens weigh 2 units of 2^-44, which a border of top-p could not tell from their rounding: no top-p there.)"""
    rng = np.random.default_rng(V)
    l = rng.choice(np.array([3e38, 1e38, -1e38, -3e38, -np.inf, np.nan], np.float32), (6, V), p=[0.05, 0.2, 0.2, 0.45, 0.05, 0.05])
    for T in (np.inf, 3e38, 1e38):
        params = [(T, 0, 1.0, 0.0), (T, 0, 0.9, 0.0), (T, V // 2, 1.0, 0.0), (T, V // 2, 0.7, 0.0), (T, 0, 1.0, 0.01), (T, 50, 0.9, 0.0)]
        print(f"sample V={V} T={T}", flush=True)
        check(dev, l, params, rng.random(6))
    for T in (2e37, 1e37, 1.0):
        params = [(T, 0, 1.0, 0.0), (T, 0, 1.0, 1e-3), (T, V // 2, 1.0, 0.0), (T, V // 4, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (T, 50, 1.0, 0.0)]
        print(f"sample V={V} T={T}", flush=True)
        check(dev, l, params, rng.random(6))


@pytest.mark.parametrize("V", [300, 8193, 131073])
def test_min_p_above_one_is_one(dev, V):
    """A min-p above 1 keeps the likeliest token and its equals, as 1 does, in rows of one launch and of four, with and without the other filters."""
    rng = np.random.default_rng(V)
    l = rows_like_logits(rng, 6, V)
    l[:, V // 2] = l[:, 7] = l.max(1)
    rest = [(1.0, 0, 1.0), (1.0, 0, 0.9), (1.0, 64, 0.95), (1.0, 290, 1.0), (1.0, 5000, 0.98), (np.inf, 0, 1.0)]
    us = rng.random(6)
    want = check(dev, l, [(*x, 1.0) for x in rest], us)
    for m in (1.5, 1e30, np.inf):
        assert check(dev, l, [(*x, m) for x in rest], us).tolist() == want.tolist()


def test_top_p_near_one_of_a_large_vocabulary(dev):
    """Bell-shaped logits: so far out in the tail that the share which an estimated sum may be off is tens of thousands of tokens, more than are kept as candidates."""
    rng = np.random.default_rng(77)
    l = (30.0 * np.tanh(rng.normal(0, 3.0, (6, 262144)) / 30.0)).astype(np.float32)
    params = [(0.8, 0, 0.995, 0.0), (1.0, 0, 0.995, 0.0), (1.0, 0, 0.999, 0.0), (1.5, 0, 0.999, 0.0), (1.5, 0, 0.9999, 0.0), (1.0, 200000, 0.999, 1e-6)]
    print("sample top-p near one", flush=True)
    check(dev, l, params, rng.random(6))
