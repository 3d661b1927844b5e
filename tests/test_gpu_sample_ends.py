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
