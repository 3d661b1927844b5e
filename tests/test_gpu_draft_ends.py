"""The operators around a verify step at the most that a call takes: sequences, rows, pages."""
import numpy as np
import pytest

from drafts import adjust, compact_ref, layers_of, rules_ref, starts_of
from serving import Device, pages_of
from test_gpu_rules import close, sets, some
from test_gpu_shared_pages import paths, pool_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def test_rules_for_the_most_rows(lg, dev):
    rng = np.random.default_rng(1)
    rows, V, n = 65535, 37, 5
    seq, hist, hist_len = rng.integers(-1, n + 1, rows), rng.integers(-2, V + 2, (n, 50)).astype(np.int32), np.array([50, 0, 3, 49, 20])
    penalty = [(1.25, 0.5, 0.25, 10), (1.0, 1.0, 0.0, 0), (0.75, 0.0, 0.5, 2), (1.0, 0.0, 0.0, 0), (1.5, -1.0, -0.5, 50)]
    bias = (np.array([0, 2, 2, 5, 7, 7]), rng.integers(0, V, 7), rng.normal(0, 1, 7).astype(np.float32))
    allow, allow_row = sets(rng, 4, V, 0.5), rng.integers(-1, 5, rows)
    x = some(rng, rows, V)
    got = adjust(lg, dev, x, seq=seq, penalty=penalty, hist=hist, hist_len=hist_len, bias=bias, allow=allow, allow_row=allow_row)
    close(got, rules_ref(x, seq, penalty, hist, hist_len, None, bias, allow, allow_row))


def test_rows_of_the_most_sequences(lg, dev):
    rng = np.random.default_rng(2)
    n, most, page = 4096, 64, 16
    sizes = rng.integers(0, most + 1, n)
    sizes[0] = most
    lens = sizes + rng.integers(0, 40, n)
    held = pages_of(lens, page)
    n_pages, blocks = int(held.sum()) + 1, int(held.max())
    table, _, _, _ = pool_of(rng, lens, page, n_pages, blocks)
    path, count = paths(rng, np.maximum(sizes, 1), most)
    pools = rng.integers(0, 1 << 16, (2, 2, n_pages, page, 64)).astype(np.uint16)
    ls, pool = layers_of(lg, pools, 1, 64, dev)
    p = [dev.up(x, np.int32) for x in (table, lens, starts_of(sizes), path, count)]
    dev.check(dev.H.lg_hip_paged_compact(ls, 2, n, most, p[0], blocks, *p[1:], None), "paged_compact")
    got = dev.back(pool, pools.shape, np.uint16)
    dev.free()
    assert np.array_equal(got, compact_ref(pools, page, n_pages, table, lens, starts_of(sizes), path, count))


def test_the_most_pages_in_one_copy(lg, dev):
    rng = np.random.default_rng(3)
    n, page = 65535, 16
    n_pages = n + 3000
    ids = rng.permutation(n_pages)
    to, frm, rows = ids[:n], ids[n + rng.integers(0, n_pages - n, n)], rng.integers(0, page + 1, n)
    pools = rng.integers(0, 1 << 16, (1, 2, n_pages, page, 64)).astype(np.uint16)
    ls, pool = layers_of(lg, pools, 1, 64, dev)
    p = [dev.up(x, np.int32) for x in (frm, to, rows)]
    dev.check(dev.H.lg_hip_paged_copy(ls, 1, n, *p, None), "paged_copy")
    got = dev.back(pool, pools.shape, np.uint16)
    dev.free()
    moved = np.arange(page)[None, :, None] < rows[:, None, None]
    for which in range(2):
        pools[0, which, to] = np.where(moved, pools[0, which, frm], pools[0, which, to])
    assert np.array_equal(got, pools)
