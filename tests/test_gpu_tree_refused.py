"""Steps of which a part is refused: trees that the plan tells to be wrong, and pages that are not enough.  What is refused leaves its sequence at the committed length, and the others as they would be alone."""
import numpy as np
import pytest

from drafts import accept_ref, random_parents, starts_of, tree_accept, tree_plan
from serving import Device, plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(lg):
    if lg.hiplib.device_count() < 1:
        pytest.fail("a test marked gpu ran without a GPU: the HIP path has no CPU fallback")
    d = Device(lg)
    yield d
    d.free()


def test_nothing_is_accepted_in_trees_that_are_refused(dev):
    """Chains whose every token is the one picked: all rows would be passed.  Refused ones keep the committed length, and no token is picked behind them."""
    n = 5
    parent = np.tile(np.arange(n) - 1, 6)
    parent[n + 2] = 3                                              # tree 1: a parent that is a later row
    parent[2 * n + 4] = -1                                         # tree 2: none, in its last row
    parent[5 * n + 1] = 64                                         # tree 5: one that no tree has; too short besides
    start, lens = np.arange(7) * n, np.array([30, 30, 30, 3, 0, 4])
    token, after = np.tile(np.arange(n), 6), np.tile(np.arange(n) + 1, 6)
    status = tree_plan(dev, start, parent, lens, 8)[3]
    assert status.tolist() == [0, 2, 2, 4, 4, 6]
    path, count, ends, last = tree_accept(dev, start, parent, token, after, lens, 8)
    assert count.tolist() == [5, 1, 1, 0, 0, 0]
    assert path[:3].tolist() == [[0, 1, 2, 3, 4, -1, -1, -1], [0] + [-1] * 7, [0] + [-1] * 7] and (path[3:] == -1).all()
    assert ends.tolist() == [30, 25, 25, 3, 0, 4]
    assert last.tolist() == [5, -1, -1, -1, -1, -1]


@pytest.mark.parametrize("n, most", [(3, 1), (7, 64), (300, 9)])
def test_the_closing_plan_takes_the_lengths_of_refused_trees(dev, n, most):
    """A batch in which a third of the trees have a parent that is no earlier row and a third a length below their rows: lengths stay what a plan takes, and the sound trees' are what they are alone."""
    rng = np.random.default_rng(n * 100 + most)
    sizes = rng.integers(1, most + 1, n)
    start = starts_of(sizes)
    parent = np.concatenate([random_parents(rng, int(x)) for x in sizes])
    lens = sizes + rng.integers(0, 50, n)
    kind = np.arange(n) % 3
    for i in range(n):
        if kind[i] == 1 and sizes[i] > 1:
            parent[start[i] + int(rng.integers(1, sizes[i]))] = int(rng.choice([-1, 64, sizes[i] - 1 if sizes[i] > 1 else 5]))
        if kind[i] == 2:
            lens[i] = int(rng.integers(0, sizes[i]))
    token, after = rng.integers(0, 3, parent.size), rng.integers(-1, 3, parent.size)
    status = tree_plan(dev, start, parent, lens, most)[3]
    path, count, ends, last = tree_accept(dev, start, parent, token, after, lens, most)
    ways = accept_ref(start, np.where(parent < 0, -1, parent), token, after, lens, most)
    for i in range(n):
        if status[i] == 0:
            assert path[i].tolist() == ways[0][i].tolist() and (count[i], ends[i], last[i]) == tuple(int(x[i]) for x in ways[1:])
        elif status[i] & 4:
            assert (path[i] == -1).all() and (count[i], ends[i], last[i]) == (0, lens[i], -1)
        else:
            assert path[i].tolist() == [0] + [-1] * (most - 1) and (count[i], ends[i], last[i]) == (1, lens[i] - sizes[i], -1)
    assert (status != 0).any() and (status == 0).any()
    # back from the grown lengths to those, in pages that hold the grown ones
    page, blocks = 16, int(-(-lens.max() // 16)) + 1
    held = -(-lens // page)
    table, at = np.full((n, blocks), -1, np.int32), 0
    for i, m in enumerate(held):
        table[i, :m] = np.arange(at, at + m)
        at += int(m)
    got = plan(dev, page, lens.tolist(), ends.tolist(), table, np.zeros(at + 1, np.int32), 0, 0)
    assert got[2] == 0 and got[5] == int((held - -(-ends // page)).sum())
