"""GPU tests of a step's pages in tables of many columns and of many sequences, against Python lists."""

import random

import pytest

from oracle import step as step_oracle
from test_gpu_pages import check_extend, i32, pool_of, sequences

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,columns", [(1, 1000), (17, 5000), (40, 1000), (250, 300), (256, 512), (257, 512), (300, 800), (1000, 257), (1030, 30), (5000, 20), (20000, 3), (9000, 0)])
def test_release(n, columns):
    """Ranges longer than a wave, or 16 lanes, count at once; sequences of several rounds of the count."""
    from fa2.pages import pages_release
    rng = random.Random(n)
    free, count, table, lens = sequences(rng, n, 16, 16 * columns, columns, min(n * columns // 2, 60000) + 7)
    for full in (False, True):
        first = [0 if full else rng.choice([0, 0, rng.randint(-2, columns)]) for _ in range(n)]
        last = [columns if full else rng.choice([0, -(-x // 16), columns + 2, rng.randint(-3, columns)]) for x in lens]
        pool, t = pool_of(free, count), i32(table).view(n, columns)
        got = pages_release(pool, t, i32(first), i32(last))
        want, want_count = step_oracle.release(free, count, table, first, last)
        assert got.count.tolist() == [want_count] and got.free.tolist() == want
        assert t.tolist() == table and pool.count.tolist() == [count]


@pytest.mark.parametrize("n,columns", [(3000, 5), (20000, 2)])
def test_extend(n, columns):
    rng = random.Random(n)
    free, count, table, lens = sequences(rng, n, 16, 16 * columns, columns, 60000)
    new = [rng.choice([0, 1, rng.randint(0, 20)]) for _ in range(n)]
    check_extend(free, count, table, lens, new, 16, sum(new) + 3)
