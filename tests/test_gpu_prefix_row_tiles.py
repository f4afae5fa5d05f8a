"""Prefix calls whose rows fill a row tile of 256, half of one or a wave's 32 to the last row, and one row to either side: in a
prefix's list, in the requests' own, and in a list of requests."""
import pytest

from prefix_reference import check
from test_gpu_paged import BF16, FP16, _cache, _cuda
from test_gpu_prefix import _both, _ints, _query

pytestmark = pytest.mark.gpu

EDGES = [31, 32, 33, 127, 128, 129, 255, 256, 257, 511, 512, 513]


@pytest.mark.parametrize("rows", EDGES)
def test_rows_of_a_prefix_in_one_list(rows):
    """As many requests of a token; then of up to three rows, as many in all."""
    dev = _cuda()
    shared, own = _both(dev, (700, 90), tuple(1 + i % 9 for i in range(rows + 5)), 1, 16, BF16, rows)
    check(_query(dev, rows + 5, 1, 1, BF16, 1), own, shared, _ints(dev, rows, 4))
    counts, left = [], rows
    while left:
        counts.append(min(left, 1 + len(counts) % 3))
        left -= counts[-1]
    n = len(counts)
    shared, own = _both(dev, (700, 90), (7,) * (n + 1), 1, 16, FP16, rows)
    check(_query(dev, n + 1, 1, 3, FP16, 2), own, shared, _ints(dev, n, 1), _ints(dev, *counts, 2))


@pytest.mark.parametrize("rows", EDGES)
def test_rows_of_a_request_over_its_own_slots(rows):
    dev = _cuda()
    own = _cache(dev, (rows + 900, rows, rows + 70), 2, 32, BF16, rows)
    check(_query(dev, 3, 2, rows, BF16, 3), own)
    check(_query(dev, 3, 2, rows + 3, BF16, 4), own, query_lengths=_ints(dev, rows, rows - 1, rows + 1))
    group = 7  # query heads of a KV head: the rows are those of all
    own = _cache(dev, (rows + 300, 50), 1, 16, FP16, rows)
    check(_query(dev, 2, group, -(-rows // group), FP16, 5), own)


@pytest.mark.parametrize("rows", EDGES)
def test_rows_of_a_request_behind_its_prefix(rows):
    """A short prefix for each: nothing to gain from one list."""
    dev = _cuda()
    shared, own = _both(dev, (64, 200, 1), (rows, rows + 100, 40), 2, 16, BF16, rows)
    check(_query(dev, 3, 2, rows, BF16, 6), own, shared, _ints(dev, 1, 1, 1))
    check(_query(dev, 3, 2, rows + 2, BF16, 7), own, shared, _ints(dev, 1, 1, 1), _ints(dev, rows + 1, rows, rows - 1))
