"""Numbers of tokens that do not fit their sums or types, on the CPU."""
import ctypes

import pytest

from r2omni_amd import _lib
from test_paged_refusals import _evict


@pytest.mark.parametrize("sinks,recent", [(1 << 62, 1 << 62), ((1 << 63) - 1, 1), (1, (1 << 63) - 1), ((1 << 62) + 3, (1 << 62) + 3)])
def test_protected_slots_whose_sum_passes_64_bits_are_refused(sinks, recent):
    assert _lib.load().r2o_paged_evict(ctypes.byref(_evict(sinks=sinks, recent=recent)), None) == 1
