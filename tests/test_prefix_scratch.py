"""A prefix call's scratch: states of whole rows where the rows of a prefix's requests are one list, and none where each request has
a list of its own.  On the CPU; test_gpu_prefix_scratch.py runs such calls."""
import ctypes

import pytest

from r2omni_amd import _lib
from test_prefix_refusals import _attention, _plain


def floats(workers, batch, rows_of_states):
    return 130 * (512 * workers + rows_of_states) + 8 * (1 + max(batch, workers))


# requests, KV heads, heads, rows, own slots, prefixes, their slots, whether counts are given
APART = [(512, 4, 28, 9, 1024, 512, 128, 0),      # a prefix for each request: nothing is read once for several
         (16, 4, 28, 12, 2048, 16, 32000, 0),     # a table of prefixes for a batch that may be of all
         (16, 4, 28, 4, 512, 0, 0, 0),            # 28 rows without a prefix
         (64, 4, 28, 18, 2048, 1, 2112, 0),       # a short prefix, 126 rows
         (5, 2, 14, 40, 320, 2, 704, 0)]
MERGED = [(24, 4, 28, 1, 1408, 1, 32641, 0), (16, 4, 28, 12, 2048, 1, 32000, 0), (1, 4, 28, 18, 32000, 0, 0, 0), (5, 2, 14, 40, 320, 2, 20000, 0)]


@pytest.mark.parametrize("call", APART + MERGED)
def test_the_scratch_is_what_the_call_uses(call):
    batch, hkv, hq, rows, slots, prefixes, shared, counted = call
    plan = _lib.host().prefix_plan(*call, 256)
    assert plan[1] == floats(plan[0], batch, 2 * batch * hq * rows if call in MERGED else 0)
    few = _attention(cache=_plain(batch=batch, hkv=hkv, max_pages=slots // 16, table_stride=slots // 16),
                     prefix=_plain(batch=prefixes, hkv=hkv, max_pages=max(1, shared // 16), table_stride=max(1, shared // 16)), members=0x16000,
                     hq=hq, rows=rows, workers=plan[0], scratch_floats=plan[1] - 1)
    assert _lib.load().r2o_paged_prefix_attention(ctypes.byref(few), None) == 1
