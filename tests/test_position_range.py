"""How many tokens a rotation takes: a launch has at most 2^32 - 1 lanes, 256 for 16 tokens.  On the CPU; more are refused before any
launch."""
import ctypes

import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib
from test_paged_refusals import I32, _c_cache, _rows, _tensors, cache  # noqa: F401
from test_position_refusals import _extend, _rope, _rotary

MOST = (1 << 28) - 16


@pytest.mark.parametrize("batch,tokens", [(1, MOST + 1), (1, 1 << 28), (16, 1 << 24), (3, 1 << 27), (1 << 20, 1 << 10), (1, 1 << 31)])
def test_more_tokens_than_a_launch_has_lanes_for_are_refused(batch, tokens):
    q, k = (_rows(1, h, 1, 128).expand(batch, h, tokens, 128) for h in (4, 2))
    at = torch.zeros(1, 1, 1, dtype=I32).expand(1, batch, tokens)
    with pytest.raises(ValueError, match="tokens"):
        ro.qk_position_rope(q, k, at, _rotary(mrope_section=(64,)))
    with pytest.raises(ValueError, match="tokens"):
        ro.qk_position_rope(q, k, at, _rotary(mrope_section=(64,)), output=(q, k))
    assert _lib.load().r2o_position_rope(ctypes.byref(_rope(batch=batch, tokens=tokens)), None) == 1


def test_more_rows_of_a_paged_call_are_refused(cache):  # noqa: F811
    """A table of 2^28 slots for each of two requests."""
    wide = ro.PagedCache(**_tensors(page_table=torch.zeros(2, 1 << 24, dtype=I32)))
    for rows in (1 << 27, 1 << 28):
        q, k = (_rows(2, h, 1, 128).expand(2, h, rows, 128) for h in (4, 2))
        with pytest.raises(ValueError, match="tokens"):
            ro.paged_rope_extend(wide, q, k, k, _rotary())
        c = _c_cache(max_pages=1 << 24, table_stride=1 << 24)
        assert _lib.load().r2o_paged_rope_extend(ctypes.byref(_extend(cache=c, rows=rows)), None) == 1
