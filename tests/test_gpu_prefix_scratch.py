"""Prefix calls that keep a list for each request, with the scratch that they ask for and no more."""
import math

import pytest
import torch

from attention_reference import close
from prefix_reference import check, want
from test_gpu_paged import BF16, FP16, _cuda
from test_gpu_prefix import _both, _ints, _query
from test_prefix_scratch import floats

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("workers", [1, 3, 50, 256])
@pytest.mark.parametrize("counted", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_states_and_notes_stay_within(dtype, counted, workers):
    from r2omni_amd import _lib, paged

    dev, rows, hq = _cuda(), 40, 14
    shared, own = _both(dev, (700, 130), (100, 64, 41, 300, 77), 2, 32, dtype, workers)
    q, members = _query(dev, 5, hq, rows, dtype, workers), _ints(dev, 2, 2)
    counts = _ints(dev, 40, 0, 7, 33, 40) if counted else None
    out, lse = torch.full_like(q, math.nan), torch.full((5, hq, rows), math.nan, device=dev)
    need = floats(workers, 5, 0)
    scratch = torch.full((need + 4096,), 3.0, device=dev)
    p = _lib.PagedPrefix(cache=paged._params_of(own), prefix=paged._params_of(shared), members=members.data_ptr(), query_lengths=_lib.ptr(counts),
                         query=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_strides=q.stride()[:3], o_strides=out.stride()[:3], hq=hq,
                         rows=rows, sm_scale=128 ** -0.5, scratch=scratch.data_ptr(), scratch_floats=need, workers=workers)
    _lib.launch("r2o_paged_prefix_attention", p, dev)
    torch.cuda.synchronize()
    o, l, bo, bl = want(q, own, shared, members, counts)
    close(out, o, bo)
    close(lse, l, bl)
    assert (scratch[need:] == 3.0).all()


def test_a_call_takes_no_more_memory_than_its_lists_use():
    """Rows that could be one list but are not: 300 requests with a prefix each."""
    import r2omni_amd as ro

    dev, batch, hq, rows = _cuda(), 300, 14, 9
    shared, own = _both(dev, (64,) * batch, (20,) * batch, 2, 16, BF16, 1)
    q, members = _query(dev, batch, hq, rows, BF16, 2), _ints(dev, *[1] * batch)
    ro.paged_prefix_attention(q, own, shared, members=members)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ro.paged_prefix_attention(q, own, shared, members=members)
    torch.cuda.synchronize()
    used = torch.cuda.max_memory_allocated() - before - sum(t.numel() * t.element_size() for t in got)
    workers = torch.cuda.get_device_properties(dev).multi_processor_count
    assert used <= 4 * floats(workers, batch, 0) + (4 << 20)
    check(q[:10], *_narrow(own, shared), members[:10])


def _narrow(own, shared):
    import dataclasses

    return [dataclasses.replace(c, page_table=c.page_table[:10], lengths=c.lengths[:10]) for c in (own, shared)]
