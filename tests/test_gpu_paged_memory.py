"""Copied caches and page tables on the GPU: which memory the paged calls read and write."""
import copy

import pytest
import torch

from test_gpu_paged import BF16, _append, _cache, _check, _cuda, _query

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", [copy.deepcopy, lambda c: c])
def test_calls_on_a_copy_leave_the_original_alone(how):
    """A prompt's cache forked for two continuations, and one whose tensors got other memory."""
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (70, 130), 2, 32, BF16, seed=1, weights=True)
    tensors = (cache.key_pages, cache.value_pages, cache.weight_pages)
    memory = [t.data for t in tensors]
    other = how(cache)
    if other is cache:
        for t in tensors:
            t.data = t.data.clone()
    was = [t.clone() for t in memory]
    new = _append(dev, 2, 2, BF16, 1)
    _check(_query(dev, 2, 8, BF16, 1), other, append=new)
    rows = torch.randn(2, 2, 9, 128, device=dev).to(BF16)
    ro.paged_extend(other, rows, -rows, weights=torch.ones(2, 2, 9, device=dev))
    for b, n in enumerate((70, 130)):
        page, at = other.page_table[b, (n - 1) // 32].long(), (n - 1) % 32
        assert torch.equal(other.key_pages[page, :, at], rows[b, :, 8]) and torch.equal(other.value_pages[page, :, at], -rows[b, :, 8])
    target = _cache(dev, (40, 40), 2, 32, BF16, seed=2, weights=True)
    target = copy.deepcopy(target)
    kept = ro.paged_evict(other, target, 40, recent=9)
    assert (target.lengths == 40).all() and torch.equal(kept[0, 0, 31:], torch.arange(61, 70, dtype=torch.int32, device=dev))
    for t, before in zip(memory, was):
        assert torch.equal(t.nan_to_num(), before.nan_to_num())
