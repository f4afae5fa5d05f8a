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


def test_requests_that_read_one_expanded_row_of_pages():
    """One prefix for four requests of different lengths, by a row of ids expanded for them: the bits of a whole table."""
    import dataclasses

    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (3001,), 2, 32, BF16, seed=3, weights=True)
    lengths = torch.tensor([3001, 17, 0, 1500], dtype=torch.int32, device=dev)
    shared = dataclasses.replace(cache, page_table=cache.page_table.expand(4, -1), lengths=lengths)
    whole = dataclasses.replace(shared, page_table=shared.page_table.contiguous())
    assert shared.page_table.stride(0) == 0 and whole.page_table.stride(0) > 0
    q = _query(dev, 4, 8, BF16, 3)
    plain = dataclasses.replace(shared, weight_pages=None)
    got = _check(q, plain)
    want = ro.paged_attention(q, dataclasses.replace(whole, weight_pages=None))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    targets = [_cache(dev, (64,) * 4, 2, 32, BF16, seed=4, weights=True) for _ in range(2)]
    kept = [ro.paged_evict(c, t, 64, sinks=2, recent=5) for c, t in zip((shared, whole), targets)]
    assert torch.equal(*kept)
    assert torch.equal(*(t.key_pages.view(torch.int16) for t in targets))
    for write in (lambda: ro.paged_attention(q, shared), lambda: ro.paged_evict(whole, dataclasses.replace(shared, lengths=lengths.clone()), 64)):
        with pytest.raises(ValueError, match="one page for several requests"):
            write()


@pytest.mark.parametrize("sinks,recent", [(1 << 62, 1 << 62), ((1 << 63) - 1, 1), (1 << 64, 0)])
def test_protected_slots_past_every_number_are_refused(sinks, recent):
    """By the host module's checks too, whose sums are 64-bit."""
    import r2omni_amd as ro

    dev = _cuda()
    cache, target = (_cache(dev, (70, 90), 2, 16, BF16, seed=s, weights=True) for s in (5, 6))
    with pytest.raises(ValueError, match="at most keep"):
        ro.paged_evict(cache, target, 40, sinks=sinks, recent=recent)


def test_new_rows_whose_offsets_pass_32_bits():
    """A layer's rows as slices of a tensor that holds all layers of long requests, and a token's as a slice of a long prompt:
    requests 2^31 elements apart give the bits of compact ones."""
    import dataclasses

    import r2omni_amd as ro

    dev, far = _cuda(), 1 << 31
    big = torch.empty(2 * far + 4096, dtype=BF16, device=dev)
    small = torch.randn(2, 2, 7, 128, device=dev).to(BF16)
    rows = big.as_strided(small.shape, (far, 7 * 128, 128, 1))
    rows.copy_(small)
    caches = [_cache(dev, (70, 90), 2, 16, BF16, seed=7, weights=True) for _ in range(2)]
    for cache, new in zip(caches, (small, rows)):
        ro.paged_extend(cache, new, new)
    for name in ("key_pages", "value_pages"):
        assert torch.equal(*(getattr(c, name).view(torch.int16) for c in caches))
    near = _query(dev, 2, 4, BF16, 7)
    query = big.as_strided(near.shape, (far, 128, 1), 2048)
    query.copy_(near)
    plain = dataclasses.replace(caches[0], weight_pages=None)
    want = ro.paged_attention(near, plain, append=(small[:, :, 0], small[:, :, 1]))
    got = ro.paged_attention(query, plain, append=(rows[:, :, 0], rows[:, :, 1]))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
