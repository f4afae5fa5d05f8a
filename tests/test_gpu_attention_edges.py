"""Calls of the prompt and paged operators that their ordinary tests do not make: NaN in a query, rows longer than a
workgroup's registers, more requests than a wave has lanes, two captured steps on one cache, equal rows in one call."""
import dataclasses
import math

import pytest
import torch

from attention_reference import close
from test_gpu_paged import BF16, FP16, _append, _cache, _check, _check_evict, _cuda, _query, _want
from test_gpu_prompt import _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sq,sk", [(40, 40), (8, 3000)])
def test_a_nan_query_row_is_nan_in_its_results_and_nowhere_else(sq, sk, dtype):
    """Every logit of such a row is NaN: its output, statistic and weights are, not the zeros of a row that sees no key."""
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 2, 8, 2, sq, sk, dtype, seed=1)
    clean, clean_lse = ro.prompt_attention(q, k, v)
    bad = q.clone()
    bad[1, 3, 5, 17] = math.nan
    out, lse = ro.prompt_attention(bad, k, v)
    hit = torch.zeros(q.shape[:3], dtype=torch.bool, device=q.device)
    hit[1, 3, 5] = True
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    w, clean_w = ro.attention_weights(bad, k, lse), ro.attention_weights(q, k, clean_lse)
    n = sk - sq + 6  # keys that row 5 sees
    assert w[1, 0, :n].isnan().all()
    assert torch.equal(w[0], clean_w[0]) and torch.equal(w[1, 1], clean_w[1, 1]) and torch.equal(w[1, 0, n:], clean_w[1, 0, n:])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_nan_query_token_is_nan_in_its_results_and_nowhere_else(dtype):
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (40, 3000), 2, 32, dtype, seed=2, weights=True)
    q = _query(dev, 2, 8, dtype, 2)
    plain = dataclasses.replace(cache, weight_pages=None)
    clean, clean_lse = ro.paged_attention(q, plain)
    q[1, 2, 100] = math.nan
    w0 = cache.weight_pages.clone()
    out, lse = ro.paged_attention(q, cache)
    hit = torch.zeros(2, 8, dtype=torch.bool, device=dev)
    hit[1, 2] = True
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    ids, was = cache.page_table[1].long(), cache.weight_pages
    assert was[ids, 0].flatten()[:3000].isnan().all()
    assert not was[ids, 1].flatten()[:3000].isnan().any() and (was[ids, 1] >= w0[ids, 1]).flatten()[:3000].all()


@pytest.mark.parametrize("keep,sinks,recent", [(300, 4, 100), (70, 0, 0)])
def test_evict_rows_behind_the_registers(keep, sinks, recent):
    """65536 slots are held in registers; what lies behind is read again.  Lengths on both sides of that."""
    cache = _cache(_cuda(), (65536, 65537, 70001, 16385, 4097), 1, 128, BF16, seed=3, weights=True)
    _check_evict(cache, keep, sinks, recent)


@pytest.mark.parametrize("n", [300, 20000, 70001])
def test_evict_when_nearly_all_weights_are_equal(n):
    """Slots that no query weighed, and a few of every sign and size: a threshold among equal ones, and just beside them."""
    dev = _cuda()
    cache = _cache(dev, (n,), 1, 64, BF16, seed=4, weights=True)
    w, ids = cache.weight_pages, cache.page_table[0].long()
    w[ids] = 0.0
    for i, x in enumerate((1e-45, 1e-38, 1.0, 3e38, math.inf, -1e-45, -1.0, -math.inf)):
        j = (7919 * (i + 1)) % n
        w[ids[j // 64], 0, j % 64] = x
    for keep in (1, 4, 5, 6, 120):
        _check_evict(cache, keep)
    _check_evict(cache, 40, 10, 30)


@pytest.mark.parametrize("n", [200, 5000, 20000])
def test_evict_nan_of_every_sign_and_payload(n):
    """All NaN are equal and the largest, the earlier first; what lies behind the filled slots may be any of them."""
    dev = _cuda()
    cache = _cache(dev, (n,), 1, 64, BF16, seed=11, weights=True)
    w, ids = cache.weight_pages.view(torch.int32), cache.page_table[0].long()
    for i, bits in enumerate((0x7FFFFFFF, -1, -0x400000, 0x7F800001, 0x7FC00000)):
        j = (6101 * (i + 1)) % n
        w[ids[j // 64], 0, j % 64] = bits
    if n % 64:
        w[ids[-1], 0, n % 64 :] = torch.tensor([0x7FFFFFFF, -1], dtype=torch.int32, device=dev).repeat(32)[: 64 - n % 64]
    for keep in (1, 3, 5, 6, 70):
        _check_evict(cache, keep)


def test_more_requests_than_lanes_with_windows_sinks_and_weights():
    dev = _cuda()
    lengths = tuple((37 * i) % 130 for i in range(150))
    cache = _cache(dev, lengths, 2, 16, BF16, seed=5, weights=True)
    _check(_query(dev, 150, 8, BF16, 5), cache, window=40, sinks=3, append=_append(dev, 150, 2, BF16, 5))
    _check(_query(dev, 150, 8, BF16, 6), cache)


def test_two_captured_steps_share_a_cache_beside_eager_calls():
    """Each graph holds its own scratch: replayed in any order, between eager calls, all give one result."""
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (4001, 70), 2, 32, BF16, seed=7, weights=True)
    queries = [_query(dev, 2, 8, BF16, 70 + i) for i in range(2)]
    stream, graphs, results = torch.cuda.Stream(), [], []
    with torch.cuda.stream(stream):
        for q in queries:
            ro.paged_attention(q, cache)
    torch.cuda.synchronize()
    for q in queries:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(ro.paged_attention(q, cache))
        graphs.append(graph)
    cache.weight_pages.zero_()
    want = [ro.paged_attention(q, dataclasses.replace(cache, weight_pages=None)) for q in queries]
    for turn in (0, 1, 1, 0, 0, 1):
        results[turn][0].zero_()
        graphs[turn].replay()
        eager = ro.paged_attention(queries[1 - turn], dataclasses.replace(cache, weight_pages=None))
        torch.cuda.synchronize()
        for got, exact in zip(results[turn] + eager, want[turn] + want[1 - turn]):
            assert torch.equal(got, exact)
    # six steps: each slot's weights are the sums of three of either query
    for b, n in enumerate((4001, 70)):
        total, bound = 0.0, 0.0
        for q in queries:
            w = _want(q, cache)[b]
            total, bound = total + 3 * w[2], bound + 3 * w[5]
        page = cache.page_table[b].long()[torch.arange(n, device=dev) // 32]
        got = cache.weight_pages[page, :, torch.arange(n, device=dev) % 32].T
        close(got, total, bound + 6 * 2.0 ** -24 * total + 2.0 ** -126)


def test_rows_and_heads_that_are_one_memory():
    """Expanded inputs (strides of 0): one key head's rows for all heads, one query for all requests."""
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 1, 4, 1, 70, 300, BF16, seed=8)
    q3, k3, v3 = q.expand(3, -1, -1, -1), k.expand(3, 2, -1, -1), v.expand(3, 2, -1, -1)
    want = ro.prompt_attention(q3.contiguous(), k3.contiguous(), v3.contiguous())
    got = ro.prompt_attention(q3, k3, v3)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert torch.equal(ro.attention_weights(q3, k3, got[1]), ro.attention_weights(q3.contiguous(), k3.contiguous(), want[1]))


def test_the_longest_scratch_is_joined_in_one_order():
    """Splits, joined by the second launch: equal calls on two streams at once give equal bits."""
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 1, 16, 2, 24, 9000, BF16, seed=9)
    want = ro.prompt_attention(q, k, v)
    weights = ro.attention_weights(q, k, want[1])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                out, lse = ro.prompt_attention(q, k, v)
                got.append((out, lse, ro.attention_weights(q, k, lse)))
    torch.cuda.synchronize()
    for out, lse, w in got:
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and torch.equal(w, weights)


def test_evict_short_requests_of_long_tables():
    """What a lane holds goes by the request, not by what the table could hold."""
    cache = _cache(_cuda(), (20000, 4096, 4097, 16384, 16385, 50), 1, 128, BF16, seed=10, weights=True)
    _check_evict(cache, 100, 4, 20)


def test_pages_whose_offsets_pass_32_bits():
    """The same rows in a small pool and in one whose pages lie 2^30 elements apart: equal bits from every call."""
    import r2omni_amd as ro

    dev, n, page = _cuda(), 280, 64
    small = _cache(dev, (n,), 2, page, BF16, seed=12, weights=True, spare=0)
    pages, stride = small.key_pages.shape[0], 1 << 30
    wide = []
    for pool in (small.key_pages, small.value_pages):
        big = torch.empty((pages - 1) * stride + 2 * page * 128, dtype=BF16, device=dev)
        view = big.as_strided(pool.shape, (stride, page * 128, 128, 1))
        view.copy_(pool)
        wide.append(view)
    assert 2 * (pages - 1) * stride > 1 << 32
    table, lengths = small.page_table, small.lengths
    large = ro.PagedCache(*wide, table, lengths.clone(), small.weight_pages.clone())
    q, new = _query(dev, 1, 8, BF16, 12), _append(dev, 1, 2, BF16, 12)
    k, v = (torch.randn(1, 2, 70, 128, device=dev).to(BF16) for _ in range(2))
    results = []
    for cache in (small, large):
        ro.paged_extend(cache, k, v, weights=torch.ones(1, 2, 70, device=dev))
        out = ro.paged_attention(q, cache, append=new)
        target = _cache(dev, (64,), 2, page, BF16, seed=13, weights=True)
        kept = ro.paged_evict(cache, target, 64, sinks=2, recent=5)
        results.append((*out, kept, target.key_pages.view(torch.int16), target.value_pages.view(torch.int16), target.weight_pages[:1]))
    torch.cuda.synchronize()
    for x, y in zip(*results):
        assert torch.equal(x, y) or (x.is_floating_point() and torch.equal(x.nan_to_num(), y.nan_to_num()))
    for pool, view in zip((small.key_pages, small.value_pages), wide):
        assert torch.equal(pool.view(torch.int16), view.contiguous().view(torch.int16))


def test_requests_whose_offsets_pass_32_bits():
    """A prompt's requests 2^31 elements apart, and rows 2^24 apart: the bits of compact ones."""
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 2, 4, 2, 90, 200, BF16, seed=13)
    want = ro.prompt_attention(q, k, v)
    weights = ro.attention_weights(q, k, want[1])

    def spread(t, strides):
        big = torch.empty(sum((n - 1) * s for n, s in zip(t.shape, strides)) + 1, dtype=t.dtype, device=t.device)
        view = big.as_strided(t.shape, strides)
        view.copy_(t)
        return view

    for far in ((1 << 31, 200 * 128, 128, 1), (128, 256, 1 << 24, 1)):
        k2, v2 = spread(k, far), spread(v, far)
        q2 = spread(q, (1 << 31, 90 * 128, 128, 1))
        got = ro.prompt_attention(q2, k2, v2)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert torch.equal(ro.attention_weights(q2, k2, got[1]), weights)
        del k2, v2, q2
