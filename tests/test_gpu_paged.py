"""The paged cache on the GPU against the definition in 64 bits: extend, attention of one token, eviction."""
import dataclasses
import math

import pytest
import torch

from attention_reference import attend, close

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")
    return torch.device("cuda:0")


def _cache(dev, lengths, hkv, page, dtype, seed, weights=False, spare=3, extra_pages=0, fused=False):
    """A cache of the given filled lengths on shuffled pages, its unfilled slots NaN, table entries behind them -1."""
    import r2omni_amd as ro

    gen = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(lengths), max(need) + extra_pages), -1, dtype=torch.int32, device=dev)
    if fused:
        pool = torch.full((pages, 2, hkv, page, 128), math.nan, dtype=dtype, device=dev)
        k, v = pool[:, 0], pool[:, 1]
    else:
        k, v = (torch.full((pages, hkv, page, 128), math.nan, dtype=dtype, device=dev) for _ in range(2))
    w = torch.full((pages, hkv, page), math.nan, device=dev) if weights else None
    at = 0
    for b, n in enumerate(lengths):
        table[b, : need[b]] = order[at : at + need[b]]
        at += need[b]
        for i in range(need[b]):
            rows = min(page, n - i * page)
            for t in (k, v):
                t[table[b, i].long(), :, :rows] = torch.randn(hkv, rows, 128, generator=gen, device=dev).to(dtype)
            if weights:
                w[table[b, i].long(), :, :rows] = torch.rand(hkv, rows, generator=gen, device=dev)
    return ro.PagedCache(k, v, table, torch.tensor(lengths, dtype=torch.int32, device=dev), w)


def _slots(cache, b, n, pool):
    """[Hkv, n, ...] of a request's first n slots (zeros where no page is mapped), and which are mapped."""
    page = cache.key_pages.shape[2]
    j = torch.arange(n, device=pool.device)
    ids = cache.page_table[b].long()[j // page]
    ok = (ids >= 0) & (ids < pool.shape[0])
    rows = pool[ids.clamp(0, pool.shape[0] - 1), :, j % page].transpose(0, 1)
    return rows, ok


def _query(dev, b, hq, dtype, seed, gain=1.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(b, hq, 128, generator=gen, device=dev) * gain).to(dtype)


def _want(q, cache, window=None, sinks=0, append=None, scale=None):
    """Per request: (out, lse, weights added [Hkv, n], bounds of the three)."""
    hkv = cache.key_pages.shape[1]
    group, results = q.shape[1] // hkv, []
    for b, n in enumerate(cache.lengths.tolist()):
        n = max(0, min(n, cache.capacity))
        k, ok = _slots(cache, b, n, cache.key_pages)
        v, _ = _slots(cache, b, n, cache.value_pages)
        k, v = k.clone(), v.clone()
        if append is not None and n:
            k[:, n - 1], v[:, n - 1] = append[0][b], append[1][b]
        j = torch.arange(n, device=q.device)
        seen = ok if window is None else ok & ((j >= n - window) | (j < sinks))
        parts = []
        for h in range(hkv):
            qs = q[b, h * group : (h + 1) * group]
            if not seen.any():
                zero = torch.zeros(group, 128, dtype=torch.float64, device=q.device)
                none = torch.full((group,), -math.inf, dtype=torch.float64, device=q.device)
                parts.append((zero, none, zero.new_zeros(n), zero, zero[:, 0], zero.new_zeros(n)))
                continue
            o, l, p, tb, tl, rel = attend(qs, k[h], v[h], seen[None].expand(group, -1), q.dtype, scale)
            parts.append((o, l, p.sum(0), tb, tl, (p * (rel + tl + l.abs() * 2.0 ** -22)[:, None]).sum(0) + group * 2.0 ** -24 * p.sum(0)))
        o, l, w, bo, bl, bw = (torch.stack(x) if i in (2, 5) else torch.cat(x) for i, x in enumerate(zip(*parts)))
        results.append((o, l, w, bo, bl, bw, seen))
    return results


def _check(q, cache, window=None, sinks=0, append=None, scale=None):
    import r2omni_amd as ro

    dev = q.device
    k0, v0 = cache.key_pages.clone(), cache.value_pages.clone()
    w0 = None if cache.weight_pages is None else cache.weight_pages.clone()
    want = _want(q, cache, window, sinks, append, scale)
    out, lse = ro.paged_attention(q, cache, window=window, sinks=sinks, append=append, sm_scale=scale)
    torch.cuda.synchronize()
    page = cache.key_pages.shape[2]
    for b, (o, l, w, bo, bl, bw, seen) in enumerate(want):
        close(out[b], o, bo)
        close(lse[b], l, bl)
        n = seen.numel()
        if w0 is not None and n:
            old, mapped = _slots(dataclasses.replace(cache, weight_pages=w0), b, n, w0)
            new, _ = _slots(cache, b, n, cache.weight_pages)
            base = torch.where(seen, old.double(), 0.0)
            if append is not None and seen[n - 1]:
                base[:, n - 1] = 0.0
            total = base + w
            close(torch.where(seen, new, 0.0), torch.where(seen, total, 0.0), bw + total.abs() * 2.0 ** -23 + 2.0 ** -126)
            same = (new == old) | (new.isnan() & old.isnan())
            assert same[:, mapped & ~seen].all()
        if append is not None and n and seen[n - 1]:
            id_, at = cache.page_table[b, (n - 1) // page].long(), (n - 1) % page
            k0[id_, :, at], v0[id_, :, at] = append[0][b], append[1][b]
    for got, was in ((cache.key_pages, k0), (cache.value_pages, v0)):  # nothing but the appended rows has changed
        assert torch.equal(got.contiguous().view(torch.int16), was.contiguous().view(torch.int16))
    return out, lse


def _append(dev, b, hkv, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed + 99)
    return tuple(torch.randn(b, hkv, 128, generator=gen, device=dev).to(dtype) for _ in range(2))


# one slot, page and tile edges and one to either side, odd ones, long next to short ones
LENGTHS = [(1,), (2,), (15, 16, 17), (31, 32, 33), (63, 64, 65, 127, 128, 129), (1000,), (5, 3001, 1), (513, 257)]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_attention_lengths_and_pages(lengths, page):
    dev = _cuda()
    cache = _cache(dev, lengths, 2, page, BF16, seed=page + len(lengths))
    _check(_query(dev, len(lengths), 14, BF16, 1), cache)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (16, 1), (28, 4), (16, 2), (32, 8), (6, 2), (3, 3)])
def test_attention_head_layouts_with_append_and_weights(hq, hkv, dtype):
    dev = _cuda()
    lengths = (70, 1, 333)
    cache = _cache(dev, lengths, hkv, 32, dtype, seed=hq, weights=True)
    _check(_query(dev, 3, hq, dtype, 2), cache, append=_append(dev, 3, hkv, dtype, 2))


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 40), (500, 17), (1 << 40, 2)])
def test_attention_windows_and_sinks(window, sinks, append, weights):
    dev = _cuda()
    lengths = (1, 40, 700, 0, 1203)
    cache = _cache(dev, lengths, 2, 16, BF16, seed=window % 999, weights=weights)
    _check(_query(dev, 5, 8, BF16, 3), cache, window, sinks, _append(dev, 5, 2, BF16, 3) if append else None)


def test_idle_requests_and_lengths_past_the_table():
    """Length 0 (and below) gives zeros and -inf and writes nothing; a length past the table is its capacity."""
    dev = _cuda()
    cache = _cache(dev, (0, 96, 5, 0), 2, 32, BF16, seed=4, weights=True)
    cache.lengths.copy_(torch.tensor([0, 1000, 5, -7], dtype=torch.int32))
    out, lse = _check(_query(dev, 4, 8, BF16, 4), cache, append=_append(dev, 4, 2, BF16, 4))
    assert not out[0].any() and not out[3].any() and (lse[[0, 3]] == -math.inf).all()
    cache.lengths.zero_()
    out, lse = _check(_query(dev, 4, 8, BF16, 4), cache, append=_append(dev, 4, 2, BF16, 4))
    assert not out.any() and (lse == -math.inf).all()


def test_pages_that_are_not_mapped_are_not_seen():
    dev = _cuda()
    cache = _cache(dev, (100, 64, 16), 2, 16, BF16, seed=5, weights=True)
    cache.page_table[0, 2] = -1
    cache.page_table[0, 6] = 1 << 30       # the appended token's page
    cache.page_table[1, 0] = cache.key_pages.shape[0]
    cache.page_table[2] = -1               # nothing of the request is mapped
    out, lse = _check(_query(dev, 3, 8, BF16, 5), cache, append=_append(dev, 3, 2, BF16, 5))
    assert not out[2].any() and (lse[2] == -math.inf).all()


def test_requests_may_share_pages():
    dev = _cuda()
    cache = _cache(dev, (96, 64), 2, 32, BF16, seed=6)
    cache.page_table[1, :2] = cache.page_table[0, :2]
    out, _ = _check(_query(dev, 2, 8, BF16, 6)[:1].expand(2, -1, -1).contiguous(), cache)
    cache.lengths.fill_(64)
    out, _ = _check(_query(dev, 2, 8, BF16, 6)[:1].expand(2, -1, -1).contiguous(), cache)
    assert torch.equal(out[0], out[1])


def test_large_batch_and_large_logits():
    dev = _cuda()
    lengths = [(37 * i) % 211 for i in range(150)]
    cache = _cache(dev, lengths, 1, 16, FP16, seed=7, weights=True)
    _check(_query(dev, 150, 4, FP16, 7, gain=20.0), cache, append=_append(dev, 150, 1, FP16, 7))


def test_strided_pools_queries_and_rows():
    """K and V as views of one pool; queries and rows as slices of one projection."""
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (50, 170), 2, 32, BF16, seed=8, weights=True, fused=True)
    gen = torch.Generator(device=dev).manual_seed(8)
    qkv = torch.randn(2, 1, 12 * 128, generator=gen, device=dev).to(BF16)
    q, k, v = (t.unflatten(2, (-1, 128)).transpose(1, 2) for t in qkv.split((8 * 128, 2 * 128, 2 * 128), dim=2))
    w0 = cache.weight_pages.clone()
    got = ro.paged_attention(q, cache, append=(k, v))
    cache.weight_pages.copy_(w0)
    _check(q[:, :, 0], cache, append=(k[:, :, 0], v[:, :, 0]))
    cache.weight_pages.copy_(w0)
    again = ro.paged_attention(q.contiguous(), cache, append=(k.contiguous(), v.contiguous()))
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_equal_calls_give_equal_bits_and_leave_the_output_beside_them_alone():
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (3000, 17, 900), 4, 64, BF16, seed=9, weights=True)
    q, w0 = _query(dev, 3, 28, BF16, 9), cache.weight_pages.clone()
    want = ro.paged_attention(q, cache)
    w1 = cache.weight_pages.clone()
    for _ in range(3):
        cache.weight_pages.copy_(w0)
        flat = torch.full((3 * 28 * 128 + 16,), 7.0, dtype=BF16, device=dev)
        out = flat[8:-8].view(3, 28, 128)
        lse = torch.full((3 * 28 + 2,), 7.0, device=dev)
        got = ro.paged_attention(q, cache, output=(out, lse[1:-1].view(3, 28)))
        assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
        assert (flat[:8] == 7).all() and (flat[-8:] == 7).all() and lse[0] == 7 and lse[-1] == 7
        assert torch.equal(cache.weight_pages.view(torch.int32), w1.view(torch.int32))


def test_captured_steps_follow_lengths_and_tables():
    """A decode step captured once: lengths advance on the device, a page is mapped when it is needed."""
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (30, 61), 2, 32, BF16, seed=10, weights=True, spare=4, extra_pages=2)
    free = [i for i in range(cache.key_pages.shape[0]) if i not in cache.page_table.unique().tolist()]
    q, (k, v) = _query(dev, 2, 8, BF16, 10), _append(dev, 2, 2, BF16, 10)
    ro.paged_attention(q, dataclasses.replace(cache, weight_pages=None))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.lengths.add_(1)
        out, lse = ro.paged_attention(q, cache, append=(k, v))
    other = dataclasses.replace(cache, key_pages=cache.key_pages.clone(), value_pages=cache.value_pages.clone(),
                                weight_pages=cache.weight_pages.clone(), lengths=cache.lengths.clone())
    for step in range(6):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        for b, n in enumerate(other.lengths.tolist()):
            if n % 32 == 0:
                cache.page_table[b, n // 32] = free.pop()
        graph.replay()
        torch.cuda.synchronize()
        other.lengths.add_(1)
        want = ro.paged_attention(q, other, append=(k, v))
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), step
        for a, b in ((cache.key_pages, other.key_pages), (cache.value_pages, other.value_pages)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        assert torch.equal(cache.weight_pages.view(torch.int32), other.weight_pages.view(torch.int32))


# ---------------------------------------------------------------------------------------- extend
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("rows", [1, 7, 100])
def test_extend(rows, page, dtype):
    """Rows into the newest slots, of padded requests fewer; other slots, and unmapped pages, are left alone."""
    import r2omni_amd as ro

    dev = _cuda()
    lengths = (150, 100, 133, 7)
    cache = _cache(dev, lengths, 3, page, dtype, seed=rows, weights=True)
    cache.page_table[2, 133 // page - 1] = -1
    gen = torch.Generator(device=dev).manual_seed(rows)
    k, v = (torch.randn(4, 3, rows, 128, generator=gen, device=dev).to(dtype) for _ in range(2))
    w = torch.rand(4, 3, rows, generator=gen, device=dev)
    for counts, weights in ((None, w), ((rows, rows // 2, 0, rows), w), (None, None)):
        want = [t.clone() for t in (cache.key_pages, cache.value_pages, cache.weight_pages)]
        for b, n in enumerate(lengths):
            c = rows if counts is None else counts[b]
            for i in range(c):
                j = n - c + i
                id_ = int(cache.page_table[b, j // page]) if j >= 0 else -1
                if id_ >= 0:
                    want[0][id_, :, j % page], want[1][id_, :, j % page] = k[b, :, i], v[b, :, i]
                    want[2][id_, :, j % page] = 0.0 if weights is None else weights[b, :, i]
        ro.paged_extend(cache, k, v, weights=weights,
                        counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev))
        torch.cuda.synchronize()
        assert torch.equal(cache.key_pages.view(torch.int16), want[0].view(torch.int16))
        assert torch.equal(cache.value_pages.view(torch.int16), want[1].view(torch.int16))
        assert torch.equal(cache.weight_pages.view(torch.int32), want[2].view(torch.int32))


def test_extend_strided_rows_and_no_weights():
    import r2omni_amd as ro

    dev = _cuda()
    a = _cache(dev, (40, 90), 2, 32, BF16, seed=11)
    b = dataclasses.replace(a, key_pages=a.key_pages.clone(), value_pages=a.value_pages.clone())
    kv = torch.randn(2, 33, 4 * 128, device=dev).to(BF16)
    k, v = (t.unflatten(2, (-1, 128)).transpose(1, 2) for t in kv.split(256, dim=2))
    ro.paged_extend(a, k, v)
    ro.paged_extend(b, k.contiguous(), v.contiguous())
    assert torch.equal(a.key_pages.view(torch.int16), b.key_pages.view(torch.int16))
    assert torch.equal(a.value_pages.view(torch.int16), b.value_pages.view(torch.int16))
    assert torch.equal(_slots(a, 1, 90, a.key_pages)[0][:, 57:], k[1])


# ----------------------------------------------------------------------------------------- evict
def _kept(w, n, keep, sinks, recent):
    """The slots that one (request, head) keeps, from its weights on the host."""
    if n <= keep:
        return list(range(n))
    order = sorted(range(sinks, n - recent), key=lambda j: (not math.isnan(w[j]), -w[j] if not math.isnan(w[j]) else 0.0, j))
    return sorted([*range(sinks), *range(n - recent, n), *order[: keep - sinks - recent]])


def _check_evict(cache, keep, sinks=0, recent=0, page=None, weights=True):
    import r2omni_amd as ro

    dev = cache.key_pages.device
    batch, hkv, page = cache.page_table.shape[0], cache.key_pages.shape[1], page or cache.key_pages.shape[2]
    target = _cache(dev, [keep] * batch, hkv, page, cache.key_pages.dtype, seed=77, weights=weights)
    target.lengths.fill_(-5)
    before = [None if t is None else t.clone() for t in (target.key_pages, target.value_pages, target.weight_pages)]
    source = [t.clone() for t in (cache.key_pages, cache.value_pages, cache.weight_pages, cache.page_table, cache.lengths)]
    kept = ro.paged_evict(cache, target, keep, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    for b, n in enumerate(cache.lengths.tolist()):
        n = max(0, min(n, cache.capacity))
        w = _slots(cache, b, n, cache.weight_pages)[0].tolist() if n else [[]] * hkv
        for h in range(hkv):
            want = _kept(w[h], n, keep, sinks, recent)
            assert kept[b, h].tolist() == want + [-1] * (keep - len(want)), (b, h)
            for i, j in enumerate(want):
                for pool, got in ((0, before[0]), (1, before[1]), (2, before[2])):
                    if got is not None:
                        src = source[pool][cache.page_table[b, j // cache.key_pages.shape[2]].long(), h, j % cache.key_pages.shape[2]]
                        got[target.page_table[b, i // page].long(), h, i % page] = src
        assert target.lengths[b] == min(n, keep)
    for t, want in zip((target.key_pages, target.value_pages), before):
        assert torch.equal(t.view(torch.int16), want.view(torch.int16))
    if before[2] is not None:
        assert torch.equal(target.weight_pages.view(torch.int32), before[2].view(torch.int32))
    for t, was in zip((cache.key_pages, cache.value_pages, cache.weight_pages, cache.page_table, cache.lengths), source):
        assert torch.equal(t.view(torch.int16) if t.dtype != torch.int32 else t, was.view(torch.int16) if t.dtype != torch.int32 else was)
    return kept


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (16, 4, 8), (33, 0, 0), (64, 64, 0), (64, 0, 64),
                                               (64, 30, 34), (150, 4, 20), (300, 4, 20)])
@pytest.mark.parametrize("page", [16, 64])
def test_evict_counts(keep, sinks, recent, page):
    cache = _cache(_cuda(), (0, 1, 64, 65, 151, 260), 2, page, BF16, seed=keep, weights=True)
    _check_evict(cache, keep, sinks, recent)


def test_evict_ties_zeros_nan_and_infinities():
    dev = _cuda()
    cache = _cache(dev, (200, 200, 200, 200), 2, 16, FP16, seed=12, weights=True)
    w = cache.weight_pages
    ids = cache.page_table.long()
    w[ids[0]] = 0.0                                         # all equal: the first stay
    w[ids[1]] = (w[ids[1]] * 4).round()                     # many equal
    w[ids[2], :, 3] = math.nan
    w[ids[2], :, 4] = math.inf
    w[ids[2], :, 5] = -math.inf
    w[ids[3]] = torch.where(w[ids[3]] > 0.5, 0.0, -0.0)     # -0 equals 0
    for keep in (1, 5, 13, 100, 199):
        _check_evict(cache, keep, 0, 0)
        _check_evict(cache, keep + 8, 3, 5)


def test_evict_to_other_pages_sizes_and_without_weights():
    cache = _cache(_cuda(), (500, 77), 3, 16, BF16, seed=13, weights=True)
    _check_evict(cache, 100, 4, 10, page=64)
    _check_evict(cache, 100, 4, 10, page=32, weights=False)


def test_evict_long():
    cache = _cache(_cuda(), (9000, 4097), 1, 64, BF16, seed=14, weights=True)
    _check_evict(cache, 1030, 4, 100)


def test_evict_into_pages_of_the_same_pool():
    """The target names pages of the source's own pools that no request holds."""
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (100, 90), 2, 16, BF16, seed=15, weights=True, spare=6)
    free = [i for i in range(cache.key_pages.shape[0]) if i not in cache.page_table.unique().tolist()]
    table = torch.tensor([free[:3], free[3:6]], dtype=torch.int32, device=dev)
    target = dataclasses.replace(cache, page_table=table, lengths=torch.zeros_like(cache.lengths))
    kept = ro.paged_evict(cache, target, 40, sinks=2, recent=8)
    for b in range(2):
        src = _slots(cache, b, int(cache.lengths[b]), cache.key_pages)[0]
        dst = _slots(target, b, 40, target.key_pages)[0]
        for h in range(2):
            assert torch.equal(dst[h], src[h, kept[b, h].long()])


# ---------------------------------------------------------------------------- the run of them
def test_prompt_to_decode_with_eviction():
    """A prompt in two chunks, its weights, the cache, an eviction, and decode steps: each stage against the
    definition on the rows that the stages before it left."""
    import r2omni_amd as ro
    from attention_reference import prompt

    dev, page, s, keep = _cuda(), 32, 300, 96
    gen = torch.Generator(device=dev).manual_seed(16)
    q, k, v = (torch.randn(2, n, s, 128, generator=gen, device=dev).to(BF16) for n in (8, 2, 2))
    cache = _cache(dev, (s, s), 2, page, BF16, seed=16, weights=True)
    for start, end in ((0, 171), (171, s)):
        out, lse = ro.prompt_attention(q[:, :, start:end], k[:, :, :end], v[:, :, :end])
        want = prompt(q[:, :, start:end], k[:, :, :end], v[:, :, :end])
        close(out, want[0], want[3])
        close(lse, want[1], want[4])
    w = ro.attention_weights(q[:, :, -64:], k, lse[:, :, -64:])
    ro.paged_extend(cache, k, v, weights=w)
    _check(q[:, :, -1], dataclasses.replace(cache, weight_pages=None))
    target = _cache(dev, (keep + 32,) * 2, 2, page, BF16, seed=17, weights=True)
    kept = ro.paged_evict(cache, target, keep, sinks=4, recent=32)
    assert target.lengths.tolist() == [keep, keep]
    for step in range(5):
        target.lengths.add_(1)
        _check(_query(dev, 2, 8, BF16, 20 + step), target, append=_append(dev, 2, 2, BF16, 20 + step))
    # the weights that decided: those kept and not protected are no smaller than any that went
    for b in range(2):
        for h in range(2):
            stay = set(kept[b, h].tolist())
            mid = [j for j in range(4, s - 32)]
            assert min(w[b, h, j].item() for j in mid if j in stay) >= max(w[b, h, j].item() for j in mid if j not in stay)
