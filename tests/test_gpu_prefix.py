"""Attention over shared prefixes on the GPU against the definition in 64 bits."""
import dataclasses
import math

import pytest
import torch

from prefix_reference import check, want
from test_gpu_paged import BF16, FP16, _cache, _cuda

pytestmark = pytest.mark.gpu


def _query(dev, b, hq, rows, dtype, seed, gain=1.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(b, hq, rows, 128, generator=gen, device=dev) * gain).to(dtype)


def _ints(dev, *values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _both(dev, prefixes, lengths, hkv, page, dtype, seed, prefix_page=None):
    """The prefixes' cache and the requests', on pools of their own."""
    return (_cache(dev, prefixes, hkv, prefix_page or page, dtype, seed),
            _cache(dev, lengths, hkv, page, dtype, seed + 1, extra_pages=1))


# one slot, group, page and tile edges and one to either side, odd ones
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("prefix", [1, 15, 16, 63, 64, 65, 128, 129, 1000, 3001])
def test_prefix_lengths_and_pages(prefix, page):
    dev = _cuda()
    shared, own = _both(dev, (prefix,), (1, 17, 64, 130), 2, page, BF16, prefix)
    check(_query(dev, 4, 14, 1, BF16, 1), own, shared)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (16, 1), (28, 4), (16, 2), (32, 8), (3, 3), (40, 2)])
@pytest.mark.parametrize("rows", [1, 3, 33])
def test_head_layouts(hq, hkv, rows, dtype):
    dev = _cuda()
    shared, own = _both(dev, (333,), (70, 33, 200), hkv, 32, dtype, hq)
    check(_query(dev, 3, hq, rows, dtype, 2), own, shared)


# rows of a KV head below, at and past a row tile of 128, and of several tiles
@pytest.mark.parametrize("rows", [2, 15, 16, 17, 31, 32, 33, 64, 100, 129])
@pytest.mark.parametrize("lengths", [(129, 129), (200, 131), (1000, 700)])
def test_chunks_are_causal_among_their_own(rows, lengths):
    dev = _cuda()
    shared, own = _both(dev, (300,), lengths, 2, 16, BF16, rows)
    check(_query(dev, 2, 8, rows, BF16, 3), own, shared)


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("members", [(3, 2, 4), (9, 0, 0), (0, 9, 0), (0, 0, 9), (1, 1, 1), (0, 0, 0), (4, -3, 2), (2, 100, 5),
                                     ((1 << 31) - 1, (1 << 31) - 1, 1), (-(1 << 31), 3, 3)])
def test_members(members, rows):
    """Requests behind the last share nothing; counts below 0 and past the batch's end are cut off."""
    dev = _cuda()
    shared, own = _both(dev, (200, 64, 700), tuple(40 + 11 * i for i in range(9)), 2, 32, BF16, rows)
    check(_query(dev, 9, 8, rows, BF16, 4), own, shared, _ints(dev, *members))


@pytest.mark.parametrize("rows", [1, 20, 40])
def test_padded_batches(rows):
    dev = _cuda()
    shared, own = _both(dev, (130, 70), (40, 41, 45, 90, 100, 300), 2, 16, BF16, rows)
    counts = _ints(dev, rows, 0, 1, max(1, rows // 2), -5, rows + 7)
    out, lse = check(_query(dev, 6, 14, rows, BF16, 5), own, shared, _ints(dev, 4, 1), counts)
    assert not out[1].any() and (lse[1] == -math.inf).all() and not out[4].any()


# the counted rows of a prefix's requests stand side by side: none, one, all, runs without any, more requests than a wave
@pytest.mark.parametrize("hq,hkv", [(14, 2), (4, 4), (28, 1)])
@pytest.mark.parametrize("rows", [1, 2, 7, 14, 18])
def test_ragged_batches_of_some_prefixes(rows, hq, hkv):
    dev = _cuda()
    gen = torch.Generator().manual_seed(rows)
    batch = 150
    counts = torch.randint(-1, rows + 2, (batch,), generator=gen)
    counts[20:40] = 0
    counts[64:70] = rows
    lengths = torch.randint(0, 60, (batch,), generator=gen).tolist()
    shared, own = _both(dev, (200, 8000, 0, 77), lengths, hkv, 16, BF16, rows)
    q = _query(dev, batch, hq, rows, BF16, 27)
    for members in ((30, 8, 2, 100), (150, 0, 0, 0), (0, 19, 3, 41)):
        check(q, own, shared, _ints(dev, *members), _ints(dev, *counts.tolist()))


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_empty_prefixes_and_requests(rows):
    """A prefix or request without slots; lengths below 0, below the rows and past the table."""
    dev = _cuda()
    shared, own = _both(dev, (100, 64, 130), (64, 64, 64, 64, 64, 64), 2, 32, BF16, rows)
    q = _query(dev, 6, 8, rows, BF16, 6)
    own.lengths.copy_(_ints(dev, 0, 5, -4, 0, 1000, 2))
    own.page_table[4, 2] = own.page_table[0, 0]  # a page for what the length counts
    shared.lengths.copy_(_ints(dev, 100, 0, 1000))
    shared.page_table[2, 3:] = shared.page_table[0, :1]
    for members in ((2, 2, 1), (0, 4, 0), (6, 0, 0)):
        check(q, own, shared, _ints(dev, *members))
    shared.lengths.zero_()
    own.lengths.zero_()
    out, lse = check(q, own, shared, _ints(dev, 2, 2, 2))
    assert not out.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_that_are_not_mapped_are_not_seen(rows):
    dev = _cuda()
    shared, own = _both(dev, (300, 90), (200, 100, 90), 2, 16, BF16, rows)
    shared.page_table[0, [2, 5, 6, 7, 18]] = _ints(dev, -1, 1 << 30, -7, shared.key_pages.shape[0], -1)
    shared.page_table[1] = -1
    own.page_table[0, 0] = -1
    own.page_table[1] = -1
    out, lse = check(_query(dev, 3, 8, rows, BF16, 7), own, shared, _ints(dev, 1, 1))
    assert not out[1].any() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("rows", [1, 7, 40])
def test_without_a_prefix(rows):
    dev = _cuda()
    own = _cache(dev, (1000, 64, 41, 300), 2, 64, FP16, rows)
    check(_query(dev, 4, 14, rows, FP16, 8), own)
    check(_query(dev, 4, 14, rows, FP16, 8), own, query_lengths=_ints(dev, 1, 0, rows, rows))


@pytest.mark.parametrize("rows", [1, 3, 18, 37, 130])
def test_one_long_request(rows):
    """Its slots are shared by all workgroups: each row has the states of many."""
    dev = _cuda()
    own = _cache(dev, (20_001,), 2, 32, BF16, rows)
    q = _query(dev, 1, 14, rows, BF16, 28)
    check(q, own)
    check(q, own, query_lengths=_ints(dev, max(1, rows - 9)))


@pytest.mark.parametrize("rows", [9, 18, 30, 60])
@pytest.mark.parametrize("lengths", [(900, 2500, 61, 130, 1777), (64, 70, 100, 90, 65)])
def test_rows_and_own_slots_in_tiles(rows, lengths):
    """A prefix's rows in one list and the requests' own slots in row tiles, or single waves where they are few."""
    dev = _cuda()
    shared, own = _both(dev, (7000, 6500), lengths, 2, 32, FP16, rows)
    q = _query(dev, 5, 14, rows, FP16, 29)
    check(q, own, shared, _ints(dev, 3, 1))
    check(q, own, shared, _ints(dev, 1, 4), _ints(dev, rows, rows // 2, 0, 1, rows))
    own.lengths[1] = 3  # fewer slots than rows
    check(q, own, shared, _ints(dev, 2, 2))


@pytest.mark.parametrize("rows", [1, 70])
def test_a_token_without_its_axis_and_pools_of_one_tensor(rows):
    """[B, Hq, 128]; prefix and own slots in pages of one pool, K and V views of it; pages of different sizes."""
    dev = _cuda()
    pool = _cache(dev, (500, 90, 33, 250), 2, 32, BF16, 9, fused=True)
    shared = dataclasses.replace(pool, page_table=pool.page_table[:1], lengths=pool.lengths[:1])
    own = dataclasses.replace(pool, page_table=pool.page_table[1:], lengths=pool.lengths[1:])
    q = _query(dev, 3, 8, rows, BF16, 9)
    got = check(q, own, shared)
    if rows == 1:
        token = check(q[:, :, 0], own, shared)
        assert torch.equal(token[0], got[0][:, :, 0]) and torch.equal(token[1], got[1][:, :, 0])
    shared = _cache(dev, (777,), 2, 128, BF16, 10)
    check(q, own, shared)


@pytest.mark.parametrize("rows", [1, 40])
def test_layouts_of_queries_and_results(rows):
    """Views of a fused projection and odd strides, read and written in place or copied."""
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (100,), (64, 41), 2, 16, BF16, 3)
    plain = _query(dev, 2, 8, rows, BF16, 11)
    out, lse = check(plain, own, shared)
    fused = torch.full((2, rows, 12, 128), math.nan, dtype=BF16, device=dev)
    fused[:, :, :8] = plain.transpose(1, 2)
    odd = torch.full((2, 8, rows, 132), math.nan, dtype=BF16, device=dev)
    odd[..., 1:129] = plain
    last = plain.transpose(2, 3).contiguous().transpose(2, 3)
    for q in (fused[:, :, :8].transpose(1, 2), odd[..., 1:129], last):
        got = ro.paged_prefix_attention(q, own, shared)
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)
    room = torch.full((2, rows, 12, 128), 7.0, dtype=BF16, device=dev)
    to = room[:, :, 2:10].transpose(1, 2), torch.empty(2, 8, rows, device=dev)
    got = ro.paged_prefix_attention(plain, own, shared, output=to)
    assert got[0].data_ptr() == to[0].data_ptr() and torch.equal(to[0], out) and torch.equal(to[1], lse)
    assert (room[:, :, :2] == 7.0).all() and (room[:, :, 10:] == 7.0).all()
    if rows == 1:
        flat = torch.empty(2, 8, 128, dtype=BF16, device=dev), torch.empty(2, 8, device=dev)
        ro.paged_prefix_attention(plain[:, :, 0], own, shared, output=flat)
        assert torch.equal(flat[0], out[:, :, 0]) and torch.equal(flat[1], lse[..., 0])


@pytest.mark.parametrize("rows", [1, 40])
def test_large_batches_and_many_prefixes(rows):
    """More requests and prefixes than a wave has lanes."""
    dev = _cuda()
    n = 150 if rows == 1 else 70
    shared, own = _both(dev, tuple(1 + 7 * (i % 13) for i in range(80)), tuple(40 + i % 29 for i in range(n)), 1, 16, BF16, 12)
    members = _ints(dev, *(i % 4 for i in range(80)))
    check(_query(dev, n, 4, rows, BF16, 12), own, shared, members)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scales(scale, rows):
    """A scale that makes every slot count alike, and some that leave one."""
    dev = _cuda()
    shared, own = _both(dev, (300,), (64, 50), 2, 16, BF16, 13)
    check(_query(dev, 2, 8, rows, BF16, 13), own, shared, scale=scale)


@pytest.mark.parametrize("workers", [1, 2, 3, 7, 50, 512, 4096])
@pytest.mark.parametrize("rows,prefix", [(1, 700), (40, 700), (40, 20000), (80, 700)])
def test_any_number_of_workers(rows, prefix, workers):
    """Each within the 64-bit bound: the joins add partial results of other cuts.  Rows of the scratch that a call has no
    right to stay as they were."""
    from r2omni_amd import _lib, paged

    dev = _cuda()
    shared, own = _both(dev, (prefix, 130), (100, 64, 41, 300, 77), 2, 32, BF16, 14)
    q, members = _query(dev, 5, 14, rows, BF16, 14), _ints(dev, 2, 2)
    out, lse = torch.full_like(q, math.nan), torch.full((5, 14, rows), math.nan, device=dev)
    floats = 130 * (512 * workers + (2 * 5 * 14 * rows if 7 * rows < 512 else 0)) + 8 * (1 + max(5, workers))
    scratch = torch.full((floats + 512,), 3.0, device=dev)
    p = _lib.PagedPrefix(cache=paged._params_of(own), prefix=paged._params_of(shared), members=members.data_ptr(), query=q.data_ptr(),
                         out=out.data_ptr(), lse=lse.data_ptr(), q_strides=q.stride()[:3], o_strides=out.stride()[:3], hq=14, rows=rows,
                         sm_scale=128 ** -0.5, scratch=scratch.data_ptr(), scratch_floats=floats, workers=workers)
    _lib.launch("r2o_paged_prefix_attention", p, dev)
    torch.cuda.synchronize()
    o, l, bo, bl = want(q, own, shared, members)
    from attention_reference import close
    close(out, o, bo)
    close(lse, l, bl)
    assert (scratch[floats:] == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,prefix", [(1, 200), (6, 200), (40, 200), (40, 6000)])
def test_infinite_and_nan_values(rows, prefix, dtype):
    """What a row sees of a channel's infinities and NaN is its result there, whatever their weights; what it does not see is
    not."""
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (prefix, 70), (100, 64, 41, 50), 2, 16, dtype, 15)
    q, members = _query(dev, 4, 8, rows, dtype, 15, gain=4.0), _ints(dev, 2, 1)

    def put(cache, row, slot, channel, x):
        cache.value_pages[cache.page_table[row, slot // 16].long(), :, slot % 16, channel] = x

    clean, _ = check(q, own, shared, members)
    put(shared, 0, 3, 5, math.inf)
    put(shared, 0, 199, 6, -math.inf)
    put(shared, 1, 10, 7, math.inf)
    put(shared, 1, 69, 7, -math.inf)
    put(own, 0, 99, 8, math.inf)    # the last row alone
    put(own, 1, 64 - rows, 9, math.nan)
    put(own, 3, 0, 10, math.inf)
    out, lse = ro.paged_prefix_attention(q, own, shared, members=members)
    want_out = clean.clone()
    want_out[:2, ..., 5], want_out[:2, ..., 6], want_out[2, ..., 7] = math.inf, -math.inf, math.nan
    want_out[0, :, -1, 8], want_out[1, ..., 9], want_out[3, ..., 10] = math.inf, math.nan, math.inf
    odd = ~torch.isfinite(want_out)
    assert torch.equal(torch.isnan(out), torch.isnan(want_out))
    assert torch.equal(out[odd & ~torch.isnan(want_out)], want_out[odd & ~torch.isnan(want_out)])
    assert torch.isfinite(lse).all()
    # the others' value is that of the values without them: at most one rounding apart, as sums may be cut elsewhere
    assert torch.equal(out[~odd], clean[~odd])


@pytest.mark.parametrize("rows,prefix", [(1, 200), (40, 200), (40, 6000)])
def test_nan_and_infinite_keys(rows, prefix):
    """A NaN logit makes its row NaN; one of -inf weighs nothing."""
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (prefix,), (100, 64), 2, 16, BF16, 16)
    q = _query(dev, 2, 8, rows, BF16, 16)
    q[..., 0] = 1.0
    clean, clean_lse = check(q, own, shared)
    own.key_pages[own.page_table[0, 6].long(), :, 3] = math.nan  # slot 99, the last row's
    out, lse = ro.paged_prefix_attention(q, own, shared)
    assert out[0, :, -1].isnan().all() and lse[0, :, -1].isnan().all()
    assert torch.equal(out[1], clean[1]) and torch.equal(out[0, :, :-1], clean[0, :, :-1]) and torch.equal(lse[1], clean_lse[1])
    own.key_pages[own.page_table[0, 6].long(), :, 3] = 0.0
    own.key_pages[own.page_table[0, 6].long(), :, 3, 0] = -math.inf
    out, lse = ro.paged_prefix_attention(q, own, shared)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_equal_calls_give_equal_bits_and_write_nothing_else():
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (3001, 500), tuple(30 + 17 * i for i in range(20)), 2, 16, BF16, 17)
    before = [t.clone() for c in (shared, own) for t in (c.key_pages, c.value_pages)]
    for rows in (1, 19, 25):
        q = _query(dev, 20, 14, rows, BF16, 17)
        first = ro.paged_prefix_attention(q, own, shared, members=_ints(dev, 11, 6))
        for _ in range(5):
            again = ro.paged_prefix_attention(q, own, shared, members=_ints(dev, 11, 6))
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    for t, was in zip((t for c in (shared, own) for t in (c.key_pages, c.value_pages)), before):
        assert torch.equal(t.view(torch.int16), was.view(torch.int16))


def test_a_captured_call_follows_lengths_tables_and_members():
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (700, 300), (200, 200, 200, 200), 2, 16, BF16, 18)
    for rows in (1, 20):
        q, members, counts = _query(dev, 4, 14, rows, BF16, 18), _ints(dev, 2, 2), _ints(dev, *(rows,) * 4)
        own.lengths.fill_(40)
        stream = torch.cuda.Stream(dev)
        with torch.cuda.stream(stream):
            ro.paged_prefix_attention(q, own, shared, members=members, query_lengths=counts)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = ro.paged_prefix_attention(q, own, shared, members=members, query_lengths=counts)
        for step in range(6):
            own.lengths.copy_(_ints(dev, 40 + step, 200 - step, 64, 0 if step == 3 else 33))
            shared.lengths.copy_(_ints(dev, 700 - 100 * step, 300 if step % 2 else 0))
            members.copy_(_ints(dev, step % 4, 2))
            counts.copy_(_ints(dev, rows, max(0, rows - step), rows, rows))
            q.normal_()
            graph.replay()
            torch.cuda.synchronize()
            eager = ro.paged_prefix_attention(q, own, shared, members=members, query_lengths=counts)
            assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
            check(q, own, shared, members, counts)


def test_calls_on_two_streams_at_once():
    import r2omni_amd as ro

    dev = _cuda()
    sides = []
    for seed in (19, 20):
        shared, own = _both(dev, (4001,), tuple(50 + 7 * i for i in range(12)), 2, 32, BF16, seed)
        q = _query(dev, 12, 14, 1, BF16, seed)
        sides.append((torch.cuda.Stream(dev), q, own, shared, ro.paged_prefix_attention(q, own, shared)))
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        for stream, q, own, shared, _ in sides:
            with torch.cuda.stream(stream):
                results.append(ro.paged_prefix_attention(q, own, shared))
    torch.cuda.synchronize()
    for i, got in enumerate(results):
        assert all(torch.equal(a, b) for a, b in zip(got, sides[i % 2][4]))


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_past_32_bits_of_bytes_and_elements(rows):
    """Pages whose offsets pass 2^31 and 2^32 elements, in a pool that few pages of are touched."""
    import r2omni_amd as ro

    dev = _cuda()
    page, hkv = 128, 2
    pages = (1 << 32) // (hkv * page * 128) + 40  # 8.6 GB a pool
    k, v = (torch.empty(pages, hkv, page, 128, dtype=BF16, device=dev) for _ in range(2))
    near = _cache(dev, (200,), hkv, page, BF16, 21), _cache(dev, (150, 140), hkv, page, BF16, 22)
    far = []
    at = pages - 1
    for cache in near:
        table = torch.full_like(cache.page_table, -1)
        for r in range(table.shape[0]):
            for c in range(table.shape[1]):
                if cache.page_table[r, c] >= 0:
                    k[at], v[at] = cache.key_pages[cache.page_table[r, c].long()], cache.value_pages[cache.page_table[r, c].long()]
                    table[r, c] = at
                    at -= 1 if at % 2 else (1 << 31) // (hkv * page * 128) - 5
                    at %= pages
        far.append(ro.PagedCache(k, v, table, cache.lengths))
    q = _query(dev, 2, 8, rows, BF16, 21)
    a, b = ro.paged_prefix_attention(q, near[1], near[0]), ro.paged_prefix_attention(q, far[1], far[0])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_the_python_path_gives_the_host_modules_results():
    import r2omni_amd as ro
    import r2omni_amd._lib as lib

    dev = _cuda()
    shared, own = _both(dev, (700, 90), (200, 100, 64), 2, 16, BF16, 23)
    for rows in (1, 40):
        q = _query(dev, 3, 14, rows, BF16, 23)
        for kw in (dict(members=_ints(dev, 1, 1)), dict(members=_ints(dev, 2, 1), query_lengths=_ints(dev, 1, rows, 0), sm_scale=0.1)):
            a = ro.paged_prefix_attention(q, own, shared, **kw)
            real = lib.host()

            class Without:
                def __getattr__(self, name):
                    return getattr(real, name) if name.startswith("prefix_") else lambda *args: None

            lib._HOST = Without()
            try:
                b = ro.paged_prefix_attention(q, own, shared, **kw)
            finally:
                lib._HOST = real
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("lengths,prefix,rows", [((1500, 3), 9001, 1), ((700, 701, 90), 2049, 150), ((2100,), 5, 1)])
def test_longer_ones(lengths, prefix, rows):
    dev = _cuda()
    lengths = tuple(max(n, rows) for n in lengths)
    shared, own = _both(dev, (prefix,), lengths, 2, 64, FP16, 24)
    check(_query(dev, len(lengths), 16, rows, FP16, 24, gain=2.0), own, shared)
