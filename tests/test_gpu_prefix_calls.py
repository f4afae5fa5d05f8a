"""Rotation into the cache and attention over shared prefixes as they are used together, and how their calls are made: behind
work that is under way, captured, refused where a derivative would be lost, and on rows that pass the caches by."""
import dataclasses
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from attention_reference import close
from position_reference import rotate
from prefix_reference import check, want
from test_gpu_call_order import _behind_long_work
from test_gpu_paged import BF16, FP16, _cache, _cuda
from test_gpu_position import _new_rows, _rotary
from test_gpu_prefix import _both, _ints, _query
from test_prefix_calls import CALLS, CASES, OUTPUTS, call, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,operand", CASES)
def test_an_operand_that_a_derivative_goes_through_is_refused(name, operand):
    t = operands(_cuda())
    plain = t[operand]
    t[operand] = plain.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(name, t, operand in OUTPUTS)
    with torch.no_grad():
        call(name, t, operand in OUTPUTS)
    with forward_ad.dual_level():
        t[operand] = forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(name, t, operand in OUTPUTS)


@pytest.mark.parametrize("name", CALLS)
def test_plain_operands_are_taken(name):
    for outputs in (False, True):
        call(name, operands(_cuda()), outputs)


def _paths(call):
    """The call by the host module, and by the Python path."""
    import r2omni_amd._lib as lib

    class Without:
        def __getattr__(self, name):
            return real.prefix_plan if name == "prefix_plan" else lambda *args: None

    real = lib.host()
    yield call
    lib._HOST = Without()
    try:
        yield call
    finally:
        lib._HOST = real


def test_calls_wait_for_their_streams_work():
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (3001, 200), (90, 70, 300), 2, 32, BF16, 1)
    members, counts, rotary = _ints(dev, 1, 1), _ints(dev, 20, 7, 20), _rotary(dev, ((16, 24, 24), False), norms=BF16)
    q, k, v = (t.contiguous() for t in _new_rows(dev, 3, 8, 2, 20, BF16, 1))
    pos = torch.randint(0, 9000, (3, 3, 20), device=dev)

    expected = ro.paged_prefix_attention(q, own, shared, members=members, query_lengths=counts)
    for path in _paths(lambda: ro.paged_prefix_attention(q, own, shared, members=members, query_lengths=counts)):
        got, early = _behind_long_work([q, own.key_pages, own.lengths, shared.page_table, shared.lengths, members, counts], path)
        assert early and torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
    expected = ro.qk_position_rope(q, k, pos, rotary, apply_hadamard=True)
    for path in _paths(lambda: ro.qk_position_rope(q, k, pos, rotary, apply_hadamard=True)):
        got, early = _behind_long_work([q, k, pos, rotary.inv_freq, rotary.k_norm_weight], path)
        assert early and torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
    cache = dataclasses.replace(own, key_pages=own.key_pages.clone(), value_pages=own.value_pages.clone())
    expected = ro.paged_rope_extend(cache, q, k, v, rotary, positions=pos, counts=counts)
    for path in _paths(lambda: ro.paged_rope_extend(other, q, k, v, rotary, positions=pos, counts=counts)):
        other = dataclasses.replace(own, key_pages=own.key_pages.clone(), value_pages=own.value_pages.clone())
        got, early = _behind_long_work([q, k, v, pos, counts, other.lengths, other.page_table], path)
        assert early and torch.equal(got, expected)
        for a, b in ((other.key_pages, cache.key_pages), (other.value_pages, cache.value_pages)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hkv,sections,norm", [(8, 2, ((16, 24, 24), False), False), (14, 2, ((24, 20, 20), True), True), (4, 4, ((64,), False), False)])
def test_a_prefix_its_questions_and_their_answers(dtype, hq, hkv, sections, norm):
    """A prefix comes in chunks, questions of several lengths follow, then answers token by token: each result against the whole
    computation in 64 bits on the rows as they lie in the cache, whose keys are checked against the rotation."""
    import r2omni_amd as ro

    dev, page, axes = _cuda(), 16, len(sections[0])
    gen = torch.Generator(device=dev).manual_seed(3)
    rotary = _rotary(dev, sections, norms=dtype if norm else None)
    pages = 64
    k_pool, v_pool = (torch.full((pages, hkv, page, 128), math.nan, dtype=dtype, device=dev) for _ in range(2))
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    prefix = ro.PagedCache(k_pool, v_pool, order[:12].view(1, 12), _ints(dev, 0))
    own = ro.PagedCache(k_pool, v_pool, order[12:36].view(4, 6), _ints(dev, 0, 0, 0, 0))

    def rows(b, s):
        x = torch.randn(b, s, hq + 2 * hkv, 128, generator=gen, device=dev).to(dtype).transpose(1, 2)
        return x[:, :hq], x[:, hq : hq + hkv], x[:, hq + hkv :]

    def positions(b, s, first):
        """Each axis its own, as of patches: the first row's a request, then steps of the axis' own."""
        at = torch.arange(s, device=dev)
        return torch.stack([(torch.tensor(first, device=dev)[:, None] + at // (a + 1)) for a in range(axes)])

    kept = []  # (table row's cache, row, first slot, keys' rotation and bound)

    def extend(cache, q, k, v, pos, counts=None):
        got = ro.paged_rope_extend(cache, q, k, v, rotary, positions=pos, counts=counts)
        (wq, bq), (wk, bk) = rotate(q, pos, rotary, rotary.q_norm_weight), rotate(k, pos, rotary, rotary.k_norm_weight)
        for b in range(q.shape[0]):
            count = q.shape[2] if counts is None else int(counts[b])
            close(got[b, :, :count], wq[b, :, :count], bq[b, :, :count])
            kept.append((cache, b, int(cache.lengths[b]) - count, wk[b, :, :count], bk[b, :, :count], v[b, :, :count]))
        return got

    before = 0
    for s in (70, 1, 90):  # the prefix, as a chunked prompt: causal attention over its own pages
        prefix.lengths.add_(s)
        q = extend(prefix, *rows(1, s), positions(1, s, [before]))
        check(q, prefix)
        before += s
    counts = _ints(dev, 9, 33, 0, 20)
    own.lengths.add_(counts)
    q = extend(own, *rows(4, 33), positions(4, 33, [before, before, 0, 7]), counts)
    members = _ints(dev, 3)  # the last request shares nothing
    out, lse = check(q, own, prefix, members, counts)
    assert not out[2].any() and (lse[2] == -math.inf).all()
    for step in range(3):
        own.lengths.add_(1)
        q = extend(own, *rows(4, 1), positions(4, 1, [before + 9 + step, before + 33 + step, before + step, 27 + step]))
        check(q[:, :, 0], own, prefix, members)
        check(q, own, prefix, members)
    for cache, b, first, k, bound, v in kept:
        for i in range(k.shape[1]):
            id_, at = int(cache.page_table[b, (first + i) // page]), (first + i) % page
            close(k_pool[id_, :, at], k[:, i], bound[:, i])
            assert torch.equal(v_pool[id_, :, at], v[:, i])


def test_a_prefix_of_no_use_leaves_the_paged_attention():
    """One token a request without a prefix, and with one of no slots: the results of the operator for single tokens, within both
    bounds."""
    import r2omni_amd as ro

    dev = _cuda()
    shared, own = _both(dev, (64,), (700, 33, 1, 130), 2, 32, BF16, 4)
    shared.lengths.zero_()
    q = _query(dev, 4, 8, 1, BF16, 4)[:, :, 0]
    out, lse = ro.paged_attention(q, own)
    _, _, bound, bound_lse = want(q[:, :, None], own)
    for got in (check(q, own), check(q, own, shared)):
        close(got[0], out.double(), 2 * bound[:, :, 0])
        close(got[1], lse.double(), 2 * bound_lse[:, :, 0])


def test_two_captured_graphs_replay_at_once():
    """Each has its scratch: replays on two streams give what each call gives by itself."""
    import r2omni_amd as ro

    dev = _cuda()
    sides = []
    for seed, rows in ((5, 1), (6, 12)):
        shared, own = _both(dev, (2001, 300), tuple(40 + 9 * i for i in range(10)), 2, 32, BF16, seed)
        q, members, stream = _query(dev, 10, 14, rows, BF16, seed), _ints(dev, 6, 3), torch.cuda.Stream(dev)
        expected = ro.paged_prefix_attention(q, own, shared, members=members)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = [ro.paged_prefix_attention(q, own, shared, members=members) for _ in range(2)]
        sides.append((graph, stream, got, expected, (shared, own, q, members)))
    for _ in range(10):
        for graph, stream, got, _, _ in sides:
            with torch.cuda.stream(stream):
                for out, lse in got:
                    out.fill_(7.0)
                    lse.fill_(7.0)
                graph.replay()
        torch.cuda.synchronize()
        for _, _, got, expected, _ in sides:
            for out, lse in got:
                assert torch.equal(out, expected[0]) and torch.equal(lse, expected[1])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_calls_give_the_rows_of_small_ones(dtype):
    """600,000 rows (154 MB), which pass the caches by, against calls of a hundredth: one row's result does not depend on the call's
    size; some rows against 64 bits."""
    import r2omni_amd as ro

    dev, b, s, hq, hkv = _cuda(), 3, 12_501, 12, 2
    rotary = _rotary(dev, ((16, 24, 24), False), norms=dtype)
    q, k, v = _new_rows(dev, b, hq, hkv, s, dtype, 7)
    pos = torch.randint(0, 1 << 30, (3, b, s), device=dev)
    for apply_hadamard in (False, True):
        got = ro.qk_position_rope(q, k, pos, rotary, apply_hadamard=apply_hadamard)
        for at in range(0, s, 1000):
            part = ro.qk_position_rope(q[:, :, at : at + 1000], k[:, :, at : at + 1000], pos[:, :, at : at + 1000], rotary,
                                       apply_hadamard=apply_hadamard)
            for x, y in zip(got, part):
                assert torch.equal(x[:, :, at : at + 1000], y)
        for x, y, w in zip(got, (q, k), (rotary.q_norm_weight, rotary.k_norm_weight)):
            close(x[:, :, -20:], *rotate(y[:, :, -20:].contiguous(), pos[:, :, -20:], rotary, w, apply_hadamard))
    del got, part
    counts = _ints(dev, s, s - 4000, 0)
    large, small = ([_cache(dev, (s + 30, s + 7, 50), hkv, 64, dtype, 8, weights=True) for _ in range(2)])
    out = ro.paged_rope_extend(large, q, k, v, rotary, positions=pos, counts=counts)
    for i in range(2):  # the same rows by the rotation, and the plain writing
        n = int(counts[i])
        one = dataclasses.replace(small, page_table=small.page_table[i : i + 1], lengths=small.lengths[i : i + 1])
        x = [ro.qk_position_rope(q[i : i + 1, :, at : min(at + 1000, n)], k[i : i + 1, :, at : min(at + 1000, n)],
                                 pos[:, i : i + 1, at : min(at + 1000, n)], rotary) for at in range(0, n, 1000)]
        assert torch.equal(out[i : i + 1, :, :n], torch.cat([a for a, _ in x], 2)) and not out[i, :, n:].any()
        ro.paged_extend(one, torch.cat([a for _, a in x], 2), v[i : i + 1, :, :n])
    assert not out[2].any()
    for a, c in ((large.key_pages, small.key_pages), (large.value_pages, small.value_pages)):
        assert torch.equal(a.view(torch.int16), c.view(torch.int16))
    assert torch.equal(large.weight_pages.nan_to_num(nan=-1.0), small.weight_pages.nan_to_num(nan=-1.0))
