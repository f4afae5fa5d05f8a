"""Calls on a stream whose operands are still being made, and sums over other numbers of splits than the calls choose."""
import dataclasses

import pytest
import torch

from attention_reference import close, prompt
from test_gpu_paged import BF16, _append, _cache, _cuda, _query
from test_gpu_prompt import _rows

pytestmark = pytest.mark.gpu


def _behind_long_work(operands, call):
    """call() on a side stream, where long work comes before the operands' values; its results, and whether the long work was
    still running when the call had returned."""
    dev = operands[0].device
    values = [t.clone() for t in operands]
    for t in operands:
        t.zero_()
    x = torch.randn(4096, 4096, device=dev)
    y, side, made = torch.empty_like(x), torch.cuda.Stream(dev), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(60):  # some 100 ms
            torch.mm(x, x, out=y)
        for t, v in zip(operands, values):
            t.copy_(v)
        made.record()
        got = call()
        early = not made.query()
    torch.cuda.synchronize()
    return got, early


def _both_paths(call):
    """The call by the host module, and by the Python path."""
    import r2omni_amd._lib as lib

    class Without:
        def __getattr__(self, name):
            found = getattr(real, name)
            return found if name in ("attention_splits", "weight_splits", "paged_workers") else lambda *args: None

    real = lib.host()
    yield call
    lib._HOST = Without()
    try:
        yield call
    finally:
        lib._HOST = real


def test_prompt_calls_wait_for_their_streams_work():
    import r2omni_amd as ro

    q, k, v = _rows(_cuda(), 2, 8, 2, 256, 900, BF16, seed=1)
    want, want_lse = ro.prompt_attention(q, k, v)
    weights = ro.attention_weights(q, k, want_lse)
    for call in _both_paths(lambda: ro.prompt_attention(q, k, v)):
        (out, lse), early = _behind_long_work([q, k, v], call)
        assert early and torch.equal(out, want) and torch.equal(lse, want_lse)
    for call in _both_paths(lambda: ro.attention_weights(q, k, want_lse)):
        got, early = _behind_long_work([q, want_lse], call)
        assert early and torch.equal(got, weights)


def test_paged_calls_wait_for_their_streams_work():
    import r2omni_amd as ro

    dev = _cuda()
    start = _cache(dev, (3001, 70), 2, 32, BF16, seed=2, weights=True)
    q, new = _query(dev, 2, 8, BF16, 2), _append(dev, 2, 2, BF16, 2)
    rows = torch.randn(2, 2, 40, 128, device=dev).to(BF16)
    w = torch.rand(2, 2, 40, device=dev)

    def fresh():
        return dataclasses.replace(start, **{n: getattr(start, n).clone() for n in ("key_pages", "value_pages", "weight_pages", "lengths")})

    def same(a, b):
        for n in ("key_pages", "value_pages", "weight_pages"):
            kind = torch.int32 if n == "weight_pages" else torch.int16
            assert torch.equal(getattr(a, n).view(kind), getattr(b, n).view(kind)), n

    cache = fresh()
    ro.paged_extend(cache, rows, -rows, weights=w)
    for path in _both_paths(None):
        other = fresh()
        _, early = _behind_long_work([rows, w, other.lengths], lambda: ro.paged_extend(other, rows, -rows, weights=w))
        assert early
        same(other, cache)

    cache = fresh()
    want = ro.paged_attention(q, cache, append=new)
    for path in _both_paths(None):
        other = fresh()
        got, early = _behind_long_work([q, *new, other.key_pages, other.weight_pages, other.lengths],
                                       lambda: ro.paged_attention(q, other, append=new))
        assert early and all(torch.equal(x, y) for x, y in zip(got, want))
        same(other, cache)

    def target():
        return _cache(dev, (64, 64), 2, 32, BF16, seed=3, weights=True)

    to = target()
    kept = ro.paged_evict(start, to, 64, sinks=2, recent=9)
    for path in _both_paths(None):
        other, to2 = fresh(), target()
        got, early = _behind_long_work([other.weight_pages, other.value_pages, other.lengths],
                                       lambda: ro.paged_evict(other, to2, 64, sinks=2, recent=9))
        assert early and torch.equal(got, kept) and torch.equal(to2.lengths, to.lengths)
        same(to2, to)


@pytest.mark.parametrize("sq,sk,window,sinks", [(900, 900, None, 0), (40, 3000, None, 0), (500, 900, 300, 4)])
def test_weights_and_attention_for_any_number_of_splits(sq, sk, window, sinks):
    """Each within the 64-bit bound: the joins add partial results of other cuts."""
    from r2omni_amd import _lib

    dev = _cuda()
    q, k, v = _rows(dev, 1, 16, 2, sq, sk, BF16, seed=sq)
    want = prompt(q, k, v, window, sinks)
    for splits in (1, 2, 3, 5, 12, 40):
        out, lse, weights = torch.empty_like(q), torch.empty(1, 16, sq, device=dev), torch.empty(1, 2, sk, device=dev)
        scratch = torch.empty(splits * max(130 * 16 * sq, 2 * sk), device=dev)
        p = _lib.PromptParams(query=q.data_ptr(), key=k.data_ptr(), value=v.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                              q_strides=q.stride()[:3], k_strides=k.stride()[:3], v_strides=v.stride()[:3], o_strides=out.stride()[:3],
                              batch=1, hq=16, hkv=2, queries=sq, keys=sk, dtype=0, window=window or 0, sinks=sinks, sm_scale=128 ** -0.5,
                              lse_in=lse.data_ptr(), weights=weights.data_ptr(), scratch=scratch.data_ptr(),
                              scratch_floats=scratch.numel(), splits=splits)
        _lib.launch("r2o_prompt_attention", p, dev)
        _lib.launch("r2o_attention_weights", p, dev)
        torch.cuda.synchronize()
        close(out, want[0], want[3])
        close(lse, want[1], want[4])
        close(weights, want[2], want[5])
