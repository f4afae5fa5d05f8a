"""Infinite and NaN values that a row sees: the row's channel is their sum, however small their weights are and wherever
their keys lie among the tiles, halves, splits and workers; every other channel has the bits of finite values."""
import dataclasses
import math

import pytest
import torch

from attention_reference import visible
from test_gpu_paged import BF16, FP16, _cache, _cuda, _slots

pytestmark = pytest.mark.gpu


def _rows(dev, b, hq, hkv, sq, sk, dtype, seed):
    """Every query points along one direction, with noise; a key's share of it spans 400 in the logits, so that weights
    of 1 stand beside ones that 16 bits, and ones that 32 bits, round to 0."""
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    along = normal(128)
    along = along / along.norm() * 128 ** 0.25
    q, k, v = normal(b, hq, sq, 128) * 0.1 + 4 * along, normal(b, hkv, sk, 128) * 0.1, normal(b, hkv, sk, 128)
    k = k + along * 100 * torch.rand(b, hkv, sk, 1, generator=gen, device=dev)
    return q.to(dtype), k.to(dtype), v.to(dtype)


def _spoil(v, gen, rate):
    """Some elements infinite of either sign, fewer NaN."""
    x = torch.rand(v.shape, generator=gen, device=v.device)
    v = torch.where(x < rate, math.inf, v.float())
    v = torch.where((x >= rate) & (x < 2 * rate), -math.inf, v)
    return torch.where((x >= 2 * rate) & (x < 2.2 * rate), math.nan, v)


def _want(clean, seen, v):
    """clean [R, 128], with what the rows see [R, S] of infinities and NaN in v [S, 128]."""
    plus, minus, nan = ((seen.double() @ bad.double()) > 0 for bad in (v == math.inf, v == -math.inf, v.isnan()))
    nan |= plus & minus
    out = torch.where(plus, math.inf, clean.double())
    out = torch.where(minus, -math.inf, out)
    return torch.where(nan, math.nan, out)


def _same(got, want):
    got = got.double()
    wrong = ~((got == want) | (got.isnan() & want.isnan()))
    assert not wrong.any(), f"{int(wrong.sum())} of {wrong.numel()}: {got[wrong][:4].tolist()} for {want[wrong][:4].tolist()}"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sq,sk,window,sinks", [(300, 300, None, 0), (300, 300, 70, 5), (16, 3000, None, 0), (1, 1000, None, 0),
                                                (130, 517, 200, 70), (700, 700, 1, 0)])
def test_prompt(sq, sk, window, sinks, dtype):
    """Whole prompts, chunks in splits, windows: keys in tiles that all of a workgroup's rows see and in others."""
    import r2omni_amd as ro

    dev, hq, hkv = _cuda(), 4, 2
    q, k, v = _rows(dev, 2, hq, hkv, sq, sk, dtype, seed=sq + sk)
    gen = torch.Generator(device=dev).manual_seed(sk)
    clean, lse = ro.prompt_attention(q, k, v, window=window, sinks=sinks)
    for rate in (2e-5, 2e-3):
        bad = _spoil(v, gen, rate).to(dtype)
        out, lse2 = ro.prompt_attention(q, k, bad, window=window, sinks=sinks)
        assert torch.equal(lse2, lse)
        seen = visible(sq, sk, sq, sk, window, sinks, dev)
        for b in range(2):
            for h in range(hq):
                _same(out[b, h], _want(clean[b, h], seen, bad[b, h // (hq // hkv)]))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_one_infinite_value_in_every_place(dtype):
    """A key of weight 0 in 16 and 32 bits with one infinite element: the rows that see it have it, whatever its tile."""
    import r2omni_amd as ro

    dev = _cuda()
    q, k, v = _rows(dev, 1, 4, 2, 200, 200, dtype, seed=5)
    clean, _ = ro.prompt_attention(q, k, v)
    for j in range(0, 200, 7):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, j] = -k[:, :, j].abs().amax() * torch.sign(q[0, 0, 0])
        v2[:, :, j, j % 128] = math.inf if j % 2 else -math.inf
        out, _ = ro.prompt_attention(q, k2, v2)
        assert (out[:, :, j:, j % 128] == (math.inf if j % 2 else -math.inf)).all(), j
        assert torch.isfinite(out[:, :, :j].float()).all() and torch.equal(out[:, :, :j], clean[:, :, :j])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_ragged_batches_and_rows_of_nan(dtype):
    """Requests of uneven length with garbage behind them; a NaN query row stays NaN, its neighbours do not."""
    import r2omni_amd as ro

    dev = _cuda()
    nq, nk = [0, 1, 90, 150, 60, 150], [0, 1, 33, 200, 0, 150]
    q, k, v = _rows(dev, 6, 4, 2, 150, 200, dtype, seed=6)
    lengths = {n + "_lengths": torch.tensor(x, dtype=torch.int32, device=dev) for n, x in (("query", nq), ("key", nk))}
    clean, _ = ro.prompt_attention(q, k, v, **lengths)
    bad = _spoil(v, torch.Generator(device=dev).manual_seed(6), 1e-3).to(dtype)
    for i, (a, n) in enumerate(zip(nq, nk)):
        q[i, :, a:], k[i, :, n:], bad[i, :, n:] = math.nan, math.inf, math.nan
    q[3, 1, 77, 4] = math.nan
    out, lse = ro.prompt_attention(q, k, bad, **lengths)
    assert out[3, 1, 77].isnan().all() and lse[3, 1, 77].isnan()
    for b in range(6):
        seen = visible(150, 200, nq[b], nk[b], None, 0, dev)
        for h in range(4):
            want = _want(clean[b, h], seen, bad[b, h // 2].nan_to_num(nan=math.nan, posinf=math.inf, neginf=-math.inf))
            if (b, h) == (3, 1):
                want[77] = math.nan
            _same(out[b, h], want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 5), (33, 40)])
def test_paged(window, sinks, append, dtype):
    """Long and short requests over many workers, an unmapped page, the appended row's values; weights as with finite ones."""
    import r2omni_amd as ro

    dev, lengths, page = _cuda(), (3001, 1, 0, 70, 517), 32
    cache = _cache(dev, lengths, 2, page, dtype, seed=7, weights=True)
    cache.page_table[0, 40] = -1
    q, k, v = _rows(dev, 5, 8, 2, 1, 3001, dtype, seed=7)
    new_k, new_v = k[:, :, 0], v[:, :, 0]
    for b, n in enumerate(lengths):
        for j0 in range(0, n, page):
            id_, rows = int(cache.page_table[b, j0 // page]), min(page, n - j0)
            if id_ >= 0:
                cache.key_pages[id_, :, :rows], cache.value_pages[id_, :, :rows] = k[b, :, j0 : j0 + rows], v[b, :, j0 : j0 + rows]
    w0 = cache.weight_pages.clone()
    options = dict(window=window, sinks=sinks)
    clean, lse = ro.paged_attention(q[:, :, 0], cache, append=(new_k, new_v) if append else None, **options)
    w1 = cache.weight_pages.clone()
    gen = torch.Generator(device=dev).manual_seed(8)
    start = cache.value_pages.clone()
    for rate in (3e-5, 2e-3):
        cache.value_pages.copy_(torch.where(start.isnan(), math.nan, _spoil(start, gen, rate)).to(dtype))
        cache.weight_pages.copy_(w0)
        bad_new = _spoil(new_v, gen, 0.01).to(dtype)
        out, lse2 = ro.paged_attention(q[:, :, 0], cache, append=(new_k, bad_new) if append else None, **options)
        assert torch.equal(lse2, lse) and torch.equal(cache.weight_pages.view(torch.int32), w1.view(torch.int32))
        for b, n in enumerate(lengths):
            if not n:
                assert not out[b].any()
                continue
            rows, mapped = _slots(cache, b, n, cache.value_pages)
            j = torch.arange(n, device=dev)
            seen = mapped if window is None else mapped & ((j >= n - window) | (j < sinks))
            for h in range(8):
                _same(out[b, h][None], _want(clean[b, h][None], seen[None], rows[h // 4]))


def test_a_nan_token_beside_infinite_values():
    import r2omni_amd as ro

    dev = _cuda()
    cache = dataclasses.replace(_cache(dev, (3000, 40), 2, 32, FP16, seed=9, weights=True), weight_pages=None)
    q, _, _ = _rows(dev, 2, 8, 2, 1, 1, FP16, seed=9)
    q[0, 3, 0, 9] = math.nan
    cache.value_pages[cache.page_table[0, 3].long(), 0, 7, 100] = math.inf
    out, lse = ro.paged_attention(q, cache)
    assert out[0, 3].isnan().all() and lse[0, 3].isnan()
    rest = torch.ones(8, dtype=torch.bool, device=dev)
    rest[3] = False
    assert (out[0, [0, 1, 2], 100] == math.inf).all()
    assert torch.isfinite(out[0, 4:]).all() and torch.isfinite(out[1]).all() and torch.isfinite(out[0, rest][:, :100]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_nan_alone_beside_rows_that_see_less(dtype):
    """The search for such values may end early where everything is NaN: not before rows that see other ones are done."""
    import r2omni_amd as ro

    dev = _cuda()
    q, k, v = _rows(dev, 1, 4, 2, 400, 400, dtype, seed=11)
    clean, _ = ro.prompt_attention(q, k, v, window=90, sinks=3)
    v[:, :, 100:140] = math.nan
    v[:, :, 250, 3], v[:, :, 310, 3], v[:, :, 2, 9] = math.inf, -math.inf, -math.inf
    for window, sinks in ((90, 3), (None, 0)):
        out, _ = ro.prompt_attention(q, k, v, window=window, sinks=sinks)
        seen = visible(400, 400, 400, 400, window, sinks, dev)
        for h in range(4):
            want = _want(clean[0, h] if window else out[0, h].nan_to_num(nan=0.0, posinf=0.0, neginf=0.0), seen, v[0, h // 2])
            _same(out[0, h], want)
