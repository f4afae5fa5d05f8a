"""Rotation by positions on the GPU against the definition in 64 bits, and the same on rows that go to a paged cache."""
import dataclasses
import math

import pytest
import torch

from attention_reference import close
from position_reference import rotate
from test_gpu_paged import BF16, FP16, _cache, _cuda

pytestmark = pytest.mark.gpu

SECTIONS = [((64,), False), ((16, 24, 24), False), ((24, 20, 20), True), ((10, 54), False), ((0, 64, 0), False), ((43, 21), True)]


def _rotary(dev, sections=((64,), False), theta=1e6, norms=None, seed=0, **more):
    import r2omni_amd as ro

    freq = theta ** (-torch.arange(0, 128, 2, dtype=torch.float32, device=dev) / 128)
    if norms is not None:
        gen = torch.Generator(device=dev).manual_seed(seed)
        more["q_norm_weight"], more["k_norm_weight"] = ((torch.rand(128, generator=gen, device=dev) * 2 - 0.5).to(norms) for _ in range(2))
    return ro.PositionRotary(freq, *sections, **more)


def _inputs(dev, b, hq, hkv, s, dtype, axes, most, seed, kind=torch.int64):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q, k = (torch.randn(b, h, s, 128, generator=gen, device=dev).to(dtype) for h in (hq, hkv))
    return q, k, torch.randint(0, most, (axes, b, s), generator=gen, device=dev).to(kind)


def _check(q, k, positions, rotary, apply_hadamard=False, **more):
    import r2omni_amd as ro

    pos = positions[None] if positions.ndim == 2 else positions
    want = [rotate(x, pos, rotary, w, apply_hadamard) for x, w in ((q, rotary.q_norm_weight), (k, rotary.k_norm_weight))]
    got = ro.qk_position_rope(q, k, positions, rotary, apply_hadamard=apply_hadamard, **more)
    torch.cuda.synchronize()
    for g, x, (y, bound) in zip(got, (q, k), want):
        assert g.shape == x.shape and g.dtype == x.dtype
        close(g, y, bound)
    return got


# one token, a wave's four and one to either side, a workgroup's sixteen, odd ones
@pytest.mark.parametrize("s", [1, 3, 4, 5, 15, 16, 17, 257])
@pytest.mark.parametrize("b,hq,hkv", [(1, 1, 1), (3, 28, 4), (2, 16, 2), (1, 32, 8), (5, 3, 3)])
def test_tokens_and_heads(b, hq, hkv, s):
    dev = _cuda()
    rotary = _rotary(dev, ((16, 24, 24), False))
    _check(*_inputs(dev, b, hq, hkv, s, BF16, 3, 40_000, s), rotary)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("apply_hadamard", [False, True])
@pytest.mark.parametrize("sections", SECTIONS)
def test_axes_norms_and_hadamard(sections, apply_hadamard, norm, dtype):
    dev = _cuda()
    rotary = _rotary(dev, sections, norms=dtype if norm else None)
    _check(*_inputs(dev, 2, 6, 2, 21, dtype, len(sections[0]), 1_000_000, 1), rotary, apply_hadamard)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("positions", [(0, 1, 2, 3), (131071, 131072, 1_000_003, 16_777_217), (2**31 - 1, 2**30 + 1, 2**31 - 2, 12345),
                                       (-1, -2, -131071, -(2**31))])
def test_far_and_negative_positions(positions, kind):
    dev = _cuda()
    q, k, _ = _inputs(dev, 1, 4, 2, 4, FP16, 1, 2, 2)
    _check(q, k, torch.tensor([positions], device=dev).to(kind), _rotary(dev))


@pytest.mark.parametrize("freq", [torch.float32, torch.float64])
def test_other_frequencies_and_scalings(freq):
    """Frequencies that are no power of a base, 0 and above a turn a position, either type; a scaling of cosine and sine."""
    dev = _cuda()
    q, k, pos = _inputs(dev, 2, 4, 2, 9, BF16, 1, 50_000, 3)
    gen = torch.Generator(device=dev).manual_seed(4)
    inv_freq = (torch.rand(64, generator=gen, device=dev) * 9).to(freq)
    inv_freq[[0, 63]] = 0.0
    for scaling in (1.0, 1.2079, -0.5, 0.0):
        _check(q, k, pos, dataclasses.replace(_rotary(dev), inv_freq=inv_freq, scaling=scaling))


def test_position_layouts():
    """[B, S] for one axis; one row of positions for all requests, one request's for all axes, every second token's."""
    dev = _cuda()
    q, k, pos = _inputs(dev, 3, 4, 2, 10, BF16, 3, 9000, 5)
    one = _rotary(dev)
    a = _check(q, k, pos[0], one)
    b = _check(q, k, pos[:1], one)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    three = _rotary(dev, ((16, 24, 24), False))
    _check(q, k, pos[:, :1].expand(3, 3, 10), three)
    _check(q, k, pos[:1].expand(3, 3, 10), three)
    wide = torch.randint(0, 9000, (3, 3, 20), device=dev)
    _check(q, k, wide[..., ::2], three)
    _check(q, k, wide[..., 1::2].transpose(1, 2).contiguous().transpose(1, 2), three)


def test_layouts_of_rows_and_results():
    """Views of a fused projection and odd strides; results of the caller's; in place; what lies beside stays."""
    import r2omni_amd as ro

    dev = _cuda()
    q, k, pos = _inputs(dev, 2, 8, 2, 19, BF16, 1, 9000, 6)
    rotary = _rotary(dev, norms=BF16)
    want = _check(q, k, pos, rotary)
    fused = torch.full((2, 19, 12, 128), 7.0, dtype=BF16, device=dev)
    fused[:, :, :8], fused[:, :, 8:10] = q.transpose(1, 2), k.transpose(1, 2)
    fq, fk = fused[:, :, :8].transpose(1, 2), fused[:, :, 8:10].transpose(1, 2)
    odd = torch.full((2, 8, 19, 132), math.nan, dtype=BF16, device=dev)
    odd[..., 1:129] = q
    last = k.transpose(2, 3).contiguous().transpose(2, 3)
    for x, y in ((fq, fk), (odd[..., 1:129], k), (q, last)):
        got = ro.qk_position_rope(x, y, pos, rotary)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    to = torch.full((2, 19, 14, 128), 5.0, dtype=BF16, device=dev)
    out = to[:, :, 1:9].transpose(1, 2), to[:, :, 9:11].transpose(1, 2)
    got = ro.qk_position_rope(q, k, pos, rotary, output=out)
    assert got[0].data_ptr() == out[0].data_ptr() and torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert (to[:, :, 0] == 5.0).all() and (to[:, :, 11:] == 5.0).all()
    ro.qk_position_rope(fq, fk, pos, rotary, output=(fq, fk))
    assert torch.equal(fq, want[0]) and torch.equal(fk, want[1]) and (fused[:, :, 10:] == 7.0).all()


def test_infinite_and_nan_rows_stay_their_own():
    import r2omni_amd as ro

    dev = _cuda()
    q, k, pos = _inputs(dev, 2, 4, 2, 9, BF16, 1, 9000, 7)
    for rotary in (_rotary(dev), _rotary(dev, norms=BF16)):
        want = _check(q, k, pos, rotary)
        bad = q.clone()
        bad[0, 1, 3] = math.nan
        bad[1, 2, 8, 5] = math.inf
        got = ro.qk_position_rope(bad, k, pos, rotary)[0]
        same = torch.ones(2, 4, 9, dtype=torch.bool, device=dev)
        same[0, 1, 3] = same[1, 2, 8] = False
        assert torch.equal(got[same], want[0][same]) and got[0, 1, 3].isnan().all() and not torch.isfinite(got[1, 2, 8, [5, 69]]).any()
    # rows of zeros: no norm to divide by but eps
    zero = torch.zeros_like(q)
    assert not ro.qk_position_rope(zero, k, pos, _rotary(dev, norms=BF16))[0].any()


def test_as_the_tables_of_a_model_give_it():
    """Against the operators that take cos and sin tables, at near positions: within the tables' fp32 angles."""
    import r2omni_amd as ro

    dev = _cuda()
    q, k, pos = _inputs(dev, 2, 28, 4, 33, BF16, 3, 500, 8)
    rotary = _rotary(dev, ((16, 24, 24), False))
    got = ro.qk_position_rope(q, k, pos, rotary)
    angle = pos[..., None].float() * rotary.inv_freq
    angle = torch.cat((angle, angle), -1)
    want = ro.qwen_qk_mrope(q, k, angle.cos(), angle.sin(), (16, 24, 24))
    for g, w, x in zip(got, want, (q, k)):
        # an angle of up to 500 in fp32 is off by 2^-16; both round once
        size = x.double().abs() + torch.cat((x[..., 64:], x[..., :64]), -1).double().abs()
        assert ((g.double() - w.double()).abs() <= size * 2.0 ** -15 + w.double().abs() * 2.0 ** -7).all()


# ------------------------------------------------------------------------------------ into the cache
def _extend_check(cache, q, k, v, rotary, positions=None, counts=None, weights=None):
    import r2omni_amd as ro

    b, s = q.shape[0], q.shape[2]
    page, capacity = cache.key_pages.shape[2], cache.capacity
    n = cache.lengths.long().tolist()
    count = [s] * b if counts is None else [max(0, min(c, s)) for c in counts.tolist()]
    slot = torch.tensor(n, device=q.device)[:, None] - torch.tensor(count, device=q.device)[:, None] + torch.arange(s, device=q.device)
    pos = slot[None].expand(len(rotary.mrope_section), b, s) if positions is None else positions
    (wq, bq), (wk, bk) = (rotate(x, pos, rotary, w) for x, w in ((q, rotary.q_norm_weight), (k, rotary.k_norm_weight)))
    want_k, bound_k = cache.key_pages.double(), torch.zeros(cache.key_pages.shape, dtype=torch.float64, device=q.device)
    want_v = cache.value_pages.clone()
    want_w = None if cache.weight_pages is None else cache.weight_pages.clone()
    for i in range(b):
        wq[i, :, count[i] :], bq[i, :, count[i] :] = 0.0, 0.0
        for r in range(count[i]):
            j = int(slot[i, r])
            if not 0 <= j < capacity:
                continue
            id_ = int(cache.page_table[i, j // page])
            if 0 <= id_ < cache.key_pages.shape[0]:
                want_k[id_, :, j % page], bound_k[id_, :, j % page] = wk[i, :, r], bk[i, :, r]
                want_v[id_, :, j % page] = v[i, :, r]
                if want_w is not None:
                    want_w[id_, :, j % page] = 0.0 if weights is None else weights[i, :, r]
    out = ro.paged_rope_extend(cache, q, k, v, rotary, positions=positions, counts=counts, weights=weights)
    torch.cuda.synchronize()
    close(out, wq, bq)
    old = torch.isnan(want_k) & (bound_k == 0)  # slots that are not filled yet hold NaN
    assert cache.key_pages[old].isnan().all()
    close(cache.key_pages[~old], want_k[~old], bound_k[~old])
    assert torch.equal(cache.value_pages.contiguous().view(torch.int16), want_v.contiguous().view(torch.int16))
    if want_w is not None:
        assert torch.equal(cache.weight_pages.nan_to_num(nan=-1.0), want_w.nan_to_num(nan=-1.0))
    return out


def _new_rows(dev, b, hq, hkv, s, dtype, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(b, s, hq + 2 * hkv, 128, generator=gen, device=dev).to(dtype).transpose(1, 2)
    return x[:, :hq], x[:, hq : hq + hkv], x[:, hq + hkv :]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("s", [1, 4, 17, 130])
@pytest.mark.parametrize("weights", [False, True])
def test_extend_pages_and_rows(page, s, weights):
    dev = _cuda()
    cache = _cache(dev, (s, s + 13, s + 127), 2, page, BF16, s, weights=weights)
    q, k, v = _new_rows(dev, 3, 14, 2, s, BF16, s)
    w = torch.rand(3, 2, s, device=dev) if weights else None
    _extend_check(cache, q, k, v, _rotary(dev), weights=w)
    if weights:
        _extend_check(cache, q, k, v, _rotary(dev))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("sections", SECTIONS)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (28, 4), (32, 8), (5, 5)])
def test_extend_axes_and_heads(hq, hkv, sections, norm, dtype):
    dev = _cuda()
    cache = _cache(dev, (40, 9), hkv, 16, dtype, 1)
    rotary = _rotary(dev, sections, norms=dtype if norm else None)
    pos = torch.randint(0, 200_000, (len(sections[0]), 2, 9), device=dev)
    _extend_check(cache, *_new_rows(dev, 2, hq, hkv, 9, dtype, 2), rotary, pos)
    _extend_check(cache, *_new_rows(dev, 2, hq, hkv, 9, dtype, 3), rotary, pos.to(torch.int32), torch.tensor([3, 9], dtype=torch.int32, device=dev))
    _extend_check(cache, *_new_rows(dev, 2, hq, hkv, 9, dtype, 4), rotary)  # a row's slot is its position


def test_extend_padded_and_out_of_range():
    """Counts of 0, below 0 and past the rows; lengths below the count and past the table; pages that are not mapped."""
    dev = _cuda()
    cache = _cache(dev, (64, 64, 64, 64, 64, 64), 2, 16, BF16, 5, weights=True)
    cache.lengths.copy_(torch.tensor([30, 64, 5, 70, 0, -9], dtype=torch.int32))
    cache.page_table[0, 1] = -1
    cache.page_table[1, 3] = cache.key_pages.shape[0]
    rows = _new_rows(dev, 6, 8, 2, 20, BF16, 5)
    _extend_check(cache, *rows, _rotary(dev), counts=torch.tensor([20, 7, 9, 40, 0, -3], dtype=torch.int32, device=dev))
    _extend_check(cache, *rows, _rotary(dev))


def test_extend_layouts_results_and_pools():
    import r2omni_amd as ro

    dev = _cuda()
    start = _cache(dev, (70, 33), 2, 32, BF16, 6, fused=True)
    q, k, v = _new_rows(dev, 2, 8, 2, 21, BF16, 6)
    rotary = _rotary(dev, norms=BF16)

    def fresh():
        pool = torch.stack((start.key_pages, start.value_pages), 1)
        return dataclasses.replace(start, key_pages=pool[:, 0], value_pages=pool[:, 1])

    cache = fresh()
    want = _extend_check(cache, q, k, v, rotary)
    odd = torch.full((2, 8, 21, 132), math.nan, dtype=BF16, device=dev)
    odd[..., 1:129] = q
    to = torch.full((2, 21, 10, 128), 5.0, dtype=BF16, device=dev)
    mine = q.contiguous()
    for x, out in ((odd[..., 1:129], None), (q.contiguous(), to[:, :, 1:9].transpose(1, 2)), (mine, mine), (q, q)):
        other = fresh()
        got = ro.paged_rope_extend(other, x, k.contiguous(), v.transpose(2, 3).contiguous().transpose(2, 3), rotary, output=out)
        assert torch.equal(got, want) and (out is None or got is out)
        for a, b in ((other.key_pages, cache.key_pages), (other.value_pages, cache.value_pages)):
            assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))
    assert (to[:, :, 0] == 5.0).all() and (to[:, :, 9:] == 5.0).all()


def test_extend_is_the_rotation_then_the_plain_extend():
    import r2omni_amd as ro

    dev = _cuda()
    for dtype in (BF16, FP16):
        a = _cache(dev, (100, 40), 4, 16, dtype, 7, weights=True)
        b = dataclasses.replace(a, key_pages=a.key_pages.clone(), value_pages=a.value_pages.clone(), weight_pages=a.weight_pages.clone())
        q, k, v = _new_rows(dev, 2, 28, 4, 33, dtype, 7)
        rotary, pos = _rotary(dev, ((16, 24, 24), False), norms=dtype), torch.randint(0, 9000, (3, 2, 33), device=dev)
        w = torch.rand(2, 4, 33, device=dev)
        out = ro.paged_rope_extend(a, q, k, v, rotary, positions=pos, weights=w)
        rq, rk = ro.qk_position_rope(q, k, pos, rotary)
        ro.paged_extend(b, rk, v, weights=w)
        assert torch.equal(out, rq)
        for x, y in zip((a.key_pages, a.value_pages), (b.key_pages, b.value_pages)):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))
        assert torch.equal(a.weight_pages.nan_to_num(nan=-1.0), b.weight_pages.nan_to_num(nan=-1.0))


def test_captured_calls_follow_positions_and_lengths():
    import r2omni_amd as ro

    dev = _cuda()
    cache = _cache(dev, (90, 60), 2, 16, BF16, 8)
    q, k, v = _new_rows(dev, 2, 8, 2, 3, BF16, 8)
    pos, rotary = torch.zeros(3, 2, 3, dtype=torch.int64, device=dev), _rotary(dev, ((16, 24, 24), False))
    counts = torch.full((2,), 3, dtype=torch.int32, device=dev)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        return (ro.paged_rope_extend(cache, q, k, v, rotary, positions=pos, counts=counts), ro.paged_rope_extend(cache, q, k, v, rotary),
                *ro.qk_position_rope(q, k, pos, rotary))

    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    for i in range(5):
        pos.random_(0, 100_000)
        cache.lengths.copy_(torch.tensor([20 + i, 60 - i], dtype=torch.int32))
        counts.copy_(torch.tensor([i % 4, 3], dtype=torch.int32))
        k.normal_()
        q.normal_()
        cache.key_pages.zero_()
        graph.replay()
        torch.cuda.synchronize()
        keys = cache.key_pages.clone()
        cache.key_pages.zero_()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        assert torch.equal(keys, cache.key_pages) and keys.any()


def test_the_python_path_gives_the_host_modules_results():
    import r2omni_amd as ro
    import r2omni_amd._lib as lib

    dev = _cuda()
    start = _cache(dev, (100, 40), 4, 16, FP16, 9, weights=True)
    q, k, v = _new_rows(dev, 2, 28, 4, 33, FP16, 9)
    pos = torch.randint(0, 9000, (3, 2, 33), device=dev)
    for sections in (((16, 24, 24), False), ((24, 20, 20), True)):
        for norms in (None, FP16):
            rotary = _rotary(dev, sections, norms=norms, scaling=1.25, eps=1e-5)
            found = []
            real = lib.host()

            class Without:
                def __getattr__(self, name):
                    return lambda *args: None

            for host in (real, Without()):
                cache = dataclasses.replace(start, key_pages=start.key_pages.clone(), value_pages=start.value_pages.clone(),
                                            weight_pages=start.weight_pages.clone())
                lib._HOST = host
                try:
                    made = ro.paged_rope_extend(cache, q, k, v, rotary, positions=pos, counts=torch.tensor([33, 7], dtype=torch.int32, device=dev))
                    found.append((made, *ro.qk_position_rope(q, k, pos, rotary, apply_hadamard=True), cache.key_pages.nan_to_num(nan=9.0),
                                  cache.value_pages.nan_to_num(nan=9.0), cache.weight_pages.nan_to_num(nan=-1.0)))
                finally:
                    lib._HOST = real
            assert all(torch.equal(a, b) for a, b in zip(*found))


def test_rows_and_pages_past_32_bits():
    """Requests whose rows lie 2^31 elements apart, and slots whose offsets pass 2^32."""
    import r2omni_amd as ro

    dev = _cuda()
    far = torch.empty((1 << 31) + 2 * 128 * 40, dtype=BF16, device=dev)
    q = far.as_strided((2, 8, 5, 128), (1 << 31, 5 * 128, 128, 1))
    k = far[8 * 5 * 128 :].as_strided((2, 2, 5, 128), (1 << 31, 5 * 128, 128, 1))
    q.normal_(), k.normal_()
    pos, rotary = torch.randint(0, 9000, (2, 5), device=dev), _rotary(dev)
    want = _check(q.contiguous(), k.contiguous(), pos, rotary)
    got = ro.qk_position_rope(q, k, pos, rotary)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ro.qk_position_rope(q, k, pos, rotary, output=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    pages = (1 << 32) // (2 * 128 * 128) + 4
    kp, vp = (torch.zeros(pages, 2, 128, 128, dtype=BF16, device=dev) for _ in range(2))
    cache = ro.PagedCache(kp, vp, torch.tensor([[pages - 1], [pages // 2 + 1]], dtype=torch.int32, device=dev),
                          torch.tensor([5, 100], dtype=torch.int32, device=dev))
    ro.paged_rope_extend(cache, q, k, k, rotary)
    near = ro.PagedCache(kp[:2].clone(), vp[:2].clone(), torch.tensor([[0], [1]], dtype=torch.int32, device=dev), cache.lengths)
    ro.paged_rope_extend(near, q, k, k, rotary)
    for i, p in ((0, pages - 1), (1, pages // 2 + 1)):
        assert torch.equal(kp[p], near.key_pages[i]) and torch.equal(vp[p], near.value_pages[i]) and kp[p].any()
