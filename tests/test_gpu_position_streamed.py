"""Large rotations, whose rows pass the caches by: every number of heads that a wave's rounds of sixteen may leave over, against small
calls of the same rows, which do not pass them by."""
import dataclasses

import pytest
import torch

from test_gpu_paged import BF16, FP16, _cache, _cuda
from test_gpu_position import _new_rows, _rotary

pytestmark = pytest.mark.gpu


# heads of both: one round, short or not; two, the last of 1 to 16 heads; three
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (8, 2), (9, 2), (15, 1), (16, 1), (16, 2), (14, 7), (20, 2), (28, 4), (32, 1), (34, 2)])
@pytest.mark.parametrize("norm", [False, True])
def test_any_number_of_heads(hq, hkv, norm):
    import r2omni_amd as ro

    dev, dtype = _cuda(), FP16 if norm else BF16
    s = (1 << 18) // (hq + hkv) + 5
    rotary = _rotary(dev, ((16, 24, 24), False), norms=dtype if norm else None)
    q, k, v = _new_rows(dev, 1, hq, hkv, s, dtype, hq)
    pos = torch.randint(0, 1 << 20, (3, 1, s), device=dev)
    got = ro.qk_position_rope(q, k, pos, rotary)
    places = ro.qk_position_rope(q, k, pos, rotary, output=(q.clone(), k.clone()))
    step, parts = s // 7 + 1, []
    for at in range(0, s, step):
        parts.append(ro.qk_position_rope(q[:, :, at : at + step], k[:, :, at : at + step], pos[:, :, at : at + step], rotary))
    for x, y, z in zip(got, places, zip(*parts)):
        assert torch.equal(x, torch.cat(z, 2)) and torch.equal(x, y)
    in_place = q.clone(), k.clone()
    ro.qk_position_rope(*in_place, pos, rotary, output=in_place)
    assert torch.equal(in_place[0], got[0]) and torch.equal(in_place[1], got[1])
    cache = _cache(dev, (s,), hkv, 64, dtype, 2)
    other = dataclasses.replace(cache, key_pages=cache.key_pages.clone(), value_pages=cache.value_pages.clone())
    assert torch.equal(ro.paged_rope_extend(cache, q, k, v, rotary, positions=pos), got[0])
    ro.paged_extend(other, got[1], v)
    for a, b in ((cache.key_pages, other.key_pages), (cache.value_pages, other.value_pages)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def _bytes_a_second(dev, hq, hkv, s):
    import r2omni_amd as ro

    sides = []
    for _ in range(3):  # no call finds its rows in the caches
        x = torch.randn(1, s, hq + hkv, 128, device=dev).to(BF16).transpose(1, 2)
        sides.append((x[:, :hq], x[:, hq:], tuple(torch.empty(1, h, s, 128, dtype=BF16, device=dev) for h in (hq, hkv))))
    pos, rotary, times = torch.arange(s, device=dev)[None], _rotary(dev), []
    for i in range(24):
        q, k, out = sides[i % 3]
        events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        events[0].record()
        for _ in range(2):
            ro.qk_position_rope(q, k, pos, rotary, output=out)
        events[1].record()
        torch.cuda.synchronize()
        times.append(events[0].elapsed_time(events[1]))
    return 1024 * (hq + hkv) * s / sorted(times)[12]


def test_few_heads_are_rotated_as_fast_as_many():
    """Four heads' rows, each read once: a round of sixteen that reads the last one's thirteen times takes half as long again."""
    dev = _cuda()
    assert _bytes_a_second(dev, 3, 1, 200_003) > 0.8 * _bytes_a_second(dev, 14, 2, 50_001)
