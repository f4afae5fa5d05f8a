"""How many workgroups share a row tile's keys: the rule alone, on the CPU."""
import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib

CUS = 256


def _seen(group, first, rows, keys, queries, window, sinks):
    """Key tiles (of 64) that a tile of 128 packed rows sees."""
    off = keys - queries
    low, high = off + first * 128 // group, off + min(first * 128 + 127, rows - 1) // group
    tiles = set(range(max(0, low - window + 1) // 64, high // 64 + 1)) if window else set(range(high // 64 + 1))
    return len(tiles | set(range(-(-min(sinks, high + 1) // 64)))) if window else len(tiles)


@pytest.mark.parametrize("hq,hkv", [(16, 2), (28, 4), (32, 8), (4, 4)])
@pytest.mark.parametrize("queries,keys,window,sinks", [(512, 16384, 256, 0), (500, 16384, 64, 0), (512, 16384, 256, 64), (100, 8192, 2048, 4),
                                                       (1, 5000, 1, 0), (300, 300, 1000, 7), (64, 30000, 700, 900)])
def test_no_more_splits_than_a_windowed_tile_has_keys_for(queries, keys, window, sinks, hq, hkv):
    """A split for each four key tiles that a row tile sees, begun ones and one for where they start among them."""
    group = hq // hkv
    rows = queries * group
    most = max(_seen(group, i, rows, keys, queries, window, sinks) for i in range(-(-rows // 128)))
    splits = _lib.host().attention_splits(1, hq, hkv, queries, keys, window, sinks, CUS)
    assert 1 <= splits <= -(-(most + 1) // 4)


@pytest.mark.parametrize("args,want", [((1, 16, 2, 257, 4097, 0, 0), 7), ((1, 28, 4, 16384, 16384, 0, 0), 1), ((1, 28, 4, 1, 300, 0, 0), 2),
                                       ((1, 28, 4, 1, 256, 0, 0), 1), ((1, 28, 4, 500, 16384, 64, 0), 1)])
def test_splits_of_known_calls(args, want):
    assert _lib.host().attention_splits(*args, CUS) == want


def test_the_call_uses_the_rule(monkeypatch):
    launched = []
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(_lib, "launch", lambda name, params, device: launched.append(params))
    monkeypatch.setattr(_lib, "num_cus", lambda device: CUS)
    q, k = torch.zeros(1, 8, 3, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 5000, 128, dtype=torch.bfloat16)
    for window, sinks in ((None, 0), (700, 0), (700, 900), (10, 0)):
        ro.prompt_attention(q, k, k, window=window, sinks=sinks)
        assert launched[-1].splits == _lib.host().attention_splits(1, 8, 2, 3, 5000, window or 0, sinks, CUS)
    assert [p.splits for p in launched] == [20, 4, 7, 1]
