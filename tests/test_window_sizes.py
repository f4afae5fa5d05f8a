"""Windows and sinks past every length, on the CPU: what a launch would get."""
import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib

BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("window", [1 << 30, (1 << 31) + 5, 1 << 40, (1 << 63) + 7, (1 << 64) + 7, 1 << 200])
def test_windows_past_every_length_see_everything(window, monkeypatch):
    """A request has at most 2^29 slots or rows; what is passed on is no smaller than that, and fits."""
    launched = []
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(_lib, "launch", lambda name, params, device: launched.append(params))
    monkeypatch.setattr(_lib, "num_cus", lambda device: 256)
    q, k = torch.zeros(2, 4, 3, 128, dtype=BF16), torch.zeros(2, 2, 5, 128, dtype=BF16)
    pool = torch.zeros(6, 2, 16, 128, dtype=BF16)
    cache = ro.PagedCache(pool, pool.clone(), torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32))
    for sinks in (0, 1 << 70):
        ro.prompt_attention(q, k, k, window=window, sinks=sinks)
        ro.attention_weights(q, k, torch.zeros(2, 4, 3), window=window, sinks=sinks)
        ro.paged_attention(q[:, :, 0], cache, window=window, sinks=sinks)
    for params in launched:
        assert 1 << 29 <= params.window < 1 << 63 and 0 <= params.sinks <= 1 << 29
