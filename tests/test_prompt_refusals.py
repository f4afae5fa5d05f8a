"""What prompt_attention and attention_weights refuse, on the CPU: shapes, types and options are checked before the
device, and the C ABI checks its own arguments before a launch."""
import ctypes

import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib

BF16 = torch.bfloat16


def _rows(b=1, hq=4, hkv=2, sq=3, sk=5, d=128, dtype=BF16):
    return torch.zeros(b, hq, sq, d, dtype=dtype), torch.zeros(b, hkv, sk, d, dtype=dtype), torch.zeros(b, hkv, sk, d, dtype=dtype)


BAD = {
    "rank": (lambda q, k, v: (q[0], k, v), {}),
    "head width": (lambda q, k, v: (q[..., :64], k[..., :64], v[..., :64]), {}),
    "batch": (lambda q, k, v: (q, k.repeat(2, 1, 1, 1), v.repeat(2, 1, 1, 1)), {}),
    "heads": (lambda q, k, v: (q[:, :3], k, v), {}),
    "no rows": (lambda q, k, v: (q[:, :, :0], k, v), {}),
    "no keys": (lambda q, k, v: (q, k[:, :, :0], v[:, :, :0]), {}),
    "fp32": (lambda q, k, v: (q.float(), k.float(), v.float()), {}),
    "types differ": (lambda q, k, v: (q.half(), k, v), {}),
    "window": (lambda q, k, v: (q, k, v), {"window": 0}),
    "sinks": (lambda q, k, v: (q, k, v), {"sinks": -1, "window": 4}),
    "scale of zero": (lambda q, k, v: (q, k, v), {"sm_scale": 0.0}),
    "scale of NaN": (lambda q, k, v: (q, k, v), {"sm_scale": float("nan")}),
    "infinite scale": (lambda q, k, v: (q, k, v), {"sm_scale": float("inf")}),
    "lengths of another type": (lambda q, k, v: (q, k, v), {"key_lengths": torch.zeros(1, dtype=torch.int64)}),
    "lengths of another batch": (lambda q, k, v: (q, k, v), {"query_lengths": torch.zeros(2, dtype=torch.int32)}),
}


@pytest.mark.parametrize("what", BAD)
def test_refused_arguments(what):
    change, options = BAD[what]
    q, k, v = change(*_rows())
    with pytest.raises((ValueError, RuntimeError)) as e:
        ro.prompt_attention(q, k, v, **options)
    assert "GPU" not in str(e.value) or "scale" in what or what in ("window", "sinks")
    with pytest.raises((ValueError, RuntimeError)):
        ro.attention_weights(q, k, torch.zeros(q.shape[:3]), **options)


def test_refused_values_statistics_and_outputs():
    q, k, v = _rows()
    with pytest.raises(ValueError, match="value"):
        ro.prompt_attention(q, k, v[:, :, :4])
    with pytest.raises(ValueError, match="lse"):
        ro.attention_weights(q, k, torch.zeros(1, 4, 4))
    with pytest.raises(ValueError, match="lse"):
        ro.attention_weights(q, k, torch.zeros(1, 4, 3, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="GPU"):
        ro.prompt_attention(q, k, v)
    with pytest.raises(RuntimeError, match="GPU"):
        ro.attention_weights(q, k, torch.zeros(1, 4, 3))
    with pytest.raises(RuntimeError, match="backward"):
        ro.prompt_attention(q.requires_grad_(), k, v)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        ro.prompt_attention(q, k, v)


def _params(**kw):
    st = (ctypes.c_int64 * 3)(128 * 64, 128 * 16, 128)
    p = _lib.PromptParams(query=0x1000, key=0x2000, value=0x3000, out=0x4000, lse=0x5000, q_strides=st, k_strides=st,
                          v_strides=st, o_strides=st, batch=1, hq=4, hkv=2, queries=16, keys=16, sm_scale=0.1,
                          lse_in=0x6000, weights=0x7000, splits=1)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


BAD_C = {
    "no query": dict(query=None), "no key": dict(key=None), "misaligned query": dict(query=0x1008),
    "type": dict(dtype=2), "no heads": dict(hkv=0), "heads": dict(hq=5), "no batch": dict(batch=0),
    "batch past the grid": dict(batch=65536), "no rows": dict(queries=0), "rows past 2^29": dict(keys=(1 << 29) + 1),
    "window": dict(window=-1), "sinks": dict(sinks=-1), "scale": dict(sm_scale=0.0), "NaN scale": dict(sm_scale=float("nan")),
    "stride off 16 bytes": dict(q_strides=(ctypes.c_int64 * 3)(128 * 64, 128 * 16, 132)),
    "negative stride": dict(k_strides=(ctypes.c_int64 * 3)(128 * 64, 128 * 16, -128)),
    "misaligned lengths": dict(key_lengths=0x8002),
}


@pytest.mark.parametrize("what", BAD_C)
def test_c_abi_refuses(what):
    p = _params(**BAD_C[what])
    assert _lib.load().r2o_prompt_attention(ctypes.byref(p), None) == 1
    assert _lib.load().r2o_attention_weights(ctypes.byref(p), None) == 1


def test_c_abi_refuses_outputs_and_scratch():
    lib = _lib.load()
    for kw in (dict(out=None), dict(out=0x4008), dict(lse=None), dict(value=None),
               dict(v_strides=(ctypes.c_int64 * 3)(1, 128, 128)), dict(splits=0), dict(splits=2),
               dict(splits=2, scratch=0x9000, scratch_floats=2 * 4 * 16 * 130 - 1), dict(splits=2, scratch=0x9008, scratch_floats=1 << 20),
               dict(q_strides=(ctypes.c_int64 * 3)(8, 8, (1 << 24) + 8))):
        assert lib.r2o_prompt_attention(ctypes.byref(_params(**kw)), None) == 1, kw
    for kw in (dict(lse_in=None), dict(weights=None), dict(splits=0), dict(splits=2), dict(splits=65536),
               dict(splits=2, scratch=0x9000, scratch_floats=2 * 2 * 16 - 1)):
        assert lib.r2o_attention_weights(ctypes.byref(_params(**kw)), None) == 1, kw
    assert lib.r2o_prompt_attention(None, None) == 1 and lib.r2o_attention_weights(None, None) == 1
