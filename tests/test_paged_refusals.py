"""What the paged cache and its calls refuse, on the CPU: the Python checks come before the device, and the C ABI
checks its own arguments before a launch."""
import ctypes

import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib

BF16, I32 = torch.bfloat16, torch.int32


def _tensors(**change):
    t = {"key_pages": torch.zeros(6, 2, 16, 128, dtype=BF16), "value_pages": torch.zeros(6, 2, 16, 128, dtype=BF16),
         "page_table": torch.zeros(2, 3, dtype=I32), "lengths": torch.zeros(2, dtype=I32), "weight_pages": torch.zeros(6, 2, 16)}
    t.update(change)
    return t


BAD = {
    "rank": dict(key_pages=torch.zeros(6, 2, 16, dtype=BF16)),
    "head width": dict(key_pages=torch.zeros(6, 2, 16, 64, dtype=BF16), value_pages=torch.zeros(6, 2, 16, 64, dtype=BF16)),
    "value shape": dict(value_pages=torch.zeros(5, 2, 16, 128, dtype=BF16)),
    "page size": dict(key_pages=torch.zeros(6, 2, 24, 128, dtype=BF16), value_pages=torch.zeros(6, 2, 24, 128, dtype=BF16)),
    "no pages": dict(key_pages=torch.zeros(0, 2, 16, 128, dtype=BF16), value_pages=torch.zeros(0, 2, 16, 128, dtype=BF16)),
    "type": dict(key_pages=torch.zeros(6, 2, 16, 128), value_pages=torch.zeros(6, 2, 16, 128)),
    "types differ": dict(value_pages=torch.zeros(6, 2, 16, 128, dtype=torch.float16)),
    "shared slots": dict(key_pages=torch.zeros(1, 2, 16, 128, dtype=BF16).expand(6, 2, 16, 128)),
    "channel stride": dict(key_pages=torch.zeros(6, 2, 128, 16, dtype=BF16).transpose(2, 3)),
    "rows off 16 bytes": dict(key_pages=torch.zeros(6 * 2 * 16 * 128 + 8, dtype=BF16)[4:-4].view(6, 2, 16, 128)),
    "row stride": dict(key_pages=torch.zeros(6, 2, 16, 132, dtype=BF16)[..., :128]),
    "table type": dict(page_table=torch.zeros(2, 3, dtype=torch.int64)),
    "table rank": dict(page_table=torch.zeros(6, dtype=I32)),
    "empty table": dict(page_table=torch.zeros(2, 0, dtype=I32)),
    "table stride": dict(page_table=torch.zeros(3, 2, dtype=I32).t()),
    "batch past 1024": dict(page_table=torch.zeros(1025, 1, dtype=I32), lengths=torch.zeros(1025, dtype=I32)),
    "lengths type": dict(lengths=torch.zeros(2, dtype=torch.int64)),
    "lengths shape": dict(lengths=torch.zeros(3, dtype=I32)),
    "weights type": dict(weight_pages=torch.zeros(6, 2, 16, dtype=torch.float64)),
    "weights shape": dict(weight_pages=torch.zeros(6, 2, 32)),
    "weights stride": dict(weight_pages=torch.zeros(6, 16, 2).transpose(1, 2)),
    "weights shared": dict(weight_pages=torch.zeros(1, 2, 16).expand(6, 2, 16)),
}


@pytest.mark.parametrize("what", BAD)
def test_refused_caches(what):
    with pytest.raises(ValueError):
        ro.PagedCache(**_tensors(**BAD[what]))


def test_a_cache_on_the_cpu_is_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        ro.PagedCache(**_tensors())


@pytest.fixture
def cache(monkeypatch):
    """A cache of CPU tensors; a launch raises."""
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)

    def launch(name, params, device):
        raise AssertionError("launched")

    monkeypatch.setattr(_lib, "launch", launch)
    monkeypatch.setattr(_lib, "num_cus", lambda device: 256)
    return ro.PagedCache(**_tensors())


def _rows(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def test_refused_extends(cache):
    k = _rows(2, 2, 5, 128)
    bad = [(k[0], k[0], {}), (k[:1], k[:1], {}), (k[:, :1], k[:, :1], {}), (k[:, :, :0], k[:, :, :0], {}), (k[..., :64], k[..., :64], {}),
           (k, k[:, :, :4], {}), (k.half(), k.half(), {}), (k, k.half(), {}), (_rows(2, 2, 49, 128), _rows(2, 2, 49, 128), {}),
           (k, k, {"counts": torch.zeros(2)}), (k, k, {"counts": torch.zeros(3, dtype=I32)}), (k, k, {"weights": torch.zeros(2, 2, 4)}),
           (k, k, {"weights": torch.zeros(2, 2, 5, dtype=torch.float64)})]
    for key, value, options in bad:
        with pytest.raises(ValueError):
            ro.paged_extend(cache, key, value, **options)
    import dataclasses
    with pytest.raises(ValueError, match="weight_pages"):
        ro.paged_extend(dataclasses.replace(cache, weight_pages=None), k, k, weights=torch.zeros(2, 2, 5))
    with pytest.raises(AssertionError, match="launched"):
        ro.paged_extend(cache, k, k, weights=torch.zeros(2, 2, 5))


def test_refused_attention(cache):
    q, k = _rows(2, 4, 128), _rows(2, 2, 128)
    bad = [(q[0], {}), (q[:1], {}), (q[..., :64], {}), (q[:, :3], {}), (_rows(2, 34, 128), {}), (q.half(), {}), (_rows(2, 4, 2, 128), {}),
           (q, {"window": 0}), (q, {"sinks": -1}), (q, {"sm_scale": -1.0}), (q, {"sm_scale": float("inf")}),
           (q, {"append": (k, k[:, :1])}), (q, {"append": (k.half(), k.half())}), (q, {"append": (_rows(2, 4, 128), _rows(2, 4, 128))}),
           (q, {"output": (q, torch.zeros(2, 3))}), (q, {"output": (q.half(), torch.zeros(2, 4))}),
           (q, {"output": (_rows(2, 4, 256)[..., :128], torch.zeros(2, 4))}), (q, {"output": (q, torch.zeros(2, 4, dtype=torch.float64))})]
    for query, options in bad:
        with pytest.raises(ValueError):
            ro.paged_attention(query, cache, **options)
    with pytest.raises(RuntimeError, match="backward"):
        ro.paged_attention(_rows(2, 4, 128).requires_grad_(), cache)
    with pytest.raises(AssertionError, match="launched"):
        ro.paged_attention(q, cache, append=(k, k), window=4, sinks=1)


def test_refused_evictions(cache):
    import dataclasses

    other = dataclasses.replace(cache, page_table=torch.zeros(2, 3, dtype=I32), lengths=torch.zeros(2, dtype=I32))
    with pytest.raises(ValueError, match="weight_pages"):
        ro.paged_evict(dataclasses.replace(cache, weight_pages=None), other, 4)
    bad = [(other, 0, {}), (other, 49, {}), (other, 8, {"sinks": -1}), (other, 8, {"recent": -1}), (other, 8, {"sinks": 4, "recent": 5}),
           (cache, 4, {}), (dataclasses.replace(other, lengths=cache.lengths), 4, {}),
           (dataclasses.replace(other, page_table=torch.zeros(1, 3, dtype=I32), lengths=torch.zeros(1, dtype=I32)), 4, {}),
           (ro.PagedCache(**_tensors(key_pages=_rows(6, 1, 16, 128), value_pages=_rows(6, 1, 16, 128), weight_pages=None)), 4, {}),
           (ro.PagedCache(**_tensors(key_pages=_rows(6, 2, 16, 128).half(), value_pages=_rows(6, 2, 16, 128).half())), 4, {})]
    for target, keep, options in bad:
        with pytest.raises(ValueError):
            ro.paged_evict(cache, target, keep, **options)
    with pytest.raises(AssertionError, match="launched"):
        ro.paged_evict(cache, other, 8, sinks=4, recent=4)


# ----------------------------------------------------------------------------------------- the C ABI
def _c(n, *v):
    return (ctypes.c_int64 * n)(*v)


def _c_cache(**kw):
    c = _lib.PagedCacheParams(key_pages=0x1000, value_pages=0x2000, weight_pages=0x3000, page_table=0x4000, lengths=0x5000,
                              key_strides=_c(3, 4096, 2048, 128), value_strides=_c(3, 4096, 2048, 128),
                              weight_strides=_c(2, 32, 16), table_stride=3, pages=6, max_pages=3, page_size=16, batch=2, hkv=2)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHE = {
    "no keys": dict(key_pages=None), "misaligned values": dict(value_pages=0x2008), "no table": dict(page_table=None),
    "no lengths": dict(lengths=None), "misaligned weights": dict(weight_pages=0x3002), "stride": dict(key_strides=_c(3, 4096, 2048, 132)),
    "negative stride": dict(value_strides=_c(3, 4096, -2048, 128)), "stride past 2^31": dict(key_strides=_c(3, 1 << 31, 2048, 128)),
    "table stride": dict(table_stride=2), "no pages": dict(pages=0), "pages past 2^31": dict(pages=1 << 31), "no slots": dict(max_pages=0),
    "slots past 2^29": dict(max_pages=(1 << 25) + 1, table_stride=1 << 26), "page size": dict(page_size=48), "no batch": dict(batch=0),
    "batch past 1024": dict(batch=1025), "no heads": dict(hkv=0), "type": dict(dtype=2),
}


def _extend(**kw):
    p = _lib.PagedExtend(cache=_c_cache(), key=0x6000, value=0x7000, key_strides=_c(3, 2048, 1024, 128), value_strides=_c(3, 2048, 1024, 128),
                         rows=8)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _attention(**kw):
    p = _lib.PagedAttention(cache=_c_cache(), query=0x6000, query_strides=_c(2, 512, 128), hq=4, sm_scale=0.1, out=0x7000, lse=0x8000,
                            partial_out=0x9000, partial_ml=0xA000, logits=0xB000, partial_states=(8 + 4) * 2, logits_floats=2 * 4 * 64,
                            workers=8)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _evict(**kw):
    p = _lib.PagedEvict(source=_c_cache(), target=_c_cache(page_table=0x6000, lengths=0x7000), keep=8, sinks=2, recent=2, kept=0x8000,
                        target_lengths=0x7000)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("what", BAD_CACHE)
def test_c_abi_refuses_caches(what):
    lib, bad = _lib.load(), _c_cache(**BAD_CACHE[what])
    assert lib.r2o_paged_extend(ctypes.byref(_extend(cache=bad)), None) == 1
    assert lib.r2o_paged_attention(ctypes.byref(_attention(cache=bad)), None) == 1
    assert lib.r2o_paged_evict(ctypes.byref(_evict(source=bad)), None) == 1
    assert lib.r2o_paged_evict(ctypes.byref(_evict(target=bad)), None) == 1


def test_c_abi_refuses_arguments():
    lib = _lib.load()
    for kw in (dict(key=None), dict(value=0x7008), dict(rows=0), dict(counts=0x8002), dict(weights=0x9001), dict(key_strides=_c(3, 2048, 1024, 4)),
               dict(weights=0x9000, cache=_c_cache(weight_pages=None)), dict(weights=0x9000, weights_strides=_c(2, -1, 8))):
        assert lib.r2o_paged_extend(ctypes.byref(_extend(**kw)), None) == 1, kw
    for kw in (dict(query=None), dict(query=0x6008), dict(query_strides=_c(2, 512, 4)), dict(hq=3), dict(hq=1), dict(hq=34), dict(out=None),
               dict(out=0x7008), dict(lse=None), dict(window=-1), dict(sinks=-1), dict(sm_scale=0.0), dict(sm_scale=float("nan")),
               dict(append_key=0xC000), dict(append_key=0xC000, append_value=0xD008), dict(partial_out=None), dict(partial_ml=0xA004),
               dict(logits=None), dict(partial_states=23), dict(logits_floats=511), dict(workers=0), dict(workers=4097)):
        assert lib.r2o_paged_attention(ctypes.byref(_attention(**kw)), None) == 1, kw
    for kw in (dict(keep=0), dict(keep=49), dict(sinks=-1), dict(recent=-1), dict(sinks=5, recent=4), dict(kept=None), dict(target_lengths=None),
               dict(target_lengths=0x5000), dict(source=_c_cache(weight_pages=None)), dict(target=_c_cache(dtype=1)),
               dict(target=_c_cache(hkv=1)), dict(target=_c_cache(batch=1))):
        assert lib.r2o_paged_evict(ctypes.byref(_evict(**kw)), None) == 1, kw
    for fn in (lib.r2o_paged_extend, lib.r2o_paged_attention, lib.r2o_paged_evict):
        assert fn(None, None) == 1


def test_struct_layouts_match_the_header(tmp_path):
    from test_abi import _c_layout

    for struct, cls in (("r2o_prompt_params", _lib.PromptParams), ("r2o_paged_cache", _lib.PagedCacheParams),
                        ("r2o_paged_extend_params", _lib.PagedExtend), ("r2o_paged_attention_params", _lib.PagedAttention),
                        ("r2o_paged_evict_params", _lib.PagedEvict)):
        names = [f[0] for f in cls._fields_]
        offsets, size = _c_layout(struct, names, tmp_path)
        assert [getattr(cls, n).offset for n in names] == offsets, struct
        assert ctypes.sizeof(cls) == size, struct


def test_rows_that_need_a_gradient_are_refused(cache):
    plain, grad = _rows(2, 2, 5, 128), _rows(2, 2, 5, 128).requires_grad_()
    for key, value in ((grad, plain), (plain, grad)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            ro.paged_extend(cache, key, value)
        with pytest.raises(RuntimeError, match="no backward pass"):
            ro.paged_attention(_rows(2, 4, 128), cache, append=(key[:, :, 0], value[:, :, 0]))
        with torch.no_grad(), pytest.raises(AssertionError, match="launched"):
            ro.paged_extend(cache, key, value)


def test_evictions_into_overlapping_lengths_are_refused(cache):
    both = torch.zeros(3, dtype=I32)
    source = ro.PagedCache(**_tensors(lengths=both[:2]))
    target = ro.PagedCache(**_tensors(lengths=both[1:]))
    with pytest.raises(ValueError, match="lengths of its own"):
        ro.paged_evict(source, target, 8)
    lib = _lib.load()
    assert lib.r2o_paged_evict(ctypes.byref(_evict(target_lengths=0x5004)), None) == 1
    assert lib.r2o_paged_evict(ctypes.byref(_evict(target_lengths=0x4ffc)), None) == 1
