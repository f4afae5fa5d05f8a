"""What attention over shared prefixes refuses, on the CPU: the Python checks come before the device, and the C ABI checks its
own arguments before a launch."""
import ctypes
import dataclasses

import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib
from test_paged_refusals import BAD_CACHE, I32, _c, _c_cache, _rows, _tensors, cache  # noqa: F401


def _pair(cache):  # noqa: F811
    own = dataclasses.replace(cache, weight_pages=None)
    return own, dataclasses.replace(own, page_table=torch.zeros(1, 3, dtype=I32), lengths=torch.zeros(1, dtype=I32))


def test_refused_calls(cache):  # noqa: F811
    own, shared = _pair(cache)
    q, two = _rows(2, 4, 5, 128), dataclasses.replace(own)
    lse = torch.zeros(2, 4, 5)
    bad = [(q[0], own, shared, {}), (q[:1], own, shared, {}), (q[..., :64], own, shared, {}), (q[:, :3], own, shared, {}), (q[:, :0], own, shared, {}),
           (q[:, :, :0], own, shared, {}), (q.half(), own, shared, {}), (q.float(), own, shared, {}), (q.to("meta"), own, shared, {}),
           (_rows(2, 4, 2, 5, 128), own, shared, {}), (q, cache, shared, {}), (q, own, dataclasses.replace(shared, weight_pages=cache.weight_pages), {}),
           (q, own, two, {}),  # two prefixes without members
           (q, own, None, {"members": torch.zeros(1, dtype=I32)}), (q, own, shared, {"members": torch.zeros(2, dtype=I32)}),
           (q, own, shared, {"members": torch.zeros(1, dtype=torch.int64)}), (q, own, shared, {"members": torch.zeros(1, dtype=I32, device="meta")}),
           (q, own, shared, {"query_lengths": torch.zeros(1, dtype=I32)}), (q, own, shared, {"query_lengths": torch.zeros(2)}),
           (q, own, shared, {"sm_scale": 0.0}), (q, own, shared, {"sm_scale": -1.0}), (q, own, shared, {"sm_scale": float("nan")}),
           (q, own, shared, {"sm_scale": float("inf")}), (q, own, shared, {"output": (q[:, :, :4], lse)}),
           (q, own, shared, {"output": (q.half(), lse)}), (q, own, shared, {"output": (_rows(2, 4, 5, 132)[..., :128], lse)}),
           (q, own, shared, {"output": (torch.zeros_like(q), lse[:, :, :4])}), (q, own, shared, {"output": (torch.zeros_like(q), lse.double())}),
           (q, own, shared, {"output": (torch.zeros_like(q), torch.zeros(2, 4, 10)[..., ::2])}),
           (q, own, shared, {"output": (torch.zeros_like(q), lse.to("meta"))})]
    for query, requests, prefix, options in bad:
        with pytest.raises(ValueError):
            ro.paged_prefix_attention(query, requests, prefix, **options)
    other = _tensors(key_pages=_rows(6, 1, 16, 128), value_pages=_rows(6, 1, 16, 128), weight_pages=None)
    half = _tensors(key_pages=_rows(6, 2, 16, 128).half(), value_pages=_rows(6, 2, 16, 128).half(), weight_pages=None)
    for tensors in (other, half):
        with pytest.raises(ValueError, match="heads, dtype and device"):
            ro.paged_prefix_attention(q, own, ro.PagedCache(**tensors), members=torch.zeros(2, dtype=I32))
    for prefix in (shared, None):
        with pytest.raises(AssertionError, match="launched"):
            ro.paged_prefix_attention(q, own, prefix, output=(torch.zeros_like(q), lse))
        with pytest.raises(AssertionError, match="launched"):
            ro.paged_prefix_attention(q[:, :, 0], own, prefix)


def test_more_tiles_than_a_call_counts_are_refused(cache):  # noqa: F811
    """2^29 slots of 1024 requests: no memory, for the cache is one table of them."""
    many = ro.PagedCache(**_tensors(page_table=torch.zeros(1, 1 << 22, dtype=I32).expand(1024, 1 << 22), lengths=torch.zeros(1024, dtype=I32),
                                    weight_pages=None))
    with pytest.raises(ValueError, match="tiles"):
        ro.paged_prefix_attention(_rows(1, 4, 1, 128).expand(1024, 4, 1, 128), many)


def test_the_tables_of_many_rows_need_no_more_memory_than_they_have(cache):  # noqa: F811
    with pytest.raises(ValueError, match="2\\^30"):
        own, _ = _pair(cache)
        ro.paged_prefix_attention(_rows(1, 1, 1, 128).expand(2, 4, 1 << 28, 128), own)


# ----------------------------------------------------------------------------------------- the C ABI
def _plain(**kw):
    return _c_cache(weight_pages=None, **kw)


SCRATCH = 130 * (512 * 8 + 2 * 2 * 4 * 5) + 8 * 9


def _attention(**kw):
    p = _lib.PagedPrefix(cache=_plain(), prefix=_plain(batch=1, page_table=0x14000, lengths=0x15000), query=0x6000, out=0x7000, lse=0x8000,
                         q_strides=_c(3, 2560, 640, 128), o_strides=_c(3, 2560, 640, 128), hq=4, rows=5, sm_scale=0.1, scratch=0x9000,
                         scratch_floats=SCRATCH, workers=8)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("what", BAD_CACHE)
def test_c_abi_refuses_caches(what):
    lib = _lib.load()
    bad = _c_cache(**{"weight_pages": None} | BAD_CACHE[what])
    assert lib.r2o_paged_prefix_attention(ctypes.byref(_attention(cache=bad)), None) == 1
    if bad.batch:  # 0: there is no prefix
        if bad.batch == 2:
            bad.batch = 1
        assert lib.r2o_paged_prefix_attention(ctypes.byref(_attention(prefix=bad)), None) == 1


def test_c_abi_refuses_arguments():
    lib = _lib.load()
    for kw in (dict(cache=_c_cache()), dict(prefix=_c_cache(batch=1)), dict(prefix=_plain(batch=1, hkv=1)), dict(prefix=_plain(batch=1, dtype=1)),
               dict(prefix=_plain(batch=2)), dict(prefix=_plain(batch=-1)), dict(members=0x16002), dict(query_lengths=0x16001), dict(query=None),
               dict(query=0x6008), dict(out=None), dict(out=0x7008), dict(lse=None), dict(lse=0x8002), dict(q_strides=_c(3, 2560, 640, 4)),
               dict(q_strides=_c(3, 2560, -640, 128)), dict(q_strides=_c(3, 2560, 640, (1 << 24) + 8)), dict(o_strides=_c(3, 2560, 640, (1 << 24) + 8)),
               dict(hq=1), dict(hq=5), dict(hq=0), dict(hq=-4), dict(hq=1 << 62), dict(hq=1 << 30), dict(rows=0), dict(rows=-1), dict(rows=1 << 29),
               dict(rows=1 << 62), dict(sm_scale=0.0), dict(sm_scale=-0.1), dict(sm_scale=float("nan")), dict(sm_scale=float("inf")),
               dict(scratch=None), dict(scratch=0x9008), dict(scratch_floats=SCRATCH - 1), dict(workers=0), dict(workers=4097),
               dict(cache=_plain(batch=1024, max_pages=1 << 25, table_stride=1 << 25), scratch_floats=1 << 40)):
        assert lib.r2o_paged_prefix_attention(ctypes.byref(_attention(**kw)), None) == 1, kw
    assert lib.r2o_paged_prefix_attention(None, None) == 1


def test_struct_layout_matches_the_header(tmp_path):
    from test_abi import _c_layout

    names = [f[0] for f in _lib.PagedPrefix._fields_]
    offsets, size = _c_layout("r2o_paged_prefix_params", names, tmp_path)
    assert [getattr(_lib.PagedPrefix, n).offset for n in names] == offsets and ctypes.sizeof(_lib.PagedPrefix) == size


@pytest.mark.parametrize("batch,hkv,hq,rows,slots,prefixes,shared,counted", [
    (1, 1, 1, 1, 16, 0, 0, 0), (1, 1, 1, 1, 16, 1, 16, 0), (2, 2, 14, 1, 1000, 1, 32000, 0), (64, 4, 28, 40, 1024, 1, 32768, 1),
    (64, 4, 28, 64, 1024, 8, 32768, 0), (1024, 2, 16, 511, 16, 3, 2048, 1), (1, 4, 28, 32768, 32768, 0, 0, 0)])
def test_the_plan_of_a_call(batch, hkv, hq, rows, slots, prefixes, shared, counted):
    """Workgroups: at most one a compute unit; the scratch that the C call asks for, not a float more or less."""
    plan = _lib.host().prefix_plan(batch, hkv, hq, rows, slots, prefixes, shared, counted, 256)
    assert 1 <= plan[0] <= 256
    packed, total = hq // hkv * rows, batch * hq * rows
    room = packed < 128 or (packed < 512 and total <= 1 << 18)
    assert plan[1] == 130 * (512 * plan[0] + (2 * total if room else 0)) + 8 * (1 + max(batch, plan[0]))
    bad = _attention(cache=_plain(batch=batch, hkv=hkv, max_pages=slots // 16 or 1, table_stride=slots // 16 or 1),
                     prefix=_plain(batch=prefixes, hkv=hkv, max_pages=max(1, shared // 16), table_stride=max(1, shared // 16)), members=0x16000, hq=hq,
                     rows=rows, workers=plan[0], scratch_floats=plan[1] - 1, query_lengths=0x17000 if counted else None)
    assert _lib.load().r2o_paged_prefix_attention(ctypes.byref(bad), None) == 1


def test_no_plan_where_the_units_are_too_many():
    assert _lib.host().prefix_plan(1024, 4, 28, 1, 1 << 29, 0, 0, 0, 256) == (0, 0)
