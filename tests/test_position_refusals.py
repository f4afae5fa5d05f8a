"""What the calls that rotate by positions refuse, on the CPU: the Python checks come before the device, and the C ABI
checks its own arguments before a launch."""
import ctypes
import dataclasses

import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib
from test_paged_refusals import BAD_CACHE, BF16, I32, _c, _c_cache, _rows, _tensors, cache  # noqa: F401

NORM = torch.ones(128, dtype=BF16)


def _rotary(**change):
    return ro.PositionRotary(**({"inv_freq": torch.ones(64)} | change))


BAD_ROTARY = {
    "inv_freq shape": dict(inv_freq=torch.ones(128)), "inv_freq rank": dict(inv_freq=torch.ones(1, 64)),
    "inv_freq type": dict(inv_freq=torch.ones(64, dtype=BF16)), "inv_freq device": dict(inv_freq=torch.ones(64, device="meta")),
    "section sum": dict(mrope_section=(16, 24, 23)), "no section": dict(mrope_section=()), "four axes": dict(mrope_section=(16, 16, 16, 16)),
    "negative section": dict(mrope_section=(72, -8)), "turns of three": dict(mrope_section=(20, 22, 22), interleaved=True),
    "more than the turns": dict(mrope_section=(0, 32, 32), interleaved=True), "one weight": dict(q_norm_weight=NORM),
    "the other weight": dict(k_norm_weight=NORM), "weight type": dict(q_norm_weight=NORM.float(), k_norm_weight=NORM.float()),
    "weight shape": dict(q_norm_weight=NORM[:64], k_norm_weight=NORM[:64]),
    "weight device": dict(q_norm_weight=NORM, k_norm_weight=NORM.to("meta")), "eps below 0": dict(eps=-1e-6),
    "eps NaN": dict(eps=float("nan")), "eps infinite": dict(eps=float("inf")), "scaling NaN": dict(scaling=float("nan")),
    "scaling infinite": dict(scaling=float("-inf")),
}


def _positions(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("what", BAD_ROTARY)
def test_refused_rotations(what, cache):  # noqa: F811
    rotary, q, k = _rotary(**BAD_ROTARY[what]), _rows(2, 4, 5, 128), _rows(2, 2, 5, 128)
    axes = len(rotary.mrope_section)
    for positions in (_positions(axes, 2, 5), _positions(2, 5)):
        with pytest.raises(ValueError):
            ro.qk_position_rope(q, k, positions, rotary)
    with pytest.raises(ValueError):
        ro.paged_rope_extend(cache, q, k, k, rotary)


def test_refused_positions(cache):  # noqa: F811
    q, k = _rows(2, 4, 5, 128), _rows(2, 2, 5, 128)
    three = _rotary(mrope_section=(16, 24, 24))
    bad = [(_rotary(), _positions(2, 4)), (_rotary(), _positions(1, 5)), (_rotary(), _positions(3, 2, 5)), (three, _positions(2, 5)),
           (three, _positions(2, 2, 5)), (_rotary(), _positions(2, 5, dtype=torch.int16)), (_rotary(), torch.zeros(2, 5)),
           (_rotary(), _positions(2, 5).to("meta")), (_rotary(), _positions(5))]
    for rotary, positions in bad:
        with pytest.raises(ValueError, match="positions"):
            ro.qk_position_rope(q, k, positions, rotary)
        with pytest.raises(ValueError, match="positions"):
            ro.paged_rope_extend(cache, q, k, k, rotary, positions=positions)
    with pytest.raises(ValueError, match="positions"):
        ro.qk_position_rope(q, k, None, _rotary())


def test_refused_rows(cache):  # noqa: F811
    q, k, r, at = _rows(2, 4, 5, 128), _rows(2, 2, 5, 128), _rotary(), _positions(2, 5)
    bad = [(q[0], k[0]), (q[..., :64], k[..., :64]), (q, k[:1]), (q, k[:, :, :4]), (q[:, :0], k), (q, k[:, :0]), (q[:, :, :0], k[:, :, :0]),
           (q, k.half()), (q.float(), k.float()), (q, k.to("meta"))]
    for query, key in bad:
        with pytest.raises(ValueError):
            ro.qk_position_rope(query, key, at, r)
        with pytest.raises(ValueError):
            ro.paged_rope_extend(cache, query, key, key, r)
    outputs = [(q[:, :, :4], k), (q, k[:, :1]), (q.half(), k), (q, k.float()), (_rows(2, 4, 5, 256)[..., ::2], k),
               (_rows(2, 4, 5, 132)[..., :128], k), (q, k.to("meta")), (_rows(1, 4, 5, 128).expand(2, 4, 5, 128), k)]
    for output in outputs:
        with pytest.raises(ValueError):
            ro.qk_position_rope(q, k, at, r, output=output)
        if output[1] is k:
            with pytest.raises(ValueError):
                ro.paged_rope_extend(cache, q, k, k, r, output=output[0])
    with pytest.raises(AssertionError, match="launched"):
        ro.qk_position_rope(q, k, at, r, output=(q, k))


def test_a_call_on_the_cpu_is_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        ro.qk_position_rope(_rows(2, 4, 5, 128), _rows(2, 2, 5, 128), _positions(2, 5), _rotary())


def test_refused_extends(cache):  # noqa: F811
    q, k, r = _rows(2, 4, 5, 128), _rows(2, 2, 5, 128), _rotary()
    bad = [(q[:1], k[:1], k[:1], {}), (_rows(3, 4, 5, 128), _rows(3, 2, 5, 128), _rows(3, 2, 5, 128), {}), (q, q, q, {}), (q, k[:, :1], k[:, :1], {}),
           (q, k, k[:, :, :4], {}), (q, k, k.half(), {}), (q.half(), k.half(), k.half(), {}),
           (_rows(2, 4, 49, 128), _rows(2, 2, 49, 128), _rows(2, 2, 49, 128), {}), (q, k, k, {"counts": torch.zeros(2)}),
           (q, k, k, {"counts": torch.zeros(3, dtype=I32)}), (q, k, k, {"weights": torch.zeros(2, 2, 4)}),
           (q, k, k, {"weights": torch.zeros(2, 2, 5, dtype=torch.float64)}), (q, k, k, {"weights": torch.zeros(2, 2, 5, device="meta")})]
    for query, key, value, options in bad:
        with pytest.raises(ValueError):
            ro.paged_rope_extend(cache, query, key, value, r, **options)
    with pytest.raises(ValueError, match="weight_pages"):
        ro.paged_rope_extend(dataclasses.replace(cache, weight_pages=None), q, k, k, r, weights=torch.zeros(2, 2, 5))
    with pytest.raises(ValueError):  # one table row for all requests: the rows of one would be another's
        ro.paged_rope_extend(dataclasses.replace(cache, page_table=torch.zeros(1, 3, dtype=I32).expand(2, 3)), q, k, k, r)
    with pytest.raises(AssertionError, match="launched"):
        ro.paged_rope_extend(cache, q, k, k, r, weights=torch.zeros(2, 2, 5), counts=torch.zeros(2, dtype=I32))


# ----------------------------------------------------------------------------------------- the C ABI
def _rotation(**kw):
    r = _lib.Rotation(positions=0x10000, position_strides=_c(3, 10, 5, 1), position_bytes=8, axes=3, inv_freq=0x11000, freq_bytes=4,
                      pairs_1=0xFF0000, pairs_2=0xFF000000, q_weight=0x12000, k_weight=0x13000, eps=1e-6, scaling=1.0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _rope(**kw):
    p = _lib.PositionRope(rotation=_rotation(), query=0x6000, key=0x7000, query_out=0x6000, key_out=0x7000, q_strides=_c(3, 2560, 640, 128),
                          k_strides=_c(3, 1280, 640, 128), qo_strides=_c(3, 2560, 640, 128), ko_strides=_c(3, 1280, 640, 128), batch=2, hq=4,
                          hkv=2, tokens=5)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _extend(**kw):
    p = _lib.PagedRopeExtend(cache=_c_cache(), rotation=_rotation(), query=0x6000, key=0x7000, value=0x8000, query_out=0x6000,
                             q_strides=_c(3, 2560, 640, 128), k_strides=_c(3, 1280, 640, 128), v_strides=_c(3, 1280, 640, 128),
                             qo_strides=_c(3, 2560, 640, 128), hq=4, rows=5)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


BAD_C_ROTATION = {
    "misaligned positions": dict(positions=0x10004), "position bytes": dict(position_bytes=2), "position stride": dict(position_strides=_c(3, 10, -5, 1)),
    "no axis": dict(axes=0), "four axes": dict(axes=4), "no inv_freq": dict(inv_freq=None), "misaligned inv_freq": dict(inv_freq=0x11002),
    "inv_freq bytes": dict(freq_bytes=2), "a pair of two axes": dict(pairs_2=0xFF0000), "a pair of a missing axis": dict(axes=2),
    "one weight": dict(k_weight=None), "misaligned weight": dict(q_weight=0x12008), "eps": dict(eps=-1.0), "eps NaN": dict(eps=float("nan")),
    "scaling": dict(scaling=float("inf")),
}


@pytest.mark.parametrize("what", BAD_C_ROTATION)
def test_c_abi_refuses_rotations(what):
    lib, bad = _lib.load(), _rotation(**BAD_C_ROTATION[what])
    assert lib.r2o_position_rope(ctypes.byref(_rope(rotation=bad)), None) == 1
    assert lib.r2o_paged_rope_extend(ctypes.byref(_extend(rotation=bad)), None) == 1


@pytest.mark.parametrize("what", BAD_CACHE)
def test_c_abi_refuses_caches(what):
    assert _lib.load().r2o_paged_rope_extend(ctypes.byref(_extend(cache=_c_cache(**BAD_CACHE[what]))), None) == 1


def test_c_abi_refuses_arguments():
    lib = _lib.load()
    for kw in (dict(query=None), dict(key=0x7008), dict(query_out=None), dict(key_out=0x7004), dict(q_strides=_c(3, 2560, 640, 132)),
               dict(k_strides=_c(3, -8, 640, 128)), dict(qo_strides=_c(3, 2564, 640, 128)), dict(ko_strides=_c(3, 1280, 640, -128)), dict(batch=0),
               dict(hq=0), dict(hkv=0), dict(tokens=0), dict(hq=1 << 31), dict(hkv=1 << 31), dict(batch=1 << 31), dict(tokens=1 << 31),
               dict(batch=1 << 20, tokens=1 << 20), dict(dtype=2), dict(dtype=-1), dict(rotation=_rotation(positions=None))):
        assert lib.r2o_position_rope(ctypes.byref(_rope(**kw)), None) == 1, kw
    for kw in (dict(query=None), dict(key=None), dict(value=0x8002), dict(query_out=None), dict(q_strides=_c(3, 2560, 640, 4)),
               dict(v_strides=_c(3, 1280, -640, 128)), dict(hq=0), dict(hq=1 << 31), dict(rows=0), dict(rows=(1 << 29) + 1), dict(counts=0x9002),
               dict(weights=0x9002), dict(weights=0x9000, weights_strides=_c(2, -1, 5)), dict(weights=0x9000, cache=_c_cache(weight_pages=None)),
               dict(cache=_c_cache(table_stride=0))):
        assert lib.r2o_paged_rope_extend(ctypes.byref(_extend(**kw)), None) == 1, kw
    assert lib.r2o_position_rope(None, None) == 1 and lib.r2o_paged_rope_extend(None, None) == 1


def test_struct_layouts_match_the_header(tmp_path):
    from test_abi import _c_layout

    for struct, cls in (("r2o_rotation", _lib.Rotation), ("r2o_position_rope_params", _lib.PositionRope),
                        ("r2o_paged_rope_extend_params", _lib.PagedRopeExtend)):
        names = [f[0] for f in cls._fields_]
        offsets, size = _c_layout(struct, names, tmp_path)
        assert [getattr(cls, n).offset for n in names] == offsets, struct
        assert ctypes.sizeof(cls) == size, struct


@pytest.mark.parametrize("section,interleaved,want", [
    ((64,), False, ("0" * 64,)), ((16, 24, 24), False, ("0" * 16 + "1" * 24 + "2" * 24,)), ((0, 64), False, ("1" * 64,)),
    ((24, 20, 20), True, ("012" * 20 + "0000",)), ((22, 21, 21), True, ("012" * 21 + "0",)), ((64, 0, 0), True, ("0" * 64,))])
def test_axes_of_the_pairs(section, interleaved, want):
    masks = _rotary(mrope_section=section, interleaved=interleaved).axis_pairs()
    assert "".join(str(next(a for a in range(3) if masks[a] >> i & 1)) for i in range(64)) == want[0]
    assert sum(masks) == (1 << 64) - 1
