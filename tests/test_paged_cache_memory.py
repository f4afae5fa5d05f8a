"""Which memory a paged call uses: that of the cache's tensors at the time of the call.  On the CPU; what would be
launched is looked at instead."""
import copy
import ctypes
import io
import pickle

import pytest
import torch

import r2omni_amd as ro
from r2omni_amd import _lib

BF16, I32 = torch.bfloat16, torch.int32


@pytest.fixture
def launched(monkeypatch):
    """Parameters of the calls that would be launched."""
    calls = []
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(_lib, "launch", lambda name, params, device: calls.append(params))
    monkeypatch.setattr(_lib, "num_cus", lambda device: 256)
    return calls


def _cache(pages=6, **change):
    t = {"key_pages": torch.zeros(pages, 2, 16, 128, dtype=BF16), "value_pages": torch.zeros(pages, 2, 16, 128, dtype=BF16),
         "page_table": torch.zeros(2, 3, dtype=I32), "lengths": torch.zeros(2, dtype=I32), "weight_pages": torch.zeros(pages, 2, 16)}
    t.update(change)
    return ro.PagedCache(**t)


def _uses(params, cache):
    """The parameters name the cache's own tensors, with their sizes."""
    for name in ("key_pages", "value_pages", "weight_pages", "page_table", "lengths"):
        assert getattr(params, name) == getattr(cache, name).data_ptr(), name
    assert params.pages == cache.key_pages.shape[0] and params.max_pages == cache.page_table.shape[1]


def _every_call(cache, launched):
    """The cache parameters of an extend, an attention and an eviction out of and into the cache."""
    del launched[:]
    rows, other = torch.zeros(2, 2, 5, 128, dtype=BF16), _cache()
    ro.paged_extend(cache, rows, rows)
    ro.paged_attention(rows[:, :, 0], cache, append=(rows[:, :, 0], rows[:, :, 1]))
    ro.paged_evict(cache, other, 8)
    ro.paged_evict(other, cache, 8)
    extend, attention, out, into = launched
    assert into.target_lengths == cache.lengths.data_ptr()
    return extend.cache, attention.cache, out.source, into.target


def _pickled(cache):
    return pickle.loads(pickle.dumps(cache))


def _saved(cache):
    buffer = io.BytesIO()
    torch.save(cache, buffer)
    buffer.seek(0)
    return torch.load(buffer, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, copy.copy, _pickled, _saved])
def test_a_copy_uses_its_own_tensors(how, launched):
    cache = _cache()
    other = how(cache)
    shared = how is copy.copy
    assert (other.key_pages.data_ptr() == cache.key_pages.data_ptr()) == shared
    for c in (other, cache):
        for params in _every_call(c, launched):
            _uses(params, c)


def test_tensors_that_got_other_memory_are_used_where_they_lie(launched):
    cache = _cache()
    for name, larger in (("key_pages", 9), ("value_pages", 9), ("weight_pages", 9)):
        t = getattr(cache, name)
        t.data = torch.zeros(larger, *t.shape[1:], dtype=t.dtype)
    cache.page_table.data = torch.zeros(2, 4, dtype=I32)
    cache.lengths.data = torch.zeros(2, dtype=I32)
    for params in _every_call(cache, launched):
        _uses(params, cache)


def test_tensors_that_no_longer_make_a_cache_are_refused(launched):
    rows = torch.zeros(2, 2, 5, 128, dtype=BF16)
    for name, bad in (("key_pages", torch.zeros(3, 2, 16, 128, dtype=BF16)), ("value_pages", torch.zeros(6, 2, 16, 128).half()),
                      ("page_table", torch.zeros(2, 3, dtype=torch.int64)), ("lengths", torch.zeros(1, dtype=I32)),
                      ("weight_pages", torch.zeros(6, 2, 8))):
        cache = _cache()
        getattr(cache, name).data = bad
        for call in (lambda: ro.paged_extend(cache, rows, rows), lambda: ro.paged_attention(rows[:, :, 0], cache),
                     lambda: ro.paged_evict(cache, _cache(), 8), lambda: ro.paged_evict(_cache(), cache, 8)):
            with pytest.raises(ValueError):
                call()
    assert not launched


@pytest.mark.parametrize("stride,ok", [(0, True), (1, False), (2, False), (3, True), (7, True)])
def test_page_table_strides_are_the_tables_own(stride, ok, launched):
    """Requests' rows lie where the table says; a row read by all is expanded, rows that overlap are refused."""
    table = torch.zeros(3 + 3 * stride, dtype=I32).as_strided((4, 3), (stride, 1))
    change = dict(page_table=table, lengths=torch.zeros(4, dtype=I32), weight_pages=None)
    if not ok:
        with pytest.raises(ValueError, match="overlap"):
            _cache(**change)
        return
    ro.paged_attention(torch.zeros(4, 2, 128, dtype=BF16), _cache(**change))
    assert launched[0].cache.table_stride == stride and launched[0].cache.batch == 4


def test_one_request_has_any_table_stride(launched):
    table = torch.zeros(3, dtype=I32).as_strided((1, 3), (1, 1))
    ro.paged_attention(torch.zeros(1, 2, 128, dtype=BF16), _cache(page_table=table, lengths=torch.zeros(1, dtype=I32), weight_pages=None))
    assert launched[0].cache.table_stride >= 3


def test_pages_of_an_expanded_table_are_not_written(launched):
    cache = _cache(page_table=torch.zeros(1, 3, dtype=I32).expand(2, -1))
    plain = _cache(page_table=torch.zeros(1, 3, dtype=I32).expand(2, -1), weight_pages=None)
    rows = torch.zeros(2, 2, 5, 128, dtype=BF16)
    for call in (lambda: ro.paged_extend(cache, rows, rows), lambda: ro.paged_attention(rows[:, :, 0], cache),
                 lambda: ro.paged_attention(rows[:, :, 0], plain, append=(rows[:, :, 0], rows[:, :, 0])),
                 lambda: ro.paged_evict(_cache(), cache, 8)):
        with pytest.raises(ValueError, match="one page for several requests"):
            call()
    assert not launched
    ro.paged_evict(cache, _cache(), 8)  # reads them
    assert launched[0].source.table_stride == 0


def test_c_abi_takes_one_row_for_reading_alone():
    """What is refused before a launch; the stride itself, and each call that writes."""
    from test_paged_refusals import _attention, _c_cache, _evict, _extend

    lib, one = _lib.load(), dict(table_stride=0)
    for overlapping in (1, 2, -3):
        assert lib.r2o_paged_attention(ctypes.byref(_attention(cache=_c_cache(table_stride=overlapping))), None) == 1
    assert lib.r2o_paged_extend(ctypes.byref(_extend(cache=_c_cache(**one))), None) == 1
    assert lib.r2o_paged_attention(ctypes.byref(_attention(cache=_c_cache(**one))), None) == 1
    plain = _attention(cache=_c_cache(weight_pages=None, **one), append_key=0xC000, append_value=0xD000)
    assert lib.r2o_paged_attention(ctypes.byref(plain), None) == 1
    assert lib.r2o_paged_evict(ctypes.byref(_evict(target=_c_cache(page_table=0x6000, lengths=0x7000, **one))), None) == 1
