"""A key-value cache of bf16 or fp16 rows in pages: writes, attention of one token, eviction by attention weight.

The packed cache (``cache.ThreePrecisionCache``) is built once from a prompt's plan; this one grows in place, in
pages that a server hands out, and gives up the tokens that received the least attention:

* ``paged_extend`` (``r2o_paged_extend``): a prompt's rows, or a chunk of them, into their slots.
* ``paged_attention`` (``r2o_paged_attention``): one new token per request over its filled slots, its own K and V
  rows appended by the same call, and the cache's accumulated weights advanced.
* ``paged_prefix_attention`` (``r2o_paged_prefix_attention``): the newest rows of each request (a step's token, or a
  question's) over a prefix that many requests share, whose rows are read once for all of them, and over its own slots.
* ``paged_evict`` (``r2o_paged_evict``): the tokens of largest accumulated weight, with the first and the newest
  ones, compacted in order into another page table.

Lengths are the caller's: a device tensor that already counts the rows being written, so one ``lengths.add_(1)``
serves every layer of a step and a captured graph reads each step's values.  No counterpart in the reference, which
keeps no unpacked cache once a prompt is packed.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .prompt import _check_like, _lengths, _like, _rows, _scale, _strides, _window

PAGE_SIZES = (16, 32, 64, 128)
MAX_BATCH = 1024


def _pool_ok(t: torch.Tensor) -> bool:
    """Rows in place, every slot its own memory."""
    return (t.stride(2) <= 1 << 24 and t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(0 < st < 1 << 31 and st % 8 == 0 for st, n in zip(t.stride()[:-1], t.shape) if n > 1))


@dataclass(frozen=True, eq=False)
class PagedCache:
    """The tensors that hold one layer's cache; the calls write them in place, where they lie at the time of the call.

    Slot j of request b is slot ``j % page_size`` of page ``page_table[b, j // page_size]``, for every KV head, and
    the first ``lengths[b]`` slots are filled.  A page id outside the pool (such as -1 for a page not handed out)
    makes its slots invisible: they are neither read nor written.  Requests may share pages that no call writes to
    (one row of ids expanded for all of them serves); a page whose rows or weights are written stands in the tables
    once.  Pool and head strides are free (views of one pool for both, or for all layers, serve), as long as channels
    are unit-strided and rows 16-byte aligned."""

    key_pages: torch.Tensor                     # bf16 / fp16 [pages, Hkv, page_size, 128]
    value_pages: torch.Tensor
    page_table: torch.Tensor                    # int32 [B, max_pages]
    lengths: torch.Tensor                       # int32 [B]
    weight_pages: torch.Tensor | None = None    # fp32 [pages, Hkv, page_size]: accumulated attention weight

    def __post_init__(self) -> None:
        if _lib.host().paged_cache(self) is None:
            _params_of(self)

    @property
    def capacity(self) -> int:
        """Slots that a row of the page table can hold."""
        return int(self.page_table.shape[1]) * int(self.key_pages.shape[2])


def _token_rows(t: torch.Tensor) -> torch.Tensor:
    """``_rows`` of [B, H, 128]; copied too where they lie farther apart than the kernels' 32 bits of elements."""
    t = _rows(t)
    return t.clone(memory_format=torch.contiguous_format) if any(st >= 1 << 31 for st, n in zip(t.stride(), t.shape) if n > 1) else t


def _params_of(cache: PagedCache) -> _lib.PagedCacheParams:
    """Where the cache's tensors lie now, checked.  Nothing is kept from one call for the next: a copied cache has tensors
    of its own, and ``t.data = ...`` gives one other memory."""
    k, v, table, n, w = cache.key_pages, cache.value_pages, cache.page_table, cache.lengths, cache.weight_pages
    if k.ndim != 4 or k.shape[-1] != 128 or min(k.shape) < 1 or v.shape != k.shape:
        raise ValueError("paged cache needs key and value pages [pages,Hkv,page_size,128] of one shape")
    if k.shape[2] not in PAGE_SIZES:
        raise ValueError("page_size must be one of 16, 32, 64, or 128")
    dtype = _lib.dtype_code(k.dtype)
    if v.dtype != k.dtype or any(t.device != k.device for t in (v, table, n)):
        raise ValueError("paged cache tensors must share a device and K/V a dtype")
    if not _pool_ok(k) or not _pool_ok(v):
        raise ValueError("paged cache pages need unit channel stride and 16-byte aligned rows of their own")
    if table.dtype != torch.int32 or table.ndim != 2 or min(table.shape) < 1 or table.stride(1) != 1 and table.shape[1] > 1:
        raise ValueError("page_table must be int32 [B,max_pages] with unit-strided rows")
    table_stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
    if 0 < table_stride < table.shape[1]:
        raise ValueError("page_table rows must not overlap (one expanded row for all requests is taken)")
    if n.dtype != torch.int32 or tuple(n.shape) != (table.shape[0],) or not n.is_contiguous():
        raise ValueError("lengths must be contiguous int32 [B]")
    if table.shape[0] > MAX_BATCH or table.shape[1] * k.shape[2] > 1 << 29 or k.shape[0] >= 1 << 31 or k.shape[1] > 1024 \
            or table_stride >= 1 << 31:
        raise ValueError("paged cache takes at most 1024 requests, 1024 heads and 2^29 slots a request")
    if w is not None and (w.shape != k.shape[:3] or w.dtype != torch.float32 or w.device != k.device
                          or any(not 0 < st < 1 << 31 for st, size in zip(w.stride(), w.shape) if size > 1) or w.stride(2) != 1):
        raise ValueError("weight_pages must be fp32 [pages,Hkv,page_size] on the cache's device with unit-strided slots")
    _lib.require_device(k, "paged cache")
    return _lib.PagedCacheParams(
        key_pages=k.data_ptr(), value_pages=v.data_ptr(), weight_pages=_lib.ptr(w), page_table=table.data_ptr(),
        lengths=n.data_ptr(), key_strides=_strides(k, 3), value_strides=_strides(v, 3),
        weight_strides=(0, 0) if w is None else _strides(w, 2), table_stride=table_stride,
        pages=k.shape[0], max_pages=table.shape[1], page_size=k.shape[2], batch=table.shape[0], hkv=k.shape[1],
        dtype=dtype)


def _pools(cache: PagedCache) -> tuple[torch.Tensor | None, ...]:
    return cache.key_pages, cache.value_pages, cache.weight_pages


def _check_written(cache: PagedCache, what: str) -> None:
    if cache.page_table.shape[0] > 1 and cache.page_table.stride(0) == 0:
        raise ValueError(f"{what} would write one page for several requests: the page table is one expanded row")


def _check_new_rows(cache: PagedCache, key: torch.Tensor, value: torch.Tensor, what: str) -> None:
    if value.shape != key.shape:
        raise ValueError(f"{what} K and V must have one shape")
    for t in (key, value):
        if t.dtype != cache.key_pages.dtype or t.device != cache.key_pages.device:
            raise ValueError(f"{what} rows must match the cache's dtype and device")
    _lib.refuse_gradients(what, key, value)


def _row_weights(cache: PagedCache, key: torch.Tensor, weights: torch.Tensor | None, what: str) -> torch.Tensor | None:
    """The new rows' weights, checked; unit-strided along the rows."""
    if weights is None:
        return None
    if cache.weight_pages is None:
        raise ValueError(f"{what} weights need a cache with weight_pages")
    if weights.shape != key.shape[:3] or weights.dtype != torch.float32 or weights.device != key.device:
        raise ValueError(f"{what} weights must be fp32 [B,Hkv,S] on the rows' device")
    return weights.contiguous() if weights.stride(2) != 1 and weights.shape[2] > 1 or min(weights.stride()) < 0 else weights


def paged_extend(cache: PagedCache, key: torch.Tensor, value: torch.Tensor, *, counts: torch.Tensor | None = None,
                 weights: torch.Tensor | None = None) -> None:
    """Write rows of key and value [B, Hkv, S, 128] into each request's newest slots.

    ``cache.lengths`` already counts them: row i of request b goes to slot ``lengths[b] - n + i``, where n is S or,
    for a padded batch, ``counts[b]`` (int32 [B]; rows behind it are not used).  Where the cache keeps weights, the
    slots get ``weights`` (fp32 [B, Hkv, S], as ``attention_weights`` returns them) or 0."""
    made = _lib.host().paged_extend(_lib.entry("r2o_paged_extend"), cache, key, value, counts, weights)
    if made is not None:
        return _lib.check(made[0], "r2o_paged_extend")
    batch, hkv = int(cache.page_table.shape[0]), int(cache.key_pages.shape[1])
    if key.ndim != 4 or key.shape[0] != batch or key.shape[1] != hkv or key.shape[2] < 1 or key.shape[3] != 128:
        raise ValueError("paged extend requires key and value [B,Hkv,S,128] of the cache's requests and heads")
    _check_new_rows(cache, key, value, "paged extend")
    _check_written(cache, "paged extend")
    if key.shape[2] > cache.capacity:
        raise ValueError("paged extend has more rows than the page table holds")
    counts = _lengths(counts, batch, key.device, "counts")
    weights = _row_weights(cache, key, weights, "paged extend")
    _lib.refuse_gradients("paged extend", weights, *_pools(cache))
    key, value = _rows(key), _rows(value)
    p = _lib.PagedExtend(cache=_params_of(cache), key=key.data_ptr(), value=value.data_ptr(), weights=_lib.ptr(weights),
                         counts=_lib.ptr(counts), key_strides=_strides(key, 3), value_strides=_strides(value, 3),
                         weights_strides=(0, 0) if weights is None else _strides(weights, 2), rows=key.shape[2])
    _lib.launch("r2o_paged_extend", p, key.device)


def paged_attention(query: torch.Tensor, cache: PagedCache, *, append: tuple[torch.Tensor, torch.Tensor] | None = None,
                    window: int | None = None, sinks: int = 0, sm_scale: float | None = None,
                    output: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Attention of one token per request, query [B, Hq, 128] or [B, Hq, 1, 128], over its filled slots; returns
    (out [B, Hq, 128] in the query's dtype, lse fp32 [B, Hq]).

    ``append=(key, value)``, [B, Hkv, 128] or [B, Hkv, 1, 128] each: the token's own rows.  ``cache.lengths`` already
    counts the token; its rows are attended, and written to slot ``lengths[b] - 1``.  With ``window``, the last
    ``window`` and the first ``sinks`` slots are seen.  Where the cache keeps weights, the weight of every slot seen
    grows by its probability summed over the query heads of its group (the appended slot's is set to it); a
    ``dataclasses.replace(cache, weight_pages=None)`` leaves them alone.  A request that sees no slot (an idle one of
    length 0) gets 0 and lse -inf; infinite and NaN values count as in ``prompt_attention``.  ``output``: the two
    contiguous result tensors."""
    if output is None:
        made = _lib.host().paged_attention(_lib.entry("r2o_paged_attention"), cache, query, append, window, sinks, sm_scale)
        if made is not None:
            _lib.check(made[0], "r2o_paged_attention")
            return made[1], made[2]
    batch, hkv = int(cache.page_table.shape[0]), int(cache.key_pages.shape[1])
    if query.ndim == 4 and query.shape[2] == 1:
        query = query[:, :, 0]
    if query.ndim != 3 or query.shape[0] != batch or query.shape[2] != 128 or query.shape[1] < 1:
        raise ValueError("paged attention requires query [B,Hq,128] of the cache's requests")
    hq = int(query.shape[1])
    if hq % hkv or hq // hkv > _lib.MAX_GQA:
        raise ValueError(f"GQA requires Hq divisible by Hkv, at most {_lib.MAX_GQA} query heads a KV head")
    if query.dtype != cache.key_pages.dtype or query.device != cache.key_pages.device:
        raise ValueError("paged attention query must match the cache's dtype and device")
    _lib.refuse_gradients("paged attention", query, *_pools(cache), *(output or ()))
    if batch * hkv * (-(-cache.capacity // 32)) > (1 << 31) - 4097:
        raise ValueError("paged attention takes at most 2^36 slots over all requests and heads")
    w, s = _window(window, sinks)
    scale = _scale(sm_scale)
    if append is not None or cache.weight_pages is not None:
        _check_written(cache, "paged attention with an append or weights")
    dev = query.device
    query = _token_rows(query)
    if output is None:
        out = torch.empty((batch, hq, 128), dtype=query.dtype, device=dev)
        lse = torch.empty((batch, hq), dtype=torch.float32, device=dev)
    else:
        out, lse = output
        if tuple(out.shape) != (batch, hq, 128) or out.dtype != query.dtype or out.device != dev or not out.is_contiguous() \
                or out.data_ptr() % 16:
            raise ValueError("paged attention output must be contiguous [B,Hq,128] of the query's dtype and device")
        if tuple(lse.shape) != (batch, hq) or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous():
            raise ValueError("paged attention lse output must be contiguous fp32 [B,Hq] on the query's device")
    p = _lib.PagedAttention(cache=_params_of(cache), query=query.data_ptr(), query_strides=_strides(query, 2), hq=hq, window=w,
                            sinks=s, sm_scale=scale, out=out.data_ptr(), lse=lse.data_ptr())
    if append is not None:
        rows = []
        for t in append:
            if t.ndim == 4 and t.shape[2] == 1:
                t = t[:, :, 0]
            if tuple(t.shape) != (batch, hkv, 128):
                raise ValueError("paged attention append requires key and value [B,Hkv,128]")
            rows.append(_token_rows(t))
        key, value = rows
        _check_new_rows(cache, key, value, "paged attention append")
        p.append_key, p.append_value = key.data_ptr(), value.data_ptr()
        p.append_strides = (*_strides(key, 2), *_strides(value, 2))
    p.workers = _lib.host().paged_workers(batch, hkv, cache.capacity, _lib.num_cus(dev))
    p.partial_states = (p.workers + batch * hkv) * (hq // hkv)
    p.logits_floats = batch * hq * (-(-cache.capacity // 32) * 32) if cache.weight_pages is not None else 0
    # partial outputs, (maximum, sum) pairs, logits
    scratch = torch.empty(130 * p.partial_states + 2 + p.logits_floats, dtype=torch.float32, device=dev)
    base = scratch.data_ptr()
    p.partial_out, p.partial_ml = base, base + 512 * p.partial_states
    if p.logits_floats:
        p.logits = base + (520 * p.partial_states + 15) // 16 * 16
    _lib.launch("r2o_paged_attention", p, dev)
    return out, lse


def paged_prefix_attention(query: torch.Tensor, cache: PagedCache, prefix: PagedCache | None = None, *,
                           members: torch.Tensor | None = None, query_lengths: torch.Tensor | None = None,
                           sm_scale: float | None = None, output: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Attention of each request's newest rows, query [B, Hq, S, 128] (or [B, Hq, 128] for one token), over the prefix that it
    shares and over its own slots; returns (out like query, lse fp32 [B, Hq, S] or [B, Hq]).

    ``prefix`` is a cache whose table has a row, and whose lengths have an entry, for each prefix; its pages may lie in
    ``cache``'s pools or others (of one type and head count; page sizes may differ).  ``members`` (int32 [prefixes] on the device):
    requests 0 .. members[0] - 1 share prefix 0, the next members[1] prefix 1, and so on, requests behind the last share
    none; without it all share the one prefix there is.  Counts past the batch's end are cut off.  Row i of a request with q
    query rows (S, or ``query_lengths[b]``) and n = ``cache.lengths[b]`` slots, the new ones among them, sees all of its
    prefix and its own slots j <= n - q + i.  A row that sees nothing, or lies behind its request's rows, is 0 with lse
    -inf; infinite and NaN values count as in ``prompt_attention``.  Own rows' positions are the caller's: they go on behind the
    prefix, where ``paged_rope_extend`` without ``positions`` counts from 0.  Without a prefix it is causal attention of a chunk
    over its paged cache.  Caches that keep weights are refused, for none are accumulated (``paged_evict`` would not know what
    was attended here): ``dataclasses.replace(cache, weight_pages=None)``.  ``output``: the two result tensors, the first with
    unit-strided channels and 16-byte aligned rows, neither overlapping an input."""
    if output is None:
        made = _lib.host().paged_prefix_attention(_lib.entry("r2o_paged_prefix_attention"), query, cache, prefix, members,
                                                  query_lengths, sm_scale)
        if made is not None:
            _lib.check(made[0], "r2o_paged_prefix_attention")
            return made[1], made[2]
    what = "paged prefix attention"
    batch, hkv, dev = int(cache.page_table.shape[0]), int(cache.key_pages.shape[1]), cache.key_pages.device
    token = query.ndim == 3
    if token:
        query = query[:, :, None]
        output = None if output is None else (output[0][:, :, None], output[1][..., None])
    if query.ndim != 4 or query.shape[0] != batch or query.shape[3] != 128 or min(query.shape) < 1:
        raise ValueError("paged prefix attention requires query [B,Hq,S,128] or [B,Hq,128] of the cache's requests")
    hq, rows = int(query.shape[1]), int(query.shape[2])
    if hq % hkv:
        raise ValueError("GQA requires Hq divisible by Hkv")
    if query.dtype != cache.key_pages.dtype or query.device != dev:
        raise ValueError("paged prefix attention query must match the cache's dtype and device")
    if batch * hq * rows > 1 << 30:
        raise ValueError("paged prefix attention takes at most 2^30 query rows over all heads")
    caches = (cache,) if prefix is None else (cache, prefix)
    if any(c.weight_pages is not None for c in caches):
        raise ValueError("paged prefix attention does not keep weights: pass caches without weight_pages")
    prefixes = 0
    if prefix is not None:
        prefixes = int(prefix.page_table.shape[0])
        if prefix.key_pages.shape[1] != hkv or prefix.key_pages.dtype != cache.key_pages.dtype or prefix.key_pages.device != dev:
            raise ValueError("paged prefix attention prefix must have the cache's heads, dtype and device")
        if members is None and prefixes > 1:
            raise ValueError("paged prefix attention of several prefixes needs members")
    elif members is not None:
        raise ValueError("paged prefix attention members need a prefix")
    members = _lengths(members, prefixes, dev, "members")
    query_lengths = _lengths(query_lengths, batch, dev, "query_lengths")
    _lib.refuse_gradients(what, query, *(t for c in caches for t in _pools(c)), *(output or ()))
    scale = _scale(sm_scale)
    params = [_params_of(c) for c in caches]
    workers, floats = _lib.host().prefix_plan(batch, hkv, hq, rows, cache.capacity, prefixes, prefix.capacity if prefixes else 0,
                                              query_lengths is not None, _lib.num_cus(dev))
    if not workers:
        raise ValueError("paged prefix attention has more tiles of slots than it can count")
    query = _rows(query)
    if output is None:
        out = _like(query)
        lse = torch.empty((batch, hq, rows), dtype=torch.float32, device=dev)
    else:
        out, lse = output
        _check_like(out, query, what)
        if tuple(lse.shape) != (batch, hq, rows) or lse.dtype != torch.float32 or lse.device != dev or not lse.is_contiguous():
            raise ValueError("paged prefix attention lse output must be contiguous fp32 [B,Hq,S] on Q's device")
    p = _lib.PagedPrefix(cache=params[0], members=_lib.ptr(members), query_lengths=_lib.ptr(query_lengths), query=query.data_ptr(),
                         out=out.data_ptr(), lse=lse.data_ptr(), q_strides=_strides(query, 3), o_strides=_strides(out, 3), hq=hq,
                         rows=rows, sm_scale=scale)
    if prefixes:
        p.prefix = params[1]
    scratch = torch.empty(floats, dtype=torch.float32, device=dev)
    p.workers, p.scratch_floats, p.scratch = workers, floats, scratch.data_ptr()
    _lib.launch("r2o_paged_prefix_attention", p, dev)
    return (out[:, :, 0], lse[..., 0]) if token else (out, lse)


def paged_evict(cache: PagedCache, target: PagedCache, keep: int, *, sinks: int = 0, recent: int = 0) -> torch.Tensor:
    """Copy what each (request, KV head) keeps into slots 0.. of ``target``, in order, and set ``target.lengths``.

    A request with more than ``keep`` filled slots keeps its first ``sinks``, its last ``recent`` and, of the others,
    those of largest accumulated weight (equal ones: the earlier; NaN counts as the largest); a shorter one keeps
    all.  Heads keep different tokens, all of them ``min(lengths, keep)``.  The weights go along where the target has
    ``weight_pages``.  The target may lie in the same pools, in pages that the source's table does not name; the
    source is left as it is, for its pages to be handed back.  Returns the kept source slots, int32 [B, Hkv, keep]
    in ascending order, -1 behind a request's length."""
    made = _lib.host().paged_evict(_lib.entry("r2o_paged_evict"), cache, target, keep, sinks, recent)
    if made is not None:
        _lib.check(made[0], "r2o_paged_evict")
        return made[1]
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if cache.weight_pages is None:
        raise ValueError("paged evict needs a cache with weight_pages")
    if cache.page_table.shape[0] != target.page_table.shape[0] or cache.key_pages.shape[1] != target.key_pages.shape[1]:
        raise ValueError("paged evict target must have the source's requests and heads")
    if cache.key_pages.dtype != target.key_pages.dtype or cache.key_pages.device != target.key_pages.device:
        raise ValueError("paged evict target must match the source's dtype and device")
    if abs(cache.lengths.data_ptr() - target.lengths.data_ptr()) < 4 * cache.lengths.numel() or cache.page_table.data_ptr() == target.page_table.data_ptr():
        raise ValueError("paged evict target needs a page table and lengths of its own")
    if not 1 <= keep <= target.capacity:
        raise ValueError("keep must be positive and at most what the target's page table holds")
    if sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError("sinks and recent must be non-negative and together at most keep")
    _check_written(target, "paged evict")
    _lib.refuse_gradients("paged evict", *_pools(cache), *_pools(target))
    dev = cache.key_pages.device
    kept = torch.empty((cache.page_table.shape[0], cache.key_pages.shape[1], keep), dtype=torch.int32, device=dev)
    p = _lib.PagedEvict(source=_params_of(cache), target=_params_of(target), keep=keep, sinks=sinks, recent=recent, kept=kept.data_ptr(),
                        target_lengths=target.lengths.data_ptr())
    _lib.launch("r2o_paged_evict", p, dev)
    return kept
