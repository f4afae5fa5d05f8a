"""Attention of a prompt's rows, and the attention weight that each of its keys received, on the gfx950 kernels.

* ``prompt_attention`` (``r2o_prompt_attention``): causal GQA attention of every row of a prompt, or of its last
  chunk over the keys so far, with an optional sliding window and sink tokens, over padded batches.
* ``attention_weights`` (``r2o_attention_weights``): the sum of each key's attention weights over query rows and
  the heads of its group, from the statistics that ``prompt_attention`` returns.  What a cache keeps is decided by
  it: ``policy.project_attention_weights_to_pages`` for the packed cache, ``paged.paged_evict`` for the paged one.

Row i of a request with q query rows and n keys stands at position p = n - q + i and sees key j where j <= p and,
with ``window=W``, p - j < W or j < sinks.  No counterpart in the reference, whose prompts run the model's own
attention (qwen_sspa_attention.py:1614) and whose scoring is torch code (policy/dual_score.py).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_MOST_ROWS = 1 << 29


def _rows(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself if the kernels can read its rows in place (unit channel stride, 16-byte aligned rows),
    otherwise a contiguous copy."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[-2] == 1 or t.stride(-2) <= 1 << 24) \
            and all(st % 8 == 0 for st, n in zip(t.stride()[:-1], t.shape) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _like(t: torch.Tensor) -> torch.Tensor:
    """An empty tensor laid out like ``t``, if the kernels can write that in place."""
    out = torch.empty_like(t)
    return out if _rows(out) is out else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _check_like(out: torch.Tensor, t: torch.Tensor, what: str, whose: str = "Q's") -> None:
    """A result tensor that a caller gave."""
    if out.shape != t.shape or out.dtype != t.dtype or out.device != t.device:
        raise ValueError(f"{what} output must match {whose} shape, dtype and device")
    if _rows(out) is not out or any(st == 0 for st, n in zip(out.stride(), out.shape) if n > 1):
        raise ValueError(f"{what} output needs unit channel stride and 16-byte aligned rows of its own")


def _strides(t: torch.Tensor, n: int):
    """Element strides of the first ``n`` axes; those of an axis of one do not matter and may be anything."""
    return (ctypes.c_int64 * n)(*[st if size > 1 else 0 for st, size in zip(t.stride()[:n], t.shape)])


def _scale(sm_scale) -> float:
    scale = 128 ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("sm_scale must be positive and finite")
    return scale


def _window(window, sinks) -> tuple[int, int]:
    """(window, sinks) as the kernels take them: a window of 0 is none, one past every length is any such."""
    if window is not None and int(window) < 1:
        raise ValueError("window must be None or at least one token")
    if int(sinks) < 0:
        raise ValueError("sinks must be non-negative")
    return (0 if window is None else min(int(window), 2 * _MOST_ROWS)), min(int(sinks), _MOST_ROWS)


def _lengths(t, batch: int, device: torch.device, what: str):
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != (batch,) or t.device != device:
        raise ValueError(f"{what} must be an int32 [B] tensor on the rows' device")
    return t.contiguous()


def _check_rows(query: torch.Tensor, key: torch.Tensor, what: str) -> None:
    if query.ndim != 4 or key.ndim != 4 or query.shape[-1] != 128 or key.shape[-1] != 128:
        raise ValueError(f"{what} requires query [B,Hq,Sq,128] and key [B,Hkv,Sk,128]")
    if query.shape[0] != key.shape[0] or min(query.shape) < 1 or min(key.shape) < 1:
        raise ValueError(f"{what} requires equal batch sizes and positive head and row counts")
    if query.shape[1] % key.shape[1]:
        raise ValueError("GQA requires Hq divisible by Hkv")
    if max(query.shape[2], key.shape[2]) > _MOST_ROWS or query.shape[0] * query.shape[1] > 65535 \
            or query.shape[1] // key.shape[1] * query.shape[2] > 1 << 30:
        raise ValueError(f"{what} takes at most 2^29 rows and 65535 (request, query head) pairs")
    if query.device != key.device or query.dtype != key.dtype:
        raise ValueError("Q/K device and dtype must match")
    _lib.dtype_code(query.dtype)
    _lib.refuse_gradients(what, query, key)


def _params(query, key, window, sinks, query_lengths, key_lengths, sm_scale) -> _lib.PromptParams:
    w, s = _window(window, sinks)
    return _lib.PromptParams(
        query=query.data_ptr(), key=key.data_ptr(), q_strides=_strides(query, 3), k_strides=_strides(key, 3),
        query_lengths=_lib.ptr(query_lengths), key_lengths=_lib.ptr(key_lengths), batch=query.shape[0], hq=query.shape[1],
        hkv=key.shape[1], queries=query.shape[2], keys=key.shape[2], dtype=_lib.dtype_code(query.dtype), window=w, sinks=s,
        sm_scale=_scale(sm_scale))


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, window: int | None = None,
                     sinks: int = 0, query_lengths: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None,
                     sm_scale: float | None = None, output: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Causal attention of query [B, Hq, Sq, 128] over key and value [B, Hkv, Sk, 128] (bf16 or fp16, query head h
    reads KV head h // (Hq // Hkv)); returns (out like query, lse fp32 [B, Hq, Sq]).

    The last query row of a request stands at its last key, so Sq < Sk is a chunk of a longer prompt.
    ``query_lengths`` / ``key_lengths`` (int32 [B] on the device): the rows of each request of a padded batch.
    With ``window``, a row sees its last ``window`` keys and the first ``sinks``.  A row that sees no key, or lies
    behind its request's length, is 0 with lse -inf; values of rows behind a length are never used.  A value that is
    infinite or NaN in a row that counts is its channel's result there, however small its weight.  Strided views
    are read in place where the channels are unit-strided and rows 16-byte aligned (copied otherwise).  ``output``:
    the two result tensors to write, the first with such strides, neither overlapping an input."""
    if output is None:
        made = _lib.host().prompt(_lib.entry("r2o_prompt_attention"), query, key, value, window, sinks, query_lengths,
                                  key_lengths, sm_scale)
        if made is not None:
            _lib.check(made[0], "r2o_prompt_attention")
            return made[1], made[2]
    _check_rows(query, key, "prompt attention")
    if value.shape != key.shape or value.device != key.device or value.dtype != key.dtype:
        raise ValueError("prompt attention value must match K's shape, device and dtype")
    _lib.refuse_gradients("prompt attention", value, *(output or ()))
    batch, hq, rows, _ = query.shape
    query_lengths = _lengths(query_lengths, batch, query.device, "query_lengths")
    key_lengths = _lengths(key_lengths, batch, query.device, "key_lengths")
    _lib.require_device(query, "prompt attention input")
    query, key, value = _rows(query), _rows(key), _rows(value)
    p = _params(query, key, window, sinks, query_lengths, key_lengths, sm_scale)
    if output is None:
        out = _like(query)
        lse = torch.empty((batch, hq, rows), dtype=torch.float32, device=query.device)
    else:
        out, lse = output
        _check_like(out, query, "prompt attention")
        if tuple(lse.shape) != (batch, hq, rows) or lse.dtype != torch.float32 or lse.device != query.device \
                or not lse.is_contiguous():
            raise ValueError("prompt attention lse output must be contiguous fp32 [B,Hq,Sq] on Q's device")
    p.splits = _lib.host().attention_splits(batch, hq, key.shape[1], rows, key.shape[2], p.window, p.sinks, _lib.num_cus(query.device))
    scratch = None
    if p.splits > 1:
        scratch = torch.empty(130 * p.splits * batch * hq * rows, dtype=torch.float32, device=query.device)
        p.scratch, p.scratch_floats = scratch.data_ptr(), scratch.numel()
    p.value, p.v_strides = value.data_ptr(), _strides(value, 3)
    p.out, p.o_strides, p.lse = out.data_ptr(), _strides(out, 3), lse.data_ptr()
    _lib.launch("r2o_prompt_attention", p, query.device)
    return out, lse


def attention_weights(query: torch.Tensor, key: torch.Tensor, lse: torch.Tensor, *, window: int | None = None,
                      sinks: int = 0, query_lengths: torch.Tensor | None = None, key_lengths: torch.Tensor | None = None,
                      sm_scale: float | None = None, output: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 [B, Hkv, Sk]: for each key, exp(sm_scale q . k - lse) summed over the rows that see it and the query
    heads of its group.

    ``query`` holds the rows that count (all of a prompt's, or the last ones of an observation window) and ``lse``
    [B, Hq, Sq] fp32 their statistics from ``prompt_attention`` with the same masks; finite rows with lse -inf give
    nothing.  Positions, lengths, masks and strides as there.  Keys behind a length get 0.  The sums are formed in
    a fixed order: equal calls give equal bits."""
    if output is None:
        made = _lib.host().weights(_lib.entry("r2o_attention_weights"), query, key, lse, window, sinks, query_lengths,
                                   key_lengths, sm_scale)
        if made is not None:
            _lib.check(made[0], "r2o_attention_weights")
            return made[1]
    _check_rows(query, key, "attention weights")
    batch, hq, rows, _ = query.shape
    if tuple(lse.shape) != (batch, hq, rows) or lse.dtype != torch.float32 or lse.device != query.device:
        raise ValueError("attention weights lse must be fp32 [B,Hq,Sq] on Q's device")
    _lib.refuse_gradients("attention weights", lse, output)
    query_lengths = _lengths(query_lengths, batch, query.device, "query_lengths")
    key_lengths = _lengths(key_lengths, batch, query.device, "key_lengths")
    _lib.require_device(query, "attention weights input")
    query, key, lse = _rows(query), _rows(key), lse.contiguous()
    hkv, keys = int(key.shape[1]), int(key.shape[2])
    if output is None:
        output = torch.empty((batch, hkv, keys), dtype=torch.float32, device=query.device)
    elif tuple(output.shape) != (batch, hkv, keys) or output.dtype != torch.float32 or output.device != query.device \
            or not output.is_contiguous():
        raise ValueError("attention weights output must be contiguous fp32 [B,Hkv,Sk] on Q's device")
    p = _params(query, key, window, sinks, query_lengths, key_lengths, sm_scale)
    p.lse_in, p.weights = lse.data_ptr(), output.data_ptr()
    p.splits = _lib.host().weight_splits(batch, hq, hkv, rows, keys, _lib.num_cus(query.device))
    scratch = None
    if p.splits > 1:
        scratch = torch.empty(p.splits * output.numel(), dtype=torch.float32, device=query.device)
        p.scratch, p.scratch_floats = scratch.data_ptr(), scratch.numel()
    _lib.launch("r2o_attention_weights", p, query.device)
    return output
