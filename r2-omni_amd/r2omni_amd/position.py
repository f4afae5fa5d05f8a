"""Queries and keys rotated by their positions, on the gfx950 kernels.

* ``qk_position_rope`` (``r2o_position_rope``): rotary embedding from integer positions on one to three axes (time, height
  and width of a video's or an image's patches, all in step for text) and the model's inverse frequencies.
* ``paged_rope_extend`` (``r2o_paged_rope_extend``): the same, the keys written with their values straight into their
  slots of a paged cache.

``rope.qwen_qk_mrope`` and ``rope.qwen3_qk_norm_rope`` take cos and sin tables that the model has rounded, for parity with
the reference's decode step; here the angles are formed in 64 bits from the positions (a position of 2^31 leaves a turn
exact to 2^-23), there is no table to make, and every row is rounded once.  No counterpart in the reference, whose rotary
tables are the model's (qwen_sspa_attention.py:1228-1247).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from .paged import PagedCache, _check_new_rows, _check_written, _params_of, _pools, _row_weights
from .prompt import _check_like, _lengths, _like, _rows, _strides

_PAIRS = 64
_POSITION_BYTES = {torch.int32: 4, torch.int64: 8}
_FREQ_BYTES = {torch.float32: 4, torch.float64: 8}
_MOST_TOKENS = (1 << 28) - 16  # of all requests: what one launch has lanes for


@dataclass(frozen=True, eq=False)
class PositionRotary:
    """How a model rotates its queries and keys.

    Channel pair (i, i + 64) turns by ``inv_freq[i]`` (fp32 or fp64 [64], the model's buffer) times the position on its axis.
    ``mrope_section``: how many pairs each of one to three axes has, one behind the other, or with ``interleaved`` in turn
    along the pairs (axes 1 and 2 have pair i where i % 3 is the axis and i < 3 * section; axis 0 the rest).  ``scaling``
    multiplies cosine and sine.  With ``q_norm_weight`` and ``k_norm_weight`` ([128], the rows' type) a row is divided by
    the root of its mean square + ``eps`` and multiplied by its weights first."""

    inv_freq: torch.Tensor
    mrope_section: tuple[int, ...] = (64,)
    interleaved: bool = False
    scaling: float = 1.0
    q_norm_weight: torch.Tensor | None = None
    k_norm_weight: torch.Tensor | None = None
    eps: float = 1e-6

    def axis_pairs(self) -> tuple[int, int, int]:
        """Bit i of entry a: pair i has axis a."""
        sections = tuple(int(n) for n in self.mrope_section)
        if not 1 <= len(sections) <= 3 or sum(sections) != _PAIRS or min(sections) < 0:
            raise ValueError("mrope_section must hold one to three counts of channel pairs that sum to 64")
        masks, first = [0, 0, 0], 0
        for axis, n in enumerate(sections):
            if not self.interleaved:
                masks[axis] = (1 << first + n) - (1 << first)
                first += n
            elif axis:
                masks[axis] = sum(1 << i for i in range(axis, min(3 * n, _PAIRS), 3))
        if self.interleaved:
            masks[0] = (1 << _PAIRS) - 1 - masks[1] - masks[2]
            if tuple(bin(m).count("1") for m in masks[: len(sections)]) != sections:
                raise ValueError("interleaved mrope_section does not fit 64 pairs in turns of three")
        return tuple(masks)


def _rotation(rotary: PositionRotary, positions: torch.Tensor | None, dtype: torch.dtype, device: torch.device, batch: int,
              tokens: int, what: str) -> tuple[_lib.Rotation, tuple]:
    """The launch's rotation, checked, and tensors that have to outlive the launch."""
    freq, sections = rotary.inv_freq, tuple(rotary.mrope_section)
    pairs = rotary.axis_pairs()
    if tuple(freq.shape) != (_PAIRS,) or freq.dtype not in _FREQ_BYTES or freq.device != device:
        raise ValueError(f"{what} inv_freq must be an fp32 or fp64 [64] tensor on the rows' device")
    weights = (rotary.q_norm_weight, rotary.k_norm_weight)
    if (weights[0] is None) != (weights[1] is None):
        raise ValueError(f"{what} takes both norm weights or neither")
    for w in weights:
        if w is not None and (tuple(w.shape) != (128,) or w.dtype != dtype or w.device != device):
            raise ValueError(f"{what} norm weights must be [128] tensors of the rows' dtype and device")
    eps, scaling = float(rotary.eps), float(rotary.scaling)
    if not 0.0 <= eps < math.inf or not math.isfinite(scaling):
        raise ValueError(f"{what} eps must be non-negative, and eps and scaling finite")
    _lib.refuse_gradients(what, freq, *weights)
    freq = freq.contiguous()
    # the kernels read norm weights by 16 bytes
    weights = tuple(w if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0) else w.clone(memory_format=torch.contiguous_format)
                    for w in weights)
    r = _lib.Rotation(axes=len(sections), inv_freq=freq.data_ptr(), freq_bytes=_FREQ_BYTES[freq.dtype], pairs_1=pairs[1], pairs_2=pairs[2],
                      q_weight=_lib.ptr(weights[0]), k_weight=_lib.ptr(weights[1]), eps=eps, scaling=scaling)
    if positions is not None:
        if positions.dtype not in _POSITION_BYTES or positions.device != device:
            raise ValueError(f"{what} positions must be an int32 or int64 tensor on the rows' device")
        if positions.ndim == 2 and len(sections) == 1:
            positions = positions[None]
        if tuple(positions.shape) != (len(sections), batch, tokens):
            raise ValueError(f"{what} positions must be [axes,B,S] of mrope_section's axes and the rows (or [B,S] for one axis)")
        r.positions, r.position_bytes = positions.data_ptr(), _POSITION_BYTES[positions.dtype]
        r.position_strides = _strides(positions, 3)
    return r, (freq, positions, *weights)


def _check_heads(query: torch.Tensor, key: torch.Tensor, what: str) -> None:
    if query.ndim != 4 or key.ndim != 4 or query.shape[-1] != 128 or key.shape[-1] != 128:
        raise ValueError(f"{what} requires query [B,Hq,S,128] and key [B,Hkv,S,128]")
    if query.shape[0] != key.shape[0] or query.shape[2] != key.shape[2] or min(query.shape) < 1 or key.shape[1] < 1:
        raise ValueError(f"{what} requires equal batch sizes and token counts, and positive head and token counts")
    if query.device != key.device or query.dtype != key.dtype:
        raise ValueError("Q/K device and dtype must match")
    if query.shape[0] * query.shape[2] > _MOST_TOKENS:
        raise ValueError(f"{what} takes at most 2^28 - 16 tokens over all requests")
    _lib.dtype_code(query.dtype)


def qk_position_rope(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, rotary: PositionRotary, *,
                     apply_hadamard: bool = False, output: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Query [B, Hq, S, 128] and key [B, Hkv, S, 128] (bf16 or fp16) rotated by ``positions`` (int32 or int64 [axes, B, S], or
    [B, S] for one axis) as ``rotary`` says, in one launch (of at most 2^28 - 16 tokens over all requests); returns (query,
    key).

    With ``apply_hadamard``, followed by the orthonormal FWHT-128 of both, as the packed cache's keys are.  Strided views
    are read in place where the channels are unit-strided and rows 16-byte aligned (copied otherwise): those of a fused
    projection serve.  ``output``: the two result tensors, with such strides; each may be its operand, rotated in place, and
    may overlap no other."""
    if output is None:
        made = _lib.host().position_rope(_lib.entry("r2o_position_rope"), query, key, positions, rotary, apply_hadamard)
        if made is not None:
            _lib.check(made[0], "r2o_position_rope")
            return made[1], made[2]
    what = "position rope"
    _check_heads(query, key, what)
    if positions is None:
        raise ValueError("position rope requires positions")
    batch, hq, tokens, _ = query.shape
    _lib.refuse_gradients(what, query, key, *(output or ()))
    rotation, held = _rotation(rotary, positions, query.dtype, query.device, batch, tokens, what)
    _lib.require_device(query, "position rope input")
    if output is None:
        outputs = _like(query), _like(key)
    else:
        outputs = output[0], output[1]
        _check_like(outputs[0], query, what)
        _check_like(outputs[1], key, what, "K's")
    query, key = _rows(query), _rows(key)
    p = _lib.PositionRope(rotation=rotation, query=query.data_ptr(), key=key.data_ptr(), query_out=outputs[0].data_ptr(),
                          key_out=outputs[1].data_ptr(), q_strides=_strides(query, 3), k_strides=_strides(key, 3),
                          qo_strides=_strides(outputs[0], 3), ko_strides=_strides(outputs[1], 3), batch=batch, hq=hq,
                          hkv=key.shape[1], tokens=tokens, dtype=_lib.dtype_code(query.dtype), hadamard=int(bool(apply_hadamard)))
    _lib.launch("r2o_position_rope", p, query.device)
    del held
    return outputs


def paged_rope_extend(cache: PagedCache, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, rotary: PositionRotary, *,
                      positions: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                      weights: torch.Tensor | None = None, output: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_extend`` of key and value [B, Hkv, S, 128], the keys rotated as ``rotary`` says on the way, and query [B, Hq,
    S, 128] rotated; returns the rotated query.

    Positions as in ``qk_position_rope``; without them a row's position is its slot in ``cache``, on every axis, which is right
    where the cache holds all of a request's tokens.  Behind a shared prefix it is not: the rows' positions go on where the
    prefix ends (its length + the slot, for text), and have to be given.  ``cache.lengths``, ``counts`` and ``weights`` as in
    ``paged_extend``.  Query rows behind a request's count are 0 in the result.  ``output``: the result tensor; it may be the
    query, rotated in place.  ``paged_attention`` (without ``append``) and, with such positions, ``paged_prefix_attention``
    take the result with the same cache."""
    if output is None:
        made = _lib.host().paged_rope_extend(_lib.entry("r2o_paged_rope_extend"), cache, query, key, value, rotary, positions, counts, weights)
        if made is not None:
            _lib.check(made[0], "r2o_paged_rope_extend")
            return made[1]
    what = "paged rope extend"
    _check_heads(query, key, what)
    batch, hkv, rows = int(cache.page_table.shape[0]), int(cache.key_pages.shape[1]), int(key.shape[2])
    if key.shape[0] != batch or key.shape[1] != hkv:
        raise ValueError("paged rope extend requires key and value [B,Hkv,S,128] of the cache's requests and heads")
    _check_new_rows(cache, key, value, what)
    _check_written(cache, what)
    if rows > cache.capacity:
        raise ValueError("paged rope extend has more rows than the page table holds")
    counts = _lengths(counts, batch, key.device, "counts")
    weights = _row_weights(cache, key, weights, what)
    _lib.refuse_gradients(what, query, weights, output, *_pools(cache))
    rotation, held = _rotation(rotary, positions, key.dtype, key.device, batch, rows, what)
    if output is None:
        output = _like(query)
    else:
        _check_like(output, query, what)
    query, key, value = _rows(query), _rows(key), _rows(value)
    p = _lib.PagedRopeExtend(cache=_params_of(cache), rotation=rotation, query=query.data_ptr(), key=key.data_ptr(),
                             value=value.data_ptr(), query_out=output.data_ptr(), weights=_lib.ptr(weights), counts=_lib.ptr(counts),
                             q_strides=_strides(query, 3), k_strides=_strides(key, 3), v_strides=_strides(value, 3),
                             qo_strides=_strides(output, 3), weights_strides=(0, 0) if weights is None else _strides(weights, 2),
                             hq=query.shape[1], rows=rows)
    _lib.launch("r2o_paged_rope_extend", p, key.device)
    del held
    return output
