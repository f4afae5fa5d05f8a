"""Rotation by positions and attention over shared prefixes have no derivative: each operand that one would be lost through is
refused, in reverse and forward mode; and their calls use the memory of the caches' tensors as it is then.  On the CPU, with the
launch looked at instead; test_gpu_prefix_calls.py makes the same calls through the host module."""
import copy
import dataclasses

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import r2omni_amd as ro
from test_gradient_refusals import launched  # noqa: F401

BF16, I32 = torch.bfloat16, torch.int32

ROTARY = ("inv_freq", "q_norm_weight", "k_norm_weight")
CALLS = {
    "position_rope": ("query", "key", "query_out", "key_out", *ROTARY),
    "paged_rope_extend": ("query", "key", "value", "weights", "query_out", "key_pages", "value_pages", "weight_pages", *ROTARY),
    "paged_prefix_attention": ("query", "query_out", "lse", "key_pages", "value_pages", "prefix.key_pages", "prefix.value_pages"),
}
OUTPUTS = ("query_out", "key_out", "lse")
CASES = [(name, operand) for name, operands_ in CALLS.items() for operand in operands_]


def operands(device):
    def rows(*shape):
        return torch.zeros(*shape, 128, dtype=BF16, device=device)

    def ints(*values):
        return torch.tensor(values, dtype=I32, device=device)

    t = {"query": rows(2, 4, 5), "key": rows(2, 2, 5), "value": rows(2, 2, 5), "query_out": rows(2, 4, 5), "key_out": rows(2, 2, 5),
         "lse": torch.zeros(2, 4, 5, device=device), "weights": torch.zeros(2, 2, 5, device=device),
         "positions": torch.zeros(2, 5, dtype=I32, device=device), "inv_freq": torch.zeros(64, device=device),
         "q_norm_weight": rows(), "k_norm_weight": rows(), "weight_pages": torch.zeros(12, 2, 16, device=device),
         "page_table": torch.arange(6, dtype=I32, device=device).view(2, 3), "lengths": ints(9, 9),
         "prefix.page_table": torch.arange(6, 8, dtype=I32, device=device).view(1, 2), "prefix.lengths": ints(20)}
    for prefix in ("", "prefix."):
        t |= {prefix + "key_pages": rows(12, 2, 16), prefix + "value_pages": rows(12, 2, 16)}
    return t


def caches(t, weights):
    own = ro.PagedCache(t["key_pages"], t["value_pages"], t["page_table"], t["lengths"], t["weight_pages"] if weights else None)
    return own, ro.PagedCache(t["prefix.key_pages"], t["prefix.value_pages"], t["prefix.page_table"], t["prefix.lengths"])


def call(name, t, outputs):
    """The call on the operands; with tensors for its results where one of them is looked at."""
    rotary = ro.PositionRotary(t["inv_freq"], q_norm_weight=t["q_norm_weight"], k_norm_weight=t["k_norm_weight"])
    if name == "position_rope":
        ro.qk_position_rope(t["query"], t["key"], t["positions"], rotary, output=(t["query_out"], t["key_out"]) if outputs else None)
    elif name == "paged_rope_extend":
        ro.paged_rope_extend(caches(t, True)[0], t["query"], t["key"], t["value"], rotary, weights=t["weights"],
                             output=t["query_out"] if outputs else None)
    else:
        ro.paged_prefix_attention(t["query"], *caches(t, False), output=(t["query_out"], t["lse"]) if outputs else None)


@pytest.mark.parametrize("name,operand", CASES)
def test_an_operand_that_needs_a_gradient_is_refused(name, operand, launched):  # noqa: F811
    t = operands("cpu")
    t[operand].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(name, t, operand in OUTPUTS)
    assert not launched
    with torch.no_grad():
        call(name, t, operand in OUTPUTS)
    assert launched == ["r2o_" + name]


@pytest.mark.parametrize("name,operand", CASES)
def test_an_operand_with_a_tangent_is_refused(name, operand, launched):  # noqa: F811
    t = operands("cpu")
    with forward_ad.dual_level():
        t[operand] = forward_ad.make_dual(t[operand], torch.ones_like(t[operand]))
        for context in (torch.enable_grad, torch.no_grad):
            with context(), pytest.raises(RuntimeError, match="forward-mode"):
                call(name, t, operand in OUTPUTS)
    assert not launched


@pytest.mark.parametrize("name", CALLS)
def test_other_operands_are_taken(name, launched):  # noqa: F811
    for outputs in (False, True):
        call(name, operands("cpu"), outputs)
    assert launched == ["r2o_" + name] * 2


@pytest.fixture
def params(monkeypatch):
    """Parameters of the calls that would be launched."""
    from r2omni_amd import _lib

    calls = []
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(_lib, "launch", lambda name, p, device: calls.append(p))
    monkeypatch.setattr(_lib, "num_cus", lambda device: 256)
    return calls


def _uses(c, cache):
    for name in ("key_pages", "value_pages", "page_table", "lengths"):
        assert getattr(c, name) == getattr(cache, name).data_ptr(), name
    assert c.pages == cache.key_pages.shape[0] and c.max_pages == cache.page_table.shape[1] and c.batch == cache.page_table.shape[0]


def test_calls_use_the_caches_tensors_as_they_are_then(params):
    """After pages move to another pool, after a copy, and with other lengths in place of the old ones."""
    t = operands("cpu")
    own, shared = caches(t, False)
    rotary = ro.PositionRotary(t["inv_freq"])
    for change in (lambda c: c, copy.copy, copy.deepcopy, dataclasses.replace):
        own, shared = change(own), change(shared)
        for c in (own, shared):
            for name in ("key_pages", "value_pages", "page_table", "lengths"):
                getattr(c, name).data = getattr(c, name).clone()
        del params[:]
        ro.paged_prefix_attention(t["query"], own, shared)
        ro.paged_rope_extend(own, t["query"], t["key"], t["value"], rotary)
        _uses(params[0].cache, own)
        _uses(params[0].prefix, shared)
        _uses(params[1].cache, own)
    ro.paged_prefix_attention(t["query"], own)
    assert params[-1].prefix.batch == 0


def test_strides_of_operands_reach_the_kernels(params):
    t = operands("cpu")
    fused = torch.zeros(2, 5, 8, 128, dtype=BF16).transpose(1, 2)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    positions = torch.zeros(5, 2, 3, dtype=torch.int64).permute(2, 1, 0)
    rotary = ro.PositionRotary(t["inv_freq"].double(), (16, 24, 24), scaling=0.5, eps=1e-3)
    own, shared = caches(t, False)
    ro.qk_position_rope(q, k, positions, rotary, apply_hadamard=True)
    ro.paged_rope_extend(own, q, k, v, rotary, positions=positions)
    ro.paged_prefix_attention(q, own, shared, sm_scale=0.25)
    rope, extend, attention = params
    for p in (rope, extend):
        assert tuple(p.q_strides) == tuple(p.k_strides) == (5 * 8 * 128, 128, 8 * 128)
        assert p.query == q.data_ptr() and p.key == k.data_ptr()
        assert tuple(p.rotation.position_strides) == (1, 3, 6) and p.rotation.position_bytes == 8 and p.rotation.freq_bytes == 8
        assert p.rotation.axes == 3 and p.rotation.pairs_1 == (1 << 40) - (1 << 16) and p.rotation.pairs_2 == (1 << 64) - (1 << 40)
        assert p.rotation.scaling == 0.5 and abs(p.rotation.eps - 1e-3) < 1e-9
    assert rope.hadamard == 1 and extend.value == v.data_ptr() and tuple(extend.v_strides) == (5 * 8 * 128, 128, 8 * 128)
    assert tuple(attention.q_strides) == (5 * 8 * 128, 128, 8 * 128) and attention.sm_scale == 0.25 and attention.query == q.data_ptr()
