"""The prompt and paged operators have no derivative: each operand that one would be lost through is refused, by every
call, in reverse and forward mode.  On the CPU, with the launch looked at instead; test_gpu_gradient_refusals.py makes
the same calls through the host module."""
import dataclasses

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import r2omni_amd as ro
from r2omni_amd import _lib

BF16, I32 = torch.bfloat16, torch.int32

CALLS = {
    "prompt_attention": ("query", "key", "value", "out", "lse"),
    "attention_weights": ("query", "key", "lse", "weights_out"),
    "paged_extend": ("key", "value", "weights", "key_pages", "value_pages", "weight_pages"),
    "paged_attention": ("token", "new_key", "new_value", "token_out", "token_lse", "key_pages", "value_pages", "weight_pages"),
    "paged_evict": ("key_pages", "value_pages", "weight_pages", "target.key_pages", "target.value_pages", "target.weight_pages"),
}


def operands(device):
    def rows(*shape):
        return torch.zeros(*shape, 128, dtype=BF16, device=device)

    t = {"query": rows(2, 4, 5), "key": rows(2, 2, 5), "value": rows(2, 2, 5), "out": rows(2, 4, 5),
         "lse": torch.zeros(2, 4, 5, device=device), "weights": torch.zeros(2, 2, 5, device=device),
         "weights_out": torch.zeros(2, 2, 5, device=device), "token": rows(2, 4), "new_key": rows(2, 2), "new_value": rows(2, 2),
         "token_out": rows(2, 4), "token_lse": torch.zeros(2, 4, device=device)}
    for prefix, first in (("", 0), ("target.", 6)):
        t |= {prefix + "key_pages": rows(12, 2, 16), prefix + "value_pages": rows(12, 2, 16),
              prefix + "weight_pages": torch.zeros(12, 2, 16, device=device),
              prefix + "page_table": torch.arange(first, first + 6, dtype=I32, device=device).view(2, 3),
              prefix + "lengths": torch.full((2,), 9, dtype=I32, device=device)}
    return t


def call(name, t, outputs):
    """The call on the operands; with tensors for its results where one of them is looked at."""
    def cache(prefix=""):
        return ro.PagedCache(*(t[prefix + f.name] for f in dataclasses.fields(ro.PagedCache)))

    if name == "prompt_attention":
        ro.prompt_attention(t["query"], t["key"], t["value"], output=(t["out"], t["lse"]) if outputs else None)
    elif name == "attention_weights":
        ro.attention_weights(t["query"], t["key"], t["lse"], output=t["weights_out"] if outputs else None)
    elif name == "paged_extend":
        ro.paged_extend(cache(), t["key"], t["value"], weights=t["weights"])
    elif name == "paged_attention":
        ro.paged_attention(t["token"], cache(), append=(t["new_key"], t["new_value"]),
                           output=(t["token_out"], t["token_lse"]) if outputs else None)
    else:
        ro.paged_evict(cache(), cache("target."), 8)


def is_output(name, operand):
    return operand in ("out", "weights_out", "token_out", "token_lse") or (name, operand) == ("prompt_attention", "lse")


CASES = [(name, operand) for name, operands_ in CALLS.items() for operand in operands_]


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(_lib, "launch", lambda name, params, device: calls.append(name))
    monkeypatch.setattr(_lib, "num_cus", lambda device: 256)
    return calls


@pytest.mark.parametrize("name,operand", CASES)
def test_an_operand_that_needs_a_gradient_is_refused(name, operand, launched):
    t = operands("cpu")
    t[operand].requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(name, t, is_output(name, operand))
    assert not launched
    with torch.no_grad():
        call(name, t, is_output(name, operand))
    assert launched == ["r2o_" + name]


@pytest.mark.parametrize("name,operand", CASES)
def test_an_operand_with_a_tangent_is_refused(name, operand, launched):
    t = operands("cpu")
    with forward_ad.dual_level():
        t[operand] = forward_ad.make_dual(t[operand], torch.ones_like(t[operand]))
        for context in (torch.enable_grad, torch.no_grad):
            with context(), pytest.raises(RuntimeError, match="forward-mode"):
                call(name, t, is_output(name, operand))
    assert not launched


@pytest.mark.parametrize("name", CALLS)
def test_other_operands_are_taken(name, launched):
    for outputs in (False, True):
        call(name, operands("cpu"), outputs)
    assert launched == ["r2o_" + name] * 2
