"""Operands that a derivative would be lost through are refused by the calls as the host module makes them."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_paged import _cuda
from test_gradient_refusals import CALLS, CASES, call, is_output, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,operand", CASES)
def test_an_operand_that_a_derivative_goes_through_is_refused(name, operand):
    t = operands(_cuda())
    plain = t[operand]
    t[operand] = plain.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        call(name, t, is_output(name, operand))
    with torch.no_grad():
        call(name, t, is_output(name, operand))
    with forward_ad.dual_level():
        t[operand] = forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(name, t, is_output(name, operand))


@pytest.mark.parametrize("name", CALLS)
def test_plain_operands_are_taken(name):
    for outputs in (False, True):
        call(name, operands(_cuda()), outputs)
