"""Layer norm, rotary positions and cross attention without a GPU: what their entry points refuse at the edges of what they document."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from detectorfreesfm_amd import _lib, ops


def test_operands_with_a_tangent():
    """The check behind every entry point, with gradients recorded or not; without a tangent, or outside of a dual level, tensors pass."""
    x = torch.zeros(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        for args in ((dual, (), ()), (x, (x, dual), (None,)), (x, (None,), (None, dual))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(_lib.DfsfmError, match="tangent"):
                    ops._operands("call", *args)
        assert ops._operands("call", x, (x,), (None, x)) == 0
    assert ops._operands("call", x, (x,), (None, x)) == 0


def test_lazily_negated_operands():
    """The imaginary part of a conjugate lies in memory with the other sign."""
    x = torch.ones(3)
    turned = torch.complex(torch.zeros(3), -x).conj().imag
    assert turned.is_neg() and torch.equal(turned, x)
    for args in ((turned, (), ()), (x, (x, turned), (None,)), (x, (None,), (None, turned))):
        with pytest.raises(_lib.DfsfmError, match="resolve_neg"):
            ops._operands("call", *args)
    assert ops._operands("call", turned.resolve_neg(), (x,), ()) == 0
