"""Layer norm, rotary positions and cross attention without a GPU: what their entry points refuse at the edges of what they document."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from detectorfreesfm_amd import _lib, ops
from test_train_ops_cpu import UNSUPPORTED, WORKSPACE, attention, attention_backward


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


def test_cross_attention_sizes_that_no_launch_holds(built_lib):
    """A launch holds less than 2^32 threads along an axis.  Sizes at that limit are refused before any launch; the largest below it get as far
    as the missing workspace."""
    L = built_lib
    one = dict(H=1, Hkv=1, nbytes=0)
    for call in (attention, attention_backward):
        # tiles of rows, tiles of keys
        assert call(L, N=64, len=(1 << 25) - 127, S=10, **one) == UNSUPPORTED
        assert call(L, N=64, len=1, S=(1 << 25) - 127, **one) == UNSUPPORTED and call(L, N=64, len=1, S=(1 << 25) - 128, **one) == WORKSPACE
    assert attention(L, N=64, len=(1 << 25) - 128, S=10, **one) == WORKSPACE
    # delta's rows; the forward pass has none
    assert attention_backward(L, N=1, len=1 << 29, S=10, **one) == UNSUPPORTED and attention(L, N=1, len=1 << 29, S=10, **one) == WORKSPACE
    assert attention_backward(L, N=1, len=(1 << 29) - 1, S=10, **one) == WORKSPACE
    assert L.dfsfm_cross_attention_workspace(64, (1 << 25) - 127, 10, 1, 1, 32, 0) == 0
    assert L.dfsfm_cross_attention_backward_workspace(1, 1 << 29, 10, 1, 1, 32, 0) == 0
