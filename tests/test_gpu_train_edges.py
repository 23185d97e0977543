"""Calls of layer norm, rotary positions and cross attention at the edges of what their documentation allows, on the GPU."""
import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import attention_norms as an
from detectorfreesfm_amd import _lib, ops
from test_gpu_cross_attention import TYPES, U, both, check, close, rounded
from test_gpu_train_norm import rotary_reference
from test_train_edges_cpu import NORM_CASES, filled

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_gradient_of_no_query_heads_is_zero(built_lib):
    """dk and dv are sums over the query heads: of none, zeros, whatever the allocator's memory held before."""
    for t in TYPES:
        q, k = torch.empty((2, 3, 0, 32), dtype=t, device=DEV), torch.randn((2, 5, 2, 32), device=DEV).to(t)
        out, lse = ops.cross_attention(q, k, k)
        assert out.shape == q.shape and lse.shape == (2, 0, 3)
        junk = [torch.full_like(k, math.nan) for _ in range(8)]
        del junk
        dq, dk, dv = ops.cross_attention_backward(q, q, k, k, out, lse)
        assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == k.shape
        assert bool((dk == 0).all()) and bool((dv == 0).all())


def operator_calls():
    """Every operator as a function of one tensor that it reads, and the tensor."""
    x, w = torch.randn((4, 64), device=DEV), torch.ones(64, device=DEV)
    h, k = torch.randn((2, 3, 4, 32), device=DEV), torch.randn((2, 5, 2, 32), device=DEV)
    pos, (inv, _) = torch.arange(3, device=DEV), ops.rotary_frequencies(32, device=DEV)
    _, m, r = ops.layernorm_forward(x, w, w)
    out, lse = ops.cross_attention(h, k, k)
    return [(x, lambda t: ops.layernorm_forward(t, w, w)), (w, lambda t: ops.layernorm_forward(x, t, w)), (w, lambda t: ops.layernorm_forward(x, w, t)),
            (x, lambda t: ops.layernorm_forward(x, w, w, residual=t)), (x, lambda t: ops.layernorm_backward(t, x, m, r, w)),
            (m, lambda t: ops.layernorm_backward(x, x, t, r, w)), (h, lambda t: ops.rotary(t, pos, inv)), (inv, lambda t: ops.rotary(h, pos, t)),
            (h, lambda t: ops.rotary_backward(t, pos, inv)), (h, lambda t: ops.cross_attention(t, k, k)), (k, lambda t: ops.cross_attention(h, t, k)),
            (k, lambda t: ops.cross_attention(h, k, t)), (h, lambda t: ops.cross_attention_backward(t, h, k, k, out, lse)),
            (out, lambda t: ops.cross_attention_backward(h, h, k, k, t, lse)), (lse, lambda t: ops.cross_attention_backward(h, h, k, k, out, t))]


def test_tangents_are_refused(built_lib):
    """A dual tensor of forward-mode differentiation would lose its tangent without a word."""
    for i, (x, call) in enumerate(operator_calls()):
        with forward_ad.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(_lib.DfsfmError, match="tangent"):
                    call(forward_ad.make_dual(x, torch.ones_like(x)))
            call(x)                                                         # tensors without one pass


def test_lazily_negated_tensors_are_refused(built_lib):
    """The imaginary part of a conjugate is a view of the values before their sign is turned."""
    for x, call in operator_calls():
        turned = torch.complex(torch.zeros_like(x), -x).conj().imag
        assert turned.is_neg() and torch.equal(turned, x)
        with pytest.raises(_lib.DfsfmError, match="resolve_neg"):
            call(turned)
        call(turned.resolve_neg())


@pytest.mark.parametrize("L, S, D, H", [(1, 60000, 32, 256), (1, 30000, 128, 256), (64, 30000, 64, 1800), (200, 9000, 32, 220), (200, 9000, 128, 220)])
def test_fp16_weights_far_below_the_largest(built_lib, L, S, D, H):
    """The first key holds nearly all of a row's weight and its value is 0: the result is what the many others add, each e^-16.5 to e^-18.5 of
    it (fp16 numbers end at e^-16.6, and halves of that round to 0).  A weight is off by ut of itself and, below fp16's normal numbers, by
    2^-25 of a scale on which the row's largest is 2^7 or above: 2^-32 of it.  out is divided by the sum of the same weights.  So many heads
    that their keys are not split: a split without the first key has a largest weight of its own."""
    g = torch.Generator().manual_seed(L + S)
    q, k, v = torch.zeros((1, L, 1, D)), torch.zeros((1, S, 1, D)), torch.rand((1, S, 1, D), generator=g) + 0.5
    q[..., 0] = 4.0
    k[..., 0] = -17.5 / 4 + 0.5 * (torch.rand((1, S, 1), generator=g) - 0.5)
    k[0, 0], v[0, 0] = 0.0, 0.0
    q, k, v = q.half(), k.half(), v.half()
    s = q[0, 0, 0].double() @ k[0, :, 0].double().T
    p, V = torch.exp(s), v[0, :, 0].double()
    out, total = p @ V / p.sum(), p.sum()
    e = p * (2.0 ** -11 + 40 * U * (s.abs() + 1)) + 2.0 ** -32 + (S + 8) * U * p
    bound = (e @ V + out * e.sum()) / total * (1 + 2.0 ** -8)
    got, lse = ops.cross_attention(*(x.to(DEV).expand(-1, -1, H, -1) for x in (q, k, v)), scale=1.0)
    close(got, out.expand(1, L, H, D), rounded(out, bound, torch.float16).expand(1, L, H, D), (L, S, D))
    assert float((lse.double().cpu() - torch.log(total)).abs().max()) < (S + 40) * U


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("mask", ["lens", "both"])
@pytest.mark.parametrize("shape", [(1, 1, 513, 2, 2, 64), (1, 130, 1500, 1, 1, 32), (1, 2000, 40, 1, 1, 64), (3, 1, 1896, 1, 1, 40), (1, 1, 9001, 1, 1, 64),
                                   (1, 4, 4500, 8, 1, 32), (1, 100, 257, 2, 2, 128), (1, 257, 513, 5, 1, 96), (1, 33, 64, 2, 1, 16), (1, 129, 1500, 1, 1, 128),
                                   (5, 60, 700, 2, 1, 64), (70, 1, 300, 2, 1, 32)])
def test_cross_attention_of_sequences_that_all_have_keys(built_lib, shape, mask, t):
    """Lengths and masks of few sequences, one above all, with keys in each: splits, joins and partial sums of results that are not zero."""
    q, k, v, do, lens, km, there = filled(*shape, t, mask, sum(shape) + 3)
    got = both(q, k, v, do, lens, km)
    assert all(bool((got[n] != 0).flatten(1).any(-1).all()) for n in got)
    check(got, q, k, v, do, there, shape[-1] ** -0.5, (shape, mask, t))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape, mask", NORM_CASES)
def test_cross_attention_rounds_its_results_alone(built_lib, shape, mask, t):
    """dq of masked or few keys, or of one tile of rows, and every result of up to 32 rows a head: in the 2-norm, where a second rounding of
    weights or score gradients shows (tests/attention_norms.py, and the test of it without a GPU)."""
    q, k, v, do, lens, km, there = filled(*shape, t, mask, sum(shape))
    got = both(q, k, v, do, lens, km)
    # above 512 keys delta is <dout, out> with the rounded out, which every key of a row shares
    c = an.terms(q, k, v, do, there, shape[-1] ** -0.5, out=got["out"] if shape[2] > 512 else None)
    exact, W = an.products(c, c["p"], c["ds"]), an.spreads(c)
    for n in ("out", "dq", "dk", "dv") if shape[1] * shape[3] // shape[4] <= 32 else ("dq",):
        off = float((got[n].double().cpu().permute(0, 2, 1, 3) - exact[n]).norm())
        assert off < an.allowed(exact[n], W[n], t), (n, off, an.allowed(exact[n], W[n], t))


def test_rotary_of_more_tokens_than_one_launch_holds(built_lib):
    """2^24 and three tokens of 129 pairs of odd number, a workgroup each (8.7 GB): the same bits as in parts, and the turn of their positions
    at the ends of the launches."""
    L, P = (1 << 24) + 3, 129
    x = torch.empty((1, L, 1, 2 * P), dtype=torch.float16, device=DEV).normal_()
    pos, inv = torch.arange(L, device=DEV), torch.rand(P, dtype=torch.float64, device=DEV)
    y = ops.rotary(x, pos, inv)
    step = 1 << 21
    assert all(torch.equal(y[:, i:i + step], ops.rotary(x[:, i:i + step], pos[i:i + step], inv)) for i in range(0, L, step))
    for i in (0, (1 << 24) - 6, L - 4):
        ref, bound = rotary_reference(x[:, i:i + 4].cpu(), pos[i:i + 4].cpu(), inv.cpu(), 1.0, 1, False, False)
        close(y[:, i:i + 4], ref, rounded(ref, bound, torch.float16), i)
    assert ops.rotary(x, pos, inv, inplace=True) is x and torch.equal(x, y)
