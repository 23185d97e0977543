"""Layer norm, rotary positions and cross attention without a GPU: what their entry points refuse at the edges of what they document."""
import math
import os
import re

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import attention_norms as an
from detectorfreesfm_amd import _lib, ops
from test_train_ops_cpu import UNSUPPORTED, WORKSPACE, attention, attention_backward


NORM_CASES = [((2, 300, 700, 2, 1, 32), "mask"), ((1, 129, 1500, 1, 1, 128), "both"), ((6, 200, 2048, 2, 2, 64), "lens"), ((2, 100, 3000, 2, 2, 64), "none"),
              ((3, 4, 512, 8, 8, 64), "none"), ((6, 32, 300, 1, 1, 48), "both"), ((40, 1, 4, 8, 8, 64), "lens")]


def filled(N, L, S, H, Hkv, D, t, mask, seed):
    """Inputs on the CPU of which every sequence has keys; padded places hold NaN, inf and the type's lowest value."""
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn((N, L, H, D), generator=g) for _ in range(2))
    k, v = (torch.randn((N, S, Hkv, D), generator=g) for _ in range(2))
    q, k, v, do = (x.to(t) for x in (1.5 * q, k, v, do))
    lens = km = None
    there = torch.ones((N, S), dtype=torch.bool)
    if mask in ("lens", "both"):
        lens = torch.tensor([[(2 * S + 2) // 3, S, S + 9, -(-S // 5)][i % 4] for i in range(N)], dtype=torch.int32)
        there &= torch.arange(S)[None] < lens[:, None]
    if mask in ("mask", "both"):
        km = torch.rand((N, S), generator=g) < 0.7
        if S > 130:
            km[:, 64:128] = False                                           # a whole tile
        km[:, 0] = True
        there &= km
    assert bool(there.any(-1).all())
    junk = torch.tensor([float("nan"), float("inf"), torch.finfo(t).min]).to(t)[torch.arange(S) % 3][None, :, None, None]
    k, v = (torch.where(there[..., None, None], x, junk) for x in (k, v))
    return q, k, v, do, lens, km, there


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


def waits_before_products(listing):
    """{kernel: number of waits for loads that the compiler, not inline assembly, put before a product in its basic block}, of kernels that
    fetch tiles by LDS-DMA."""
    found, name, inline, wait = {}, None, False, False
    for line in listing:
        line = line.strip()
        label = re.match(r"(_Z\w*attn_\w+):", line)
        if label:
            name, tiles, count, wait = label.group(1), False, 0, False
        if name is None:
            continue
        if line.startswith(";;#ASMSTART") or line.startswith(";;#ASMEND"):
            inline = line.startswith(";;#ASMSTART")
        elif re.match(r"\.LBB\w+:|s_c?branch", line):
            wait = False
        elif line.startswith("buffer_load") and line.endswith(" lds"):
            tiles = True
        elif line.startswith("s_waitcnt") and "vmcnt" in line:
            wait = not inline
        elif line.startswith("v_mfma") and wait:
            count, wait = count + 1, False
        elif line.startswith("s_endpgm"):
            if tiles:
                found[name] = count
            name = None
    return found


def test_waits_are_found():
    code = ["_Z3attn_a:", ";;#ASMSTART", "buffer_load_dwordx4 v1, s[0:3], 0 offen lds", ";;#ASMEND", ".LBB0_1:", "s_waitcnt vmcnt(0) lgkmcnt(1)", "v_mfma_x", "s_endpgm",
            "_Z3attn_b:", "buffer_load_dwordx4 v1, s[0:3], 0 offen lds", ";;#ASMSTART", "s_waitcnt vmcnt(0)", ";;#ASMEND", "v_mfma_x", "s_waitcnt vmcnt(0)", ".LBB1_2:",
            "v_mfma_x", "s_endpgm", "_Z3attn_c:", "s_waitcnt vmcnt(0)", "v_mfma_x", "s_endpgm"]
    assert waits_before_products(code) == {"_Z3attn_a": 1, "_Z3attn_b": 0}


def test_products_do_not_wait_for_the_next_tile(built_lib):
    """In the assembly of the build that is loaded: a tile's products run beside the next tile's fetch in every kernel and instance of cross
    attention that is not left to wait on purpose (csrc/cross_attention.hip, Few::NEXT_TOO and the settled operands of attn_dkdv_kernel)."""
    listing = os.path.join(os.path.dirname(_lib.__file__), "csrc", "build", "cross_attention.s")
    with open(listing) as f:
        found = waits_before_products(f)
    waiting = re.compile(r"attn_forward_few_kernelI(DF16[b_]Li64|fLi32)E|attn_dkdv_kernelI(fLi\d+|DF16[b_]Li32)ELb|attn_dkdv_kernelIDF16[b_]Li\d+ELb1")
    for kernel, least in (("attn_forward_kernel", 12), ("attn_forward_few_kernel", 6), ("attn_dq_kernel", 40), ("attn_dkdv_kernel", 7)):
        checked = {n: c for n, c in found.items() if kernel in n and not waiting.search(n)}
        assert len(checked) >= least and not any(checked.values()), (kernel, checked)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape, mask", NORM_CASES)
def test_norms_see_a_second_rounding(shape, mask, t):
    """The bound in the 2-norm lets the two-operand form pass and the form that rounds weights and score gradients once fail, for every result
    that is a sum over keys or rows."""
    q, k, v, do, _, _, there = filled(*shape, t, mask, sum(shape))
    c = an.terms(q, k, v, do, there, shape[-1] ** -0.5)
    exact, W = an.products(c, c["p"], c["ds"]), an.spreads(c)
    top = c["p"].amax(-1, keepdim=True)

    def operands(form):
        """out from weights relative to the row's largest, the gradients from ones relative to the row's sum, as the kernels have them."""
        return {**an.products(c, form(c["p"], t), form(c["ds"], t)), "out": an.products(c, form(c["p"] / top, t), c["ds"])["out"]}
    two, once = operands(an.two_operands), operands(an.rounded_to)
    for n, x in exact.items():
        limit = an.allowed(x, W[n], t)
        assert float((two[n].to(t).double() - x).norm()) < limit, n
        if n != "out" or shape[2] > 16:                                     # of a few weights the largest, 1, is exact
            assert float((once[n].to(t).double() - x).norm()) > limit, n


@pytest.mark.parametrize("rotated, axes, factor, trained", [(64, 1, 8.0, 4096), (128, 1, 2.0, 2048), (96, 2, 16.0, 8192)])
def test_rotary_frequencies_yarn_between_its_limits(rotated, axes, factor, trained):
    """The blend runs linearly in the pair's number from the (fractional) pair that turns 32 times over the trained length to the one that turns
    once: base^(-p / P) trained / 2 pi = 32 and 1 at p = P log(trained / (2 pi turns)) / log(base)."""
    P, base = rotated // (2 * axes), 10000.0
    first, last = (P * math.log(trained / (2 * math.pi * turns)) / math.log(base) for turns in (32.0, 1.0))
    inv, _ = ops.rotary_frequencies(rotated, base=base, axes=axes, scaling="yarn", factor=factor, trained=trained, device="cpu")
    between = 0
    for p in range(P):
        divided = min(1.0, max(0.0, (p - first) / (last - first)))          # share of the divided frequency
        between += 0.0 < divided < 1.0
        want = base ** (-p / P) * ((1.0 - divided) + divided / factor)
        assert abs(float(inv[p]) - want) < 1e-13 * want, p
    assert between >= 5
