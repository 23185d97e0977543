"""The entry points of layer norm, rotary positions and cross attention without a GPU: what they refuse before any launch, their workspaces,
the frequencies of rotary positions, and the order of a tile's chunks in LDS."""
import itertools
import math

import pytest
import torch

from detectorfreesfm_amd import _lib, ops

OK, BADARG, UNSUPPORTED, WORKSPACE = 0, -1, -2, -3
P = 1 << 20          # a pointer that nothing reads: every call below ends before a launch
F32, BF16, F16 = 0, 1, 2


def norm_forward(L, x=P, ldx=64, gamma=P, beta=P, wtype=F32, residual=None, ldr=0, y=P, mean=P, rstd=P, rows=4, C=64, dtype=F32):
    return L.dfsfm_layernorm_forward(x, ldx, gamma, beta, wtype, 1e-5, residual, ldr, y, mean, rstd, rows, C, dtype, None)


def norm_backward(L, dy=P, x=P, gamma=P, wtype=F32, dx=P, dg=P, db=P, rows=4, C=64, dtype=F32, ws=P, nbytes=1 << 30):
    return L.dfsfm_layernorm_backward(dy, C, x, C, P, P, gamma, wtype, dx, dg, db, rows, C, dtype, ws, nbytes, None)


def test_layernorm_refusals(built_lib):
    L = built_lib
    assert norm_forward(L, rows=0, x=None) == OK
    assert norm_backward(L, rows=0, dg=None, db=None, dx=None) == OK
    for kw in ({"x": None}, {"gamma": None}, {"beta": None}, {"y": None}, {"mean": None}, {"rstd": None}, {"rows": -1}, {"C": 0}, {"ldx": -1},
               {"residual": P, "ldr": -1}):
        assert norm_forward(L, **kw) == BADARG, kw
    for kw in ({"C": 16385}, {"dtype": 3}, {"dtype": -1}, {"wtype": BF16}, {"dtype": BF16, "wtype": F16}):
        assert norm_forward(L, **kw) == UNSUPPORTED, kw
    for kw in ({"dy": None}, {"x": None}, {"gamma": None}, {"dx": None}, {"dg": None}, {"db": None}, {"rows": -1}, {"C": 0}):
        assert norm_backward(L, **kw) == BADARG, kw
    for kw in ({"C": 16385}, {"dtype": 3}, {"wtype": F16}):
        assert norm_backward(L, **kw) == UNSUPPORTED, kw
    need = L.dfsfm_layernorm_backward_workspace(1000, 64, F32)
    assert norm_backward(L, rows=1000, nbytes=need - 1) == WORKSPACE and norm_backward(L, rows=1000, ws=None) == WORKSPACE
    assert L.dfsfm_layernorm_backward_workspace(0, 64, F32) == 0 and L.dfsfm_layernorm_backward_workspace(5, 16385, F32) == 0


def rotary(L, x=P, y=P + 4096, yn=640, pos=P, inv=P, pairs=16, axes=1, N=2, len=10, H=2, D=32, dtype=F32):
    return L.dfsfm_rotary(x, 640, 64, 32, y, yn, 64, 32, pos, 10, 1, 0, inv, pairs, axes, 0, 0, 1.0, N, len, H, D, dtype, None)


def test_rotary_refusals(built_lib):
    L = built_lib
    assert all(rotary(L, **kw) == OK for kw in ({"N": 0}, {"len": 0}, {"H": 0, "x": None}))
    for kw in ({"x": None}, {"y": None}, {"pos": None}, {"inv": None}, {"pairs": 0}, {"pairs": 17}, {"axes": 0}, {"axes": 2}, {"D": 0}, {"N": -1},
               {"x": P, "y": P, "yn": 641}):
        assert rotary(L, **kw) == BADARG, kw
    for kw in ({"D": 513}, {"axes": 3, "pairs": 4}, {"H": 65536}, {"len": 1 << 31}, {"dtype": 3}):
        assert rotary(L, **kw) == UNSUPPORTED, kw


def attention(L, q=P, qs=(640, 64, 32), k=P, ks=(640, 64, 32), v=P, vs=(640, 64, 32), out=P, lse=P, N=2, len=10, S=10, H=2, Hkv=2, D=32, scale=0.1,
              dtype=F32, ws=P, nbytes=1 << 40):
    return L.dfsfm_cross_attention(q, *qs, k, *ks, v, *vs, None, None, out, lse, N, len, S, H, Hkv, D, scale, dtype, ws, nbytes, None)


def attention_backward(L, dout=P, out=P, lse=P, q=P, qs=(640, 64, 32), k=P, v=P, ks=(640, 64, 32), dq=P, dk=P, dv=P, N=2, len=10, S=10, H=2, Hkv=2,
                       D=32, scale=0.1, dtype=F32, ws=P, nbytes=1 << 40):
    return L.dfsfm_cross_attention_backward(dout, *qs, q, *qs, k, *ks, v, *ks, out, *qs, lse, None, None, dq, dk, dv, N, len, S, H, Hkv, D, scale,
                                            dtype, ws, nbytes, None)


def test_cross_attention_refusals(built_lib):
    L = built_lib
    assert all(attention(L, **kw) == OK for kw in ({"N": 0}, {"len": 0}, {"H": 0}))
    assert all(attention_backward(L, **kw) == OK for kw in ({"N": 0}, {"H": 0}, {"len": 0, "S": 0}))
    for call, names in ((attention, ("q", "k", "v", "out", "lse")), (attention_backward, ("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv"))):
        for kw in [{n: None} for n in names] + [{"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": 1e-30}, {"scale": 1e30}, {"N": -1}, {"len": -1}, {"S": -1}]:
            assert call(L, **kw) == BADARG, (call, kw)
        bad = [{"D": 12}, {"D": 136, "qs": (10 ** 5, 10 ** 4, 136), "ks": (10 ** 5, 10 ** 4, 136)}, {"D": 0}, {"H": 3}, {"Hkv": 0}, {"dtype": 3},
               {"qs": (640, 24, 32)}, {"ks": (640, 1 << 23, 32)}, {"qs": (641, 64, 32)}, {"q": P + 8}, {"k": P + 4}, {"S": 1 << 30}, {"len": 1 << 30}]
        for kw in bad:
            assert call(L, **kw) == UNSUPPORTED, (call, kw)
    assert attention(L, out=P + 2) == UNSUPPORTED and attention_backward(L, dk=P + 2) == UNSUPPORTED
    need = L.dfsfm_cross_attention_workspace(1, 1, 4096, 1, 1, 32, F16)
    kw = dict(N=1, len=1, S=4096, H=1, Hkv=1, dtype=F16)
    assert need > 0 and attention(L, nbytes=need - 1, **kw) == WORKSPACE and attention(L, ws=None, **kw) == WORKSPACE
    assert attention(L, ws=P + 4, **kw) == WORKSPACE
    assert attention_backward(L, nbytes=L.dfsfm_cross_attention_backward_workspace(2, 10, 10, 2, 2, 32, F32) - 1) == WORKSPACE


def test_cross_attention_workspaces(built_lib):
    """Every size the checks let through has a workspace, without a division by an empty side; 16-bit calls that need no join need none."""
    L = built_lib
    for N, len, S, (H, Hkv), D, t in itertools.product((1, 3, 64), (0, 1, 33, 2000), (0, 1, 77, 5000), ((1, 1), (8, 2)), (8, 40, 64, 128), (F32, BF16)):
        f, b = (g(N, len, S, H, Hkv, D, t) for g in (L.dfsfm_cross_attention_workspace, L.dfsfm_cross_attention_backward_workspace))
        assert f >= 0 and b >= 4 * N * len * H and f % 4 == 0
    assert L.dfsfm_cross_attention_workspace(64, 4096, 1024, 8, 8, 64, BF16) == 0
    assert L.dfsfm_cross_attention_workspace(64, 4096, 1024, 8, 8, 64, F32) == 2 * 3 * 2 * 64 * 1024 * 8 * 64       # three bf16 planes of k and v
    assert L.dfsfm_cross_attention_workspace(1, 1, 4096, 1, 1, 12, F16) == 0
    # a few heads are split too: partials of dq (one row), and of dk and dv (one block of keys), behind delta's 16 bytes a row
    assert L.dfsfm_cross_attention_backward_workspace(3, 1, 4096, 1, 1, 40, F32) >= 16 + 8 * 3 * 40 * 4
    assert L.dfsfm_cross_attention_backward_workspace(3, 4096, 40, 1, 1, 40, BF16) >= 8 * 3 * 40 * 40 * 4 * 2


def test_ops_refuse_cpu_tensors(built_lib):
    x, w, h = torch.zeros(4, 64), torch.ones(64), torch.zeros(1, 4, 2, 32)
    pos, inv = torch.arange(4), ops.rotary_frequencies(32, device="cpu")[0]
    for call in (lambda: ops.layernorm_forward(x, w, w), lambda: ops.layernorm_backward(x, x, w[:4], w[:4], w), lambda: ops.rotary(h, pos, inv),
                 lambda: ops.rotary_backward(h, pos, inv), lambda: ops.cross_attention(h, h, h),
                 lambda: ops.cross_attention_backward(h, h, h, h, h, w)):
        with pytest.raises(_lib.DfsfmError):
            call()


def test_first_operand_by_name(built_lib):
    """The checks find the first operand where it is named, and say so where it is no tensor or is missing."""
    x, w, h = torch.zeros(4, 64), torch.ones(64), torch.zeros(1, 4, 2, 32)
    for call in (lambda: ops.layernorm_forward(x=x, gamma=w, beta=w), lambda: ops.cross_attention(k=h, v=h, q=h), lambda: ops.cross_attention(k=h, v=h),
                 lambda: ops.rotary_backward(dy=h, positions=w, inv_freq=w), lambda: ops.cross_attention(None, h, h)):
        with pytest.raises(_lib.DfsfmError, match="device tensors"):
            call()


def test_rotary_frequencies():
    inv, a = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert a == 1.0 and inv.dtype == torch.float64 and torch.allclose(inv, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert ops.rotary_frequencies(8, axes=2, device="cpu")[0].shape == (2,)
    lin, _ = ops.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin * 4, inv, rtol=1e-15)
    ntk, _ = ops.rotary_frequencies(8, base=100.0, scaling="ntk", factor=4.0, device="cpu")
    assert abs(float(ntk[0]) - 1) < 1e-15 and abs(float(ntk[-1]) * 4 - float(inv[-1])) < 1e-15
    yarn, a = ops.rotary_frequencies(64, scaling="yarn", factor=8.0, trained=4096, device="cpu")
    full, _ = ops.rotary_frequencies(64, device="cpu")
    turns = 4096 * full / (2 * math.pi)
    assert abs(a - (1 + 0.1 * math.log(8))) < 1e-15
    assert torch.equal(yarn[turns >= 32], full[turns >= 32]) and torch.allclose(yarn[turns <= 1] * 8, full[turns <= 1], rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert int(between.sum()) > 2 and bool(((yarn < full) & (yarn > full / 8))[between].all())
    assert ops.rotary_frequencies(2, scaling="ntk", factor=4.0, device="cpu")[0].tolist() == [1.0]
    for kw in ({"rotated": 7}, {"rotated": 6, "axes": 2}, {"rotated": 8, "axes": 3}, {"rotated": 0}, {"rotated": 8, "base": 0.0}, {"rotated": 8, "factor": 0.5},
               {"rotated": 8, "scaling": "other"}, {"rotated": 8, "scaling": "yarn", "factor": 2.0}):
        with pytest.raises(_lib.DfsfmError):
            ops.rotary_frequencies(device="cpu", **kw)


def order(CH, r):
    """cross_attention.hip: chunk c of row r of a tile with CH 16-byte chunks a row lies at c ^ order(r)."""
    return ((r & 3) << 2 | (r >> 2 & 3)) if CH >= 16 else ((r >> 1 & 1) << 2 | (r >> 2 & 3)) if CH == 8 else r >> 2 & 3


@pytest.mark.parametrize("CH", [4, 8, 16, 32])
def test_lds_chunk_order_has_no_conflicts(CH):
    """16 lanes that read a chunk of 16 different rows, and 16 lanes that read four rows x two chunks (half a chunk each), touch each of the 16
    bank groups (16 bytes of the 256 a cycle serves) at most as often as their bytes need; the order is linear, as the kernels use it."""
    def group(r, c):
        return (r * CH + (c ^ order(CH, r))) % 16
    for r0, c in itertools.product((0, 16), range(CH)):
        assert len({group(r0 + i, c) for i in range(16)}) == 16
    for r0, c in itertools.product(range(0, 32, 4), range(0, CH, 2)):
        assert len({group(r0 + i, c + j) for i in range(4) for j in range(2)}) == 8
    for a, b in itertools.product(range(16), range(16)):
        assert order(CH, a ^ b) == order(CH, a) ^ order(CH, b)
    assert all((c ^ order(CH, r)) < CH for r in range(16) for c in range(CH))
