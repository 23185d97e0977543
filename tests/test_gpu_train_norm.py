"""Layer norm with its gradient and rotary positions on the GPU (csrc/norm_train.hip, csrc/rotary.hip) against their formulas in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32; ``rounded`` adds half a step of the output type.  A 32-bit sum of n terms added along a tree or
chain of depth d is off by at most d * u * sum|terms|; the kernels' rows are summed at depth <= 16 (a lane) + 6 (a wave) + 16 (waves) < 40.
"""
import itertools

import pytest
import torch

from detectorfreesfm_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rounded(ref, bound, t):
    """bound + half a step of the output type at a value of up to |ref| + bound: eps / 2 of it, and below the smallest normal number half of
    the subnormals' spacing eps * smallest_normal (fp16: 2^-10 * 2^-14 / 2 = 2^-25; dgamma of one row is a product of any size)."""
    f = torch.finfo(t)
    return bound + torch.clamp(f.eps / 2 * (ref.abs() + bound), min=f.eps * f.smallest_normal / 2)


def close(got, ref, bound, what):
    off = (got.double().cpu() - ref.cpu()).abs()
    bad = off > bound.cpu()
    assert not bool(bad.any()), (what, off[bad].max().item(), bound.cpu()[bad].min().item(), int(bad.sum()))


def norm_case(rows, C, t, wt, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, C), generator=g) * 1.5 + 0.3).to(t)
    gamma, beta = (1 + 0.3 * torch.randn(C, generator=g)).to(wt), (0.3 * torch.randn(C, generator=g)).to(wt)
    res, dy = torch.randn((rows, C), generator=g).to(t), torch.randn((rows, C), generator=g).to(t)
    return x, gamma, beta, res, dy


def check_norm(x, gamma, beta, res, dy, eps=1e-5):
    """Forward and gradient of device copies against 64 bits; every quantity's bound follows its formula term by term."""
    t, wt = x.dtype, gamma.dtype
    rows, C = x.shape
    X, G, B, DY = x.double(), gamma.double(), beta.double(), dy.double()
    m = X.mean(-1, keepdim=True)
    var = ((X - m) ** 2).mean(-1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    h = (X - m) * r
    y = h * G + B + (0 if res is None else res.double())
    gy, gm, gr = ops.layernorm_forward(x.to(DEV), gamma.to(DEV), beta.to(DEV), eps=eps, residual=None if res is None else res.to(DEV))
    mb = 42 * U * X.abs().mean(-1, keepdim=True)                     # error of the mean (the sum, its scale)
    # the centred values are off by e = mb + u|x - m|; their squares' mean by 2 e sqrt(var) + e^2 + 42 u var, r by half of that relative
    e = mb + U * (X - m).abs()
    eb = e.max(-1, keepdim=True)[0]
    rb = r * (0.5 * (2 * eb * var.sqrt() + eb * eb + 42 * U * var) / (var + eps) + 4 * U)
    hb = e * r + (X - m).abs() * rb + 2 * U * h.abs()
    close(gm, m[:, 0], mb[:, 0], "mean")
    close(gr, r[:, 0], rb[:, 0], "rstd")
    yb = hb * G.abs() + 4 * U * ((h * G).abs() + B.abs() + (0 if res is None else res.double().abs()))
    close(gy, y, rounded(y, yb, t), "y")
    gdx, gdg, gdb = ops.layernorm_backward(dy.to(DEV), x.to(DEV), gm, gr, gamma.to(DEV))
    w = DY * G
    c1, c2 = w.mean(-1, keepdim=True), (w * h).mean(-1, keepdim=True)
    dx = r * (w - c1 - h * c2)
    c1b = 43 * U * w.abs().mean(-1, keepdim=True)
    c2b = 44 * U * (w * h).abs().mean(-1, keepdim=True) + (w.abs() * hb).mean(-1, keepdim=True)
    dxb = r * (2 * U * w.abs() + c1b + h.abs() * c2b + hb * c2.abs() + 4 * U * (w.abs() + c1.abs() + (h * c2).abs())) + dx.abs() * rb / r
    close(gdx, dx, rounded(dx, dxb, t), "dx")
    depth = rows + 40                                                # a chain over all rows is the worst order there is
    dg, db = (DY * h).sum(0), DY.sum(0)
    dgb = depth * U * (DY * h).abs().sum(0) + (DY.abs() * hb).sum(0)
    dbb = depth * U * DY.abs().sum(0)
    close(gdg, dg, rounded(dg, dgb, wt), "dgamma")
    close(gdb, db, rounded(db, dbb, wt), "dbeta")
    assert gy.dtype == t and gdx.dtype == t and gdg.dtype == wt and gdb.dtype == wt


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("C", [1, 2, 7, 8, 9, 31, 64, 100, 128, 129, 255, 256, 257, 511, 512, 513, 769, 1000, 1024, 1025, 2047, 2048, 2050, 4096,
                               4100, 8191, 8192, 16384])
def test_layernorm_widths(built_lib, C, t):
    for rows, wt, with_res in ((1, t, False), (5, torch.float32, True), (37, t, True)):
        x, gamma, beta, res, dy = norm_case(rows, C, t, wt, C + rows)
        if C == 1:
            beta = beta * 0 + 0.5
        check_norm(x, gamma, beta, res if with_res else None, dy)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,C", [(9000, 128), (4097, 100), (2500, 769), (700, 4096), (130, 9001), (20001, 16)])
def test_layernorm_many_rows(built_lib, rows, C, t):
    check_norm(*norm_case(rows, C, t, t, rows))


def test_layernorm_views(built_lib):
    """Column slices, broadcast rows, permuted leading dims, an odd byte offset, a 1-D row."""
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((6, 10, 301), generator=g).to(torch.bfloat16).to(DEV)
    gamma, beta = torch.randn(77, generator=g).to(DEV), torch.randn(77, generator=g).to(DEV)
    views = [wide[..., 3:80], wide[:, 2:5, 101:178], wide.transpose(0, 1)[..., 1:78], wide[:1, :1, :77].expand(6, 10, 77), wide[0, 0, 5:82],
             wide[:, :, ::3][..., :77]]
    for v in views:
        dense = v.clone(memory_format=torch.contiguous_format)
        a, b = ops.layernorm_forward(v, gamma, beta, residual=v), ops.layernorm_forward(dense, gamma, beta, residual=dense)
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[0].shape == v.shape and a[1].shape == v.shape[:-1]
        p, q = ops.layernorm_backward(v, v, a[1], a[2], gamma), ops.layernorm_backward(dense, dense, b[1], b[2], gamma)
        assert all(torch.equal(s, t) for s, t in zip(p, q))


def test_layernorm_empty_and_weights(built_lib):
    x = torch.empty((0, 64), device=DEV)
    gamma = torch.ones(64, device=DEV)
    y, m, r = ops.layernorm_forward(x, gamma, gamma)
    assert y.shape == (0, 64) and m.shape == (0,)
    dx, dg, db = ops.layernorm_backward(x, x, m, r, gamma)
    assert dx.shape == (0, 64) and float(dg.abs().sum()) == 0 and float(db.abs().sum()) == 0
    x = torch.randn((300, 64), device=DEV)
    y, m, r = ops.layernorm_forward(x, gamma, gamma)
    dx, dg, db = ops.layernorm_backward(x, x, m, r, gamma, need_weights=False)
    assert dg is None and db is None and torch.equal(dx, ops.layernorm_backward(x, x, m, r, gamma)[0])


def test_layernorm_differences(built_lib):
    """dx, dgamma, dbeta against central differences of the forward pass in 64 bits, and the kernels' dx against them."""
    g = torch.Generator().manual_seed(3)
    x, gamma, beta, _, dy = (t.double() for t in norm_case(4, 24, torch.float32, torch.float32, 3))

    def loss(x, gamma, beta):
        m = x.mean(-1, keepdim=True)
        return (((x - m) / (((x - m) ** 2).mean(-1, keepdim=True) + 1e-5).sqrt() * gamma + beta) * dy).sum()

    f32 = [t.float().to(DEV) for t in (x, gamma, beta, dy)]
    _, m, r = ops.layernorm_forward(*f32[:3])
    got = ops.layernorm_backward(f32[3], f32[0], m, r, f32[1])
    step = 1e-6
    for i, v in enumerate((x, gamma, beta)):
        for _ in range(12):
            at = tuple(int(torch.randint(0, s, (1,), generator=g)) for s in v.shape)
            args = [[t.clone() for t in (x, gamma, beta)] for _ in range(2)]
            args[0][i][at] += step
            args[1][i][at] -= step
            d = (loss(*args[0]) - loss(*args[1])) / (2 * step)
            assert abs(float(got[i][at]) - float(d)) < 2e-5          # 32-bit sums of ~24 terms of size 1; differences are off by 1e-9


def test_layernorm_same_bits_and_streams(built_lib):
    x, gamma, beta, res, dy = (t.to(DEV) for t in norm_case(5000, 200, torch.bfloat16, torch.bfloat16, 9))
    y, m, r = ops.layernorm_forward(x, gamma, beta, residual=res)
    ref = ops.layernorm_backward(dy, x, m, r, gamma)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            y2, m2, r2 = ops.layernorm_forward(x, gamma, beta, residual=res)
            outs.append((y2, *ops.layernorm_backward(dy, x, m2, r2, gamma)))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, (y, *ref)))


def test_layernorm_graph(built_lib):
    """Forward and gradient captured, replayed on changed inputs between eager calls."""
    x, gamma, beta, res, dy = (t.to(DEV) for t in norm_case(3000, 256, torch.float32, torch.float32, 4))

    def step():
        y, m, r = ops.layernorm_forward(x, gamma, beta, residual=res)
        return (y, *ops.layernorm_backward(dy, x, m, r, gamma))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        x.mul_(1.25).add_(0.1 * k)
        dy.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


# ---------------------------------------------------------------- rotary
def rotary_reference(x, pos, inv, amplitude, axes, interleaved, backward):
    """64-bit result and its bound before the output's rounding: cos and sin off by 2^-22 (the fraction of a turn in 32 bits: pi * 2^-25 *
    2, two ulp of sincospi, the factor), three roundings of the products and their sum."""
    N, L, H, D = x.shape
    P = inv.numel()
    pos = pos.expand((N, L) if axes == 1 else (N, L, axes))
    out, bound = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    for a in range(axes):
        angle = (pos if axes == 1 else pos[..., a]).double()[:, :, None, None] * inv
        c, s = amplitude * angle.cos(), amplitude * angle.sin() * (-1 if backward else 1)
        lo = 2 * P * a
        i, j = (slice(lo, lo + 2 * P, 2), slice(lo + 1, lo + 2 * P, 2)) if interleaved else (slice(lo, lo + P), slice(lo + P, lo + 2 * P))
        u, v = x[..., i].double(), x[..., j].double()
        out[..., i], out[..., j] = u * c - v * s, v * c + u * s
        bound[..., i] = bound[..., j] = (2.0 ** -22 + 3 * U) * amplitude * (u.abs() + v.abs())
    return out, bound


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_shapes(built_lib, t, interleaved):
    g = torch.Generator().manual_seed(5)
    for (N, L, H, D), (axes, P), far, scaling in itertools.product(
            [(1, 1, 1, 16), (3, 5, 2, 40), (2, 33, 5, 64), (1, 7, 3, 130), (2, 300, 8, 128)], [(1, 8), (1, 3), (2, 4), (2, 1), (1, 5)],
            [0, 10 ** 6, -40000], ["none", "yarn"]):
        if 2 * axes * P > D:
            continue
        x = torch.randn((N, L, H, D), generator=g).to(t)
        pos = torch.randint(-50, 5000, (N, L) if axes == 1 else (N, L, 2), generator=g) + far
        inv, amp = ops.rotary_frequencies(2 * axes * P, axes=axes, scaling=scaling, factor=4.0, trained=1024, device="cpu")
        for backward in (False, True):
            call = ops.rotary_backward if backward else ops.rotary
            got = call(x.to(DEV), pos.to(DEV), inv.to(DEV), amplitude=amp, axes=axes, interleaved=interleaved)
            ref, bound = rotary_reference(x, pos, inv, amp, axes, interleaved, backward)
            close(got, ref, rounded(ref, bound, t), ("rotary", (N, L, H, D), axes, P, far, backward))
            assert torch.equal(got[..., 2 * axes * P:].cpu(), x[..., 2 * axes * P:])


@pytest.mark.parametrize("D,P,axes", [(512, 128, 2), (512, 255, 1), (512, 256, 1), (256, 127, 1), (96, 24, 2), (2, 1, 1)])
def test_rotary_wide(built_lib, D, P, axes):
    g = torch.Generator().manual_seed(D + P)
    inv = torch.rand(P, generator=g, dtype=torch.float64) * 2
    for t, il in itertools.product(TYPES, (False, True)):
        x = torch.randn((2, 9, 3, D), generator=g).to(t)
        pos = torch.randint(0, 100000, (9,) if axes == 1 else (9, 2), generator=g).to(torch.int32)
        got = ops.rotary(x.to(DEV), pos.to(DEV), inv.to(DEV), axes=axes, interleaved=il)
        ref, bound = rotary_reference(x, pos.long(), inv, 1.0, axes, il, False)
        close(got, ref, rounded(ref, bound, t), ("rotary", D, P, axes, t, il))


def test_rotary_inplace_and_views(built_lib):
    """q | k columns of a fused projection turned in place: the columns beside them stay; strided reads equal dense ones; positions
    broadcast over the batch; the gradient of the turn is its inverse."""
    g = torch.Generator().manual_seed(8)
    fused = torch.randn((2, 50, 3 * 4 * 32), generator=g).to(DEV)
    pos = torch.arange(50, device=DEV)
    inv, _ = ops.rotary_frequencies(24, device=DEV)
    view = fused[..., :256].view(2, 50, 8, 32)
    want = ops.rotary(view, pos, inv)
    assert torch.equal(want, ops.rotary(view.clone(), pos.expand(2, 50).contiguous(), inv))
    tail = fused[..., 256:].clone()
    got = ops.rotary(view, pos, inv, inplace=True)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want) and torch.equal(fused[..., 256:], tail)
    head_major = torch.randn((2, 4, 50, 32), generator=g).to(DEV).transpose(1, 2)
    assert torch.equal(ops.rotary(head_major, pos, inv), ops.rotary(head_major.contiguous(), pos, inv))
    odd = torch.randn((2, 50, 4, 33), generator=g).to(torch.float16).to(DEV)[..., 1:]
    assert torch.equal(ops.rotary(odd, pos, inv), ops.rotary(odd.contiguous(), pos, inv))
    back = ops.rotary_backward(want, pos, inv)
    ref = ops.rotary_backward(ops.rotary(view.clone(), pos, inv), pos, inv)
    assert back.shape == ref.shape and float((ref - view).abs().max()) < 16 * 2.0 ** -22 * float(view.abs().max())
    assert ops.rotary(torch.empty((0, 5, 2, 32), device=DEV), torch.arange(5, device=DEV), inv).shape == (0, 5, 2, 32)


def test_rotary_graph(built_lib):
    x, pos = torch.randn((4, 1, 8, 64), device=DEV).to(torch.bfloat16), torch.full((4, 1), 100, device=DEV)
    inv, _ = ops.rotary_frequencies(64, device=DEV)
    ops.rotary(x, pos, inv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rotary(x, pos, inv)
    for _ in range(3):
        pos.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.rotary(x, pos, inv))


def test_refusals_on_device(built_lib):
    x, g = torch.randn((4, 64), device=DEV), torch.ones(64, device=DEV)
    bad = [lambda: ops.layernorm_forward(x.double(), g, g), lambda: ops.layernorm_forward(x, g[:32], g[:32]),
           lambda: ops.layernorm_forward(x, g.half(), g.half()), lambda: ops.layernorm_forward(x, g, g, residual=x[:2]),
           lambda: ops.layernorm_forward(x, g, g.half()), lambda: ops.layernorm_forward(x.clone().requires_grad_(), g, g),
           lambda: ops.layernorm_forward(torch.randn((2, 16385), device=DEV), torch.ones(16385, device=DEV), torch.ones(16385, device=DEV)),
           lambda: ops.layernorm_backward(x, x, g, g, g), lambda: ops.layernorm_forward(x, g, g.cpu())]
    h = torch.randn((2, 3, 4, 32), device=DEV)
    pos, inv = torch.arange(3, device=DEV), ops.rotary_frequencies(32, device=DEV)[0]
    bad += [lambda: ops.rotary(h, pos.float(), inv), lambda: ops.rotary(h, pos, inv.float()), lambda: ops.rotary(h, pos[:2], inv),
            lambda: ops.rotary(h, pos, inv, axes=2), lambda: ops.rotary(h[0], pos, inv), lambda: ops.rotary(h, pos, inv.repeat(2)),
            lambda: ops.rotary(h[:1].expand(2, 3, 4, 32), pos, inv, inplace=True), lambda: ops.rotary(h.transpose(2, 3), pos, inv[:2], inplace=True),
            lambda: ops.rotary(h.double(), pos, inv), lambda: ops.rotary(h, pos.cpu(), inv),
            lambda: ops.rotary(torch.randn((1, 2, 2, 520), device=DEV), pos[:2], inv)]
    for call in bad:
        with pytest.raises(_lib.DfsfmError):
            call()
    with torch.no_grad():
        ops.layernorm_forward(x.clone().requires_grad_(), g, g)
