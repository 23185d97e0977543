"""How far cross attention's results may be from 64 bits in the 2-norm, where weights and score gradients enter their products as two operands.

A bound on each element grows with the sum of all absolute terms and cannot see whether a term was rounded once more.  The 2-norm can: a
result is off by its own rounding, R = |round(x) - x|, and by the operands' errors.  n terms w_i x_i whose operands w_i are each off by at
most f of themselves, in either direction, give an error of expected square at most f^2 sum w_i^2 x_i^2 =: (f W)^2, so the result's is at
most sqrt(R^2 + (f W)^2).  As two operands, 7/8 and the rounded rest, a weight is off by f = ut (1/8 + 1/256), ut half a step of the type
(the rest is at most 1/8 and 7/8's rounding error, 2^-8 at most); rounded once, by up to ut, which alone is as large as the result's own
rounding.  ``SLACK`` is for the spread of a norm over the results of one test (6144 at least: 1 / sqrt(2 n) = 0.9 %), the 32-bit sums,
below 1 % of a 16-bit type's step, and nothing else."""
import math

import torch

SLACK = 1.1


def half_step(t):
    return torch.finfo(t).eps / 2


def terms(q, k, v, do, there, scale, out=None):
    """64-bit {name: (result, 2-norm W of its terms)} by heads, [N, H or Hkv, rows, D]; delta from ``out`` where given, else exact."""
    G = q.shape[2] // k.shape[2]
    z = there[:, :, None, None]
    Q, DO = (x.double().permute(0, 2, 1, 3) for x in (q, do))
    K, V = (torch.where(z, x.double(), 0.0).permute(0, 2, 1, 3).repeat_interleave(G, 1) for x in (k, v))
    s = (scale * Q @ K.transpose(2, 3)).masked_fill(~there[:, None, None, :], -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)                                # a sequence without keys
    exact = p @ V
    delta = (DO * (exact if out is None else out.double().cpu().permute(0, 2, 1, 3))).sum(-1, keepdim=True)
    ds = p * (DO @ V.transpose(2, 3) - delta)
    return {"Q": Q, "K": K, "V": V, "DO": DO, "p": p, "ds": ds, "G": G, "scale": scale}


def products(c, p, ds):
    """The results for weights p and score gradients ds."""
    def shared(x):
        return x.unflatten(1, (-1, c["G"])).sum(2)
    return {"out": p @ c["V"] / p.sum(-1, keepdim=True).clamp(min=1e-300), "dq": c["scale"] * ds @ c["K"],
            "dk": c["scale"] * shared(ds.transpose(2, 3) @ c["Q"]), "dv": shared(p.transpose(2, 3) @ c["DO"])}


def spreads(c):
    """W of each result."""
    def shared(x):
        return x.unflatten(1, (-1, c["G"])).sum(2)
    p2, ds2 = c["p"] ** 2, c["ds"] ** 2
    w = {"out": p2 @ c["V"] ** 2, "dq": ds2 @ c["K"] ** 2, "dk": shared(ds2.transpose(2, 3) @ c["Q"] ** 2), "dv": shared(p2.transpose(2, 3) @ c["DO"] ** 2)}
    return {n: math.sqrt(float(x.sum())) * (c["scale"] if n in ("dq", "dk") else 1.0) for n, x in w.items()}


def allowed(exact, W, t):
    own = float((exact.to(t).double() - exact).norm())
    return SLACK * math.hypot(own, half_step(t) * (1 / 8 + 1 / 256) * W)


def rounded_to(x, t):
    """x to t's digits, of any exponent (the kernels carry fp16 gradients with a power of two a column)."""
    m, e = torch.frexp(x)
    digits = 8 if t == torch.bfloat16 else 11
    return torch.ldexp(torch.round(m * 2.0 ** digits), e - digits)


def two_operands(x, t):
    p = rounded_to(0.875 * x, t)
    return p + rounded_to(x - p, t)
