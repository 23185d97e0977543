"""What the training and serving operators beside the matching path are measured on: layer norm with its gradient, rotary positions,
and softmax cross attention to an encoder's states of another length with its gradient and its single-token form.

``run`` computes a case either with elementary torch operations in 32 bits (``own`` False) or with this package's entry points (``own``
True); both read the same inputs.  ``exact`` is the definition of each operator in 64 bits, gradients by automatic differentiation.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
DEVICE = "cuda"


def listed():
    return [
        # A coarse transformer layer's norm2 over both images of a 480 x 640 pair (60 x 80 tokens each), residual added behind it.
        {"name": "norm_coarse_tokens", "op": "norm", "pass": "forward", "type": "fp32", "rows": 9600, "width": 256, "residual": True},
        # A training step over the refinement head's tokens: 2000 windows of 15 x 15, d_model 128, in 32 bits.
        {"name": "norm_refine_train", "op": "norm", "pass": "train", "type": "fp32", "rows": 450000, "width": 128, "residual": True},
        # A wide model's training step in bf16.
        {"name": "norm_wide_train", "op": "norm", "pass": "train", "type": "bf16", "rows": 8192, "width": 4096, "residual": False},
        # Three tokens of an odd width: latency.
        {"name": "norm_few_odd", "op": "norm", "pass": "forward", "type": "fp16", "rows": 3, "width": 769, "residual": False},
        # One new token for each of 16 sequences, far into them.
        {"name": "rotary_single", "op": "rotary", "pass": "forward", "type": "bf16", "batch": 16, "length": 1, "heads": 8, "dim": 64,
         "rotated": 64, "axes": 1, "interleaved": True, "scaling": "none", "start": 900000},
        # Row and column positions of the coarse tokens of four images, each axis on a half of the head.
        {"name": "rotary_grid", "op": "rotary", "pass": "forward", "type": "fp32", "batch": 4, "length": 4800, "heads": 8, "dim": 32,
         "rotated": 32, "axes": 2, "interleaved": False, "scaling": "none", "start": 0},
        # The gradient of a long sequence whose heads are rotated in part, frequencies stretched for long contexts.
        {"name": "rotary_long_backward", "op": "rotary", "pass": "backward", "type": "bf16", "batch": 1, "length": 131072, "heads": 16,
         "dim": 128, "rotated": 64, "axes": 1, "interleaved": False, "scaling": "yarn", "start": 5},
        # A handful of query points that look at five states: latency.
        {"name": "cross_tiny", "op": "cross", "pass": "forward", "type": "bf16", "batch": 1, "queries": 7, "keys": 5, "heads": 8,
         "kv_heads": 8, "dim": 32, "mask": "none"},
        # One token of each of 16 sequences against the states of a 104 x 104 token map, ragged lengths.
        {"name": "cross_single", "op": "cross", "pass": "forward", "type": "fp16", "batch": 16, "queries": 1, "keys": 10816, "heads": 8,
         "kv_heads": 8, "dim": 64, "mask": "lens"},
        # Coarse tokens of a 480 x 640 image against those of an 832 x 832 one padded on two sides, d_model 256 and 8 heads in 32 bits.
        {"name": "cross_grid", "op": "cross", "pass": "forward", "type": "fp32", "batch": 2, "queries": 4800, "keys": 10816, "heads": 8,
         "kv_heads": 8, "dim": 32, "mask": "grid"},
        # A training step with shared key heads and ragged lengths, one of them empty.
        {"name": "cross_train", "op": "cross", "pass": "train", "type": "bf16", "batch": 4, "queries": 4800, "keys": 6400, "heads": 16,
         "kv_heads": 4, "dim": 128, "mask": "lens"},
        # A training step of many tokens against a few states of odd number.
        {"name": "cross_short_train", "op": "cross", "pass": "train", "type": "fp16", "batch": 8, "queries": 4800, "keys": 77, "heads": 8,
         "kv_heads": 8, "dim": 64, "mask": "none"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["fp32", "bf16", "fp16"])
    op = rng.choice(["norm", "norm", "rotary", "cross", "cross"])
    if op == "norm":
        width = _log_uniform(rng, 8, 8192)
        if rng.random() < 0.5:
            width = -(-width // 64) * 64
        rows = _log_uniform(rng, 1, max(1, min(450000, 57600000 // width)))
        return {"op": op, "pass": rng.choice(["forward", "train"]), "type": kind, "rows": rows, "width": width, "residual": rng.random() < 0.5}
    if op == "rotary":
        axes = rng.choice([1, 1, 2])
        dim = rng.choice([16, 32, 48, 64, 96, 128, 256])
        rotated = rng.choice([dim, dim, dim // 2])
        heads = rng.choice([1, 2, 5, 8, 16, 32])
        batch = rng.choice([1, 2, 3, 8, 16])
        length = _log_uniform(rng, 1, max(1, 134217728 // (dim * heads * batch * (2 if kind == "fp32" else 1))))
        return {"op": op, "pass": rng.choice(["forward", "backward"]), "type": kind, "batch": batch, "length": min(length, 131072), "heads": heads,
                "dim": dim, "rotated": rotated, "axes": axes, "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "start": rng.choice([0, 0, 17, _log_uniform(rng, 1, 1000000)])}
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([16, 32, 32, 40, 64, 64, 80, 128])
    batch = rng.choice([1, 2, 3, 4, 8, 16])
    queries = rng.choice([1, _log_uniform(rng, 1, 10816), _log_uniform(rng, 16, 10816)])
    # scores of all heads stay under those of the largest listed case, and its 32-bit ones under the listed 32-bit case's
    most = (1966080000 if kind != "fp32" else 830668800) * 32 // max(dim, 32) // (batch * heads * queries)
    keys = _log_uniform(rng, 1, max(1, min(16384, most)))
    mask = rng.choice(["none", "lens", "lens", "grid"])
    # a softmax over one key has no gradient for queries and keys: what is left of it in 32 bits is rounding alone
    return {"op": op, "pass": rng.choice(["forward", "train"]) if keys >= 8 else "forward", "type": kind, "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "mask": mask}


# ---------------------------------------------------------------- inputs
#: Shares of the keys that the sequences of a ragged batch hold; 0 is a sequence with none, which only batches of four and more have.
_SHARES = [1.0, 0.6, 0.85, 0.0, 0.35, 0.95, 0.1, 0.7]


def _lengths(case):
    return [int(math.ceil(_SHARES[i % 8] * case["keys"])) for i in range(case["batch"])]


def _grids(case):
    """(rows, columns, valid rows, valid columns) of each sequence's key map: padded below and at the right, as images of other shapes are."""
    h = int(math.isqrt(case["keys"]))
    w = -(-case["keys"] // h)
    return [(h, w, max(1, int(h * (1.0, 0.75, 1.0, 0.5)[i % 4])), max(1, int(w * (0.75, 1.0, 0.5, 1.0)[i % 4]))) for i in range(case["batch"])]


def _grid_valid(case, i):
    h, w, hv, wv = _grids(case)[i]
    s = torch.arange(case["keys"])
    return (s // w < hv) & (s % w < wv)


def _valid_keys(case):
    """Keys that each sequence may look at, in the order before the seed's permutation."""
    if case["mask"] == "lens":
        return _lengths(case)
    if case["mask"] == "grid":
        return [int(_grid_valid(case, i).sum()) for i in range(case["batch"])]
    return [case["keys"]] * case["batch"]


def _frequencies(case):
    """Angles per position of the pairs of one axis, in 64 bits, and the factor on the rotated values."""
    pairs = case["rotated"] // (2 * case["axes"])
    base, factor, trained = 10000.0, 8.0, 4096
    i = torch.arange(pairs, dtype=torch.float64)
    if case["scaling"] == "ntk" and pairs > 1:
        base = base * factor ** (pairs / (pairs - 1))
    inv = base ** (-i / pairs)
    if case["scaling"] == "linear":
        return inv / factor, 1.0
    if case["scaling"] == "yarn":
        turns = trained * inv / (2 * math.pi)
        keep = ((torch.log(turns) - math.log(1.0)) / (math.log(32.0) - math.log(1.0))).clamp(0, 1)
        return inv * keep + inv / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale + shift).to(t)

    state = {"case": dict(case)}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        state["x"] = normal(rows, width, scale=1.7, shift=0.4)
        state["gamma"] = (torch.randn(width, generator=g, device=DEVICE) * 0.2 + 1.0).to(t)
        state["beta"] = (torch.randn(width, generator=g, device=DEVICE) * 0.2).to(t)
        state["residual"] = normal(rows, width) if case["residual"] else None
        state["dy"] = normal(rows, width, scale=0.1) if case["pass"] == "train" else None
        return state
    if case["op"] == "rotary":
        batch, length = case["batch"], case["length"]
        state["x"] = normal(batch, length, case["heads"], case["dim"])
        first = case["start"] + torch.randint(0, 1000, (batch, 1), generator=host)
        at = torch.arange(length)[None] + first
        if case["axes"] == 2:
            wide = max(1, math.isqrt(length))
            at = torch.stack([torch.arange(length)[None] // wide + first, torch.arange(length)[None] % wide + first], -1)
        state["positions"] = at.to(DEVICE)
        inv, state["amplitude"] = _frequencies(case)
        state["inv_freq"] = inv.to(DEVICE)
        return state
    batch, keys = case["batch"], case["keys"]
    state["q"] = normal(batch, case["queries"], case["heads"], case["dim"], scale=1.5)
    state["k"] = normal(batch, keys, case["kv_heads"], case["dim"])
    state["v"] = normal(batch, keys, case["kv_heads"], case["dim"])
    state["dout"] = normal(batch, case["queries"], case["heads"], case["dim"], scale=0.1) if case["pass"] == "train" else None
    state["kv_lens"] = state["kv_mask"] = None
    order = torch.randperm(batch, generator=host)
    if case["mask"] == "lens":
        lens = torch.tensor(_lengths(case))[order]
        state["kv_lens"] = lens.to(torch.int32).to(DEVICE)
        valid = torch.arange(keys)[None] < lens[:, None]
    elif case["mask"] == "grid":
        valid = torch.stack([_grid_valid(case, int(i)) for i in order])
        state["kv_mask"] = valid.to(DEVICE)
    if case["mask"] != "none":
        # what stands in padded places is whatever the memory held
        junk = torch.tensor([float("nan"), float("inf"), -60000.0], device=DEVICE).to(t)
        at = (~valid).to(DEVICE)[:, :, None, None]
        fill = junk[torch.arange(keys, device=DEVICE) % 3][None, :, None, None]
        state["k"] = torch.where(at, fill, state["k"])
        state["v"] = torch.where(at, fill, state["v"])
    return state


# ---------------------------------------------------------------- plain forms
def _plain_norm(s):
    t = s["x"].dtype
    x, gamma, beta = s["x"].float(), s["gamma"].float(), s["beta"].float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    hat = centred * rstd
    y = hat * gamma + beta
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if s["dy"] is None:
        return {"y": y.to(t)}
    dy = s["dy"].float()
    dh = dy * gamma
    dx = rstd * (dh - dh.mean(-1, keepdim=True) - hat * (dh * hat).mean(-1, keepdim=True))
    return {"y": y.to(t), "dx": dx.to(t), "dgamma": (dy * hat).sum(0).to(t), "dbeta": dy.sum(0).to(t)}


def _plain_rotary(s):
    case, x = s["case"], s["x"]
    t, axes = x.dtype, case["axes"]
    at = s["positions"].double()
    at = at[..., None] if axes == 1 else at
    angle = at[..., None] * s["inv_freq"]                                     # [batch, length, axes, pairs], 64 bits
    cos = (angle.cos() * s["amplitude"]).float()[:, :, None]
    sin = (angle.sin() * s["amplitude"]).float()[:, :, None]
    sin = -sin if case["pass"] == "backward" else sin
    pairs = s["inv_freq"].numel()
    part = x[..., :case["rotated"]].float()
    if case["interleaved"]:
        part = part.reshape(*part.shape[:3], axes, pairs, 2)
        a, b = part[..., 0], part[..., 1]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        part = part.reshape(*part.shape[:3], axes, 2, pairs)
        a, b = part[..., 0, :], part[..., 1, :]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -2)
    turned = turned.reshape(*x.shape[:3], case["rotated"]).to(t)
    return torch.cat([turned, x[..., case["rotated"]:]], -1)


def _plain_valid(s):
    keys = s["case"]["keys"]
    if s["kv_lens"] is not None:
        return torch.arange(keys, device=s["k"].device)[None] < s["kv_lens"][:, None]
    return s["kv_mask"]


def _plain_cross(s):
    case, t = s["case"], s["q"].dtype
    group = case["heads"] // case["kv_heads"]
    scale = 1.0 / math.sqrt(case["dim"])
    valid = _plain_valid(s)
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if valid is not None:
        k = torch.where(valid[:, :, None, None], k, 0.0)
        v = torch.where(valid[:, :, None, None], v, 0.0)
    q = q.permute(0, 2, 1, 3).contiguous()                                   # [batch, heads, queries, dim]
    k = k.permute(0, 2, 1, 3).repeat_interleave(group, 1).contiguous()
    v = v.permute(0, 2, 1, 3).repeat_interleave(group, 1).contiguous()
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if valid is not None:
        scores = scores.masked_fill(~valid[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    p = e / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, v)
    result = {"out": out.permute(0, 2, 1, 3).to(t), "lse": lse}
    if s["dout"] is None:
        return result
    dout = s["dout"].float().permute(0, 2, 1, 3).contiguous()
    dp = torch.matmul(dout, v.transpose(2, 3).contiguous())
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    shared = (case["batch"], case["kv_heads"], group, case["keys"], case["dim"])
    result["dq"] = dq.permute(0, 2, 1, 3).to(t)
    result["dk"] = dk.reshape(shared).sum(2).permute(0, 2, 1, 3).to(t)
    result["dv"] = dv.reshape(shared).sum(2).permute(0, 2, 1, 3).to(t)
    return result


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        return {"norm": _plain_norm, "rotary": _plain_rotary, "cross": _plain_cross}[case["op"]](state)
    from detectorfreesfm_amd import ops
    if case["op"] == "norm":
        y, mean, rstd = ops.layernorm_forward(state["x"], state["gamma"], state["beta"], eps=1e-5, residual=state["residual"])
        if state["dy"] is None:
            return {"y": y}
        dx, dgamma, dbeta = ops.layernorm_backward(state["dy"], state["x"], mean, rstd, state["gamma"])
        return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if case["op"] == "rotary":
        call = ops.rotary_backward if case["pass"] == "backward" else ops.rotary
        return call(state["x"], state["positions"], state["inv_freq"], amplitude=state["amplitude"], axes=case["axes"],
                    interleaved=case["interleaved"])
    out, lse = ops.cross_attention(state["q"], state["k"], state["v"], kv_lens=state["kv_lens"], kv_mask=state["kv_mask"])
    if state["dout"] is None:
        return {"out": out, "lse": lse}
    dq, dk, dv = ops.cross_attention_backward(state["dout"], state["q"], state["k"], state["v"], out, lse, kv_lens=state["kv_lens"],
                                              kv_mask=state["kv_mask"])
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        passes = 2 + (1 if case["residual"] else 0)
        per = 8
        if case["pass"] == "train":
            passes, per = passes + 2, 8 + 14                                  # dy in, dx out; x is read once
        return {"bytes": n * passes * size + case["width"] * size * (4 if case["pass"] == "train" else 2), "flops": n * per}
    if case["op"] == "rotary":
        n = case["batch"] * case["length"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * size + case["batch"] * case["length"] * case["axes"] * 8,
                "flops": 3 * case["batch"] * case["length"] * case["heads"] * case["rotated"]}
    keys = sum(_valid_keys(case))
    scores = case["queries"] * keys * case["heads"]
    rows = case["batch"] * case["queries"] * case["heads"] * case["dim"]
    states = keys * case["kv_heads"] * case["dim"]
    lse = case["batch"] * case["queries"] * case["heads"] * 4
    if case["pass"] == "train":
        whole = case["batch"] * case["keys"] * case["kv_heads"] * case["dim"]
        return {"bytes": size * (4 * rows + 2 * states + 2 * whole) + lse, "flops": 14 * scores * case["dim"]}
    return {"bytes": size * (2 * rows + 2 * states) + lse, "flops": 4 * scores * case["dim"]}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(s):
    leaves = [s[n].double().requires_grad_(s["dy"] is not None) for n in ("x", "gamma", "beta")]
    x, gamma, beta = leaves
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    y = (x - mean) / (var + 1e-5).sqrt() * gamma + beta
    y = y if s["residual"] is None else y + s["residual"].double()
    if s["dy"] is None:
        return {"y": y}
    dx, dgamma, dbeta = torch.autograd.grad(y, leaves, s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _exact_rotary(s):
    """Each pair as a complex number times amplitude * exp(i angle), its conjugate for the gradient."""
    case, pairs = s["case"], s["inv_freq"].numel()
    out = s["x"].double().clone()
    for axis in range(case["axes"]):
        at = s["positions"] if case["axes"] == 1 else s["positions"][..., axis]
        angle = at.double()[:, :, None, None] * s["inv_freq"].double()
        turn = torch.polar(torch.full_like(angle, s["amplitude"]), -angle if case["pass"] == "backward" else angle)
        lo = axis * 2 * pairs
        real, imag = ((slice(lo, lo + 2 * pairs, 2), slice(lo + 1, lo + 2 * pairs, 2)) if case["interleaved"]
                      else (slice(lo, lo + pairs), slice(lo + pairs, lo + 2 * pairs)))
        z = torch.complex(out[..., real].contiguous(), out[..., imag].contiguous()) * turn
        out[..., real], out[..., imag] = z.real, z.imag
    return out


def _exact_cross(s):
    """Head by head over the keys that are there alone; a sequence without any gives zeros."""
    case = s["case"]
    train, group = s["dout"] is not None, case["heads"] // case["kv_heads"]
    outs = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE),
            "lse": torch.full((case["batch"], case["heads"], case["queries"]), float("-inf"), dtype=torch.float64, device=DEVICE)}
    if train:
        outs |= {"d" + n: torch.zeros(s[n].shape, dtype=torch.float64, device=DEVICE) for n in "qkv"}
    for n in range(case["batch"]):
        if s["kv_lens"] is not None:
            there = torch.arange(int(s["kv_lens"][n]), device=DEVICE)
        else:
            there = torch.arange(case["keys"], device=DEVICE) if s["kv_mask"] is None else s["kv_mask"][n].nonzero()[:, 0]
        if not there.numel():
            continue
        for h in range(case["heads"]):
            q = s["q"][n, :, h].double().requires_grad_(train)
            k, v = (s[m][n, there, h // group].double().requires_grad_(train) for m in "kv")
            a = q @ k.T / math.sqrt(case["dim"])
            out = torch.softmax(a, -1) @ v
            outs["out"][n, :, h] = out.detach()
            outs["lse"][n, h] = torch.logsumexp(a.detach(), -1)
            if train:
                dq, dk, dv = torch.autograd.grad(out, (q, k, v), s["dout"][n, :, h].double())
                outs["dq"][n, :, h] = dq
                outs["dk"][n, there, h // group] += dk
                outs["dv"][n, there, h // group] += dv
    return outs


def exact(case, seed):
    if case["op"] == "cross" and case["batch"] * case["heads"] > 1024:
        return None
    return {"norm": _exact_norm, "rotary": _exact_rotary, "cross": _exact_cross}[case["op"]](prepare(case, seed))
