"""Operators of a decoder layer whose activations are held in 8 bits, as cases that can be timed and compared.

RMSNorm (with the residual's addition) whose output is e4m3 with one power-of-two scale for every 32 values, the product of such
rows with a weight in the same form, SwiGLU whose checkpoint for the backward is held that way, and the two halves of a
decoder layer made of them: norm and projection, SwiGLU and projection.  ``own`` False computes them from elementary operations
in 32 bits, True through the package.  Sizes are those of the repository's configurations (hidden 576, 2048 and 4096, intermediate
8192 and 11008, 4 x 1024 tokens a step) and what lies between and around them; ``draw`` spreads over the same ranges, odd
numbers of tokens and of output features included.

The 8-bit form Q(v): with s the smallest power of two (2^-127 at least) for which a block's largest |v| / s is at most 448, the
largest e4m3 value, each v becomes s times the e4m3 value nearest to v / s, ties to the even one.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "fp32": F32}
EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # the norm in front of a projection, for the one token that is decoded
        dict(name="norm_token", op="norm", rows=1, cols=2048, dtype="bf16", residual=True),
        # the same for a training batch of 16 sequences
        dict(name="norm_train", op="norm", rows=16384, cols=2048, dtype="bf16", residual=True),
        # fp32 activations of the small model, a length that is a multiple of nothing, the head of the residual stream
        dict(name="norm_ragged_fp32", op="norm", rows=3001, cols=576, dtype="fp32", residual=False),
        # SwiGLU of a training batch: forward, what it keeps, and the gradient from that
        dict(name="swiglu_train", op="swiglu", rows=16384, cols=8192, dtype="bf16"),
        # the same for a short batch of fp32 activations
        dict(name="swiglu_short_fp32", op="swiglu", rows=517, cols=1408, dtype="fp32"),
        # one token through a projection whose weight was laid out beforehand
        dict(name="linear_token", op="linear", rows=1, cols=2048, out=16384, train=False),
        # a few prompts of a frozen reference through a down projection
        dict(name="linear_ragged", op="linear", rows=1003, cols=11008, out=4096, train=False),
        # a training step of an attention projection: forward, both gradients
        dict(name="linear_train", op="linear", rows=16384, cols=4096, out=4096, train=True),
        # the norm and the gate and up projections, forward, of a short batch of the small model
        dict(name="norm_linear_short", op="norm_linear", rows=333, cols=576, out=1728, train=False),
        # the same in a training step: all gradients
        dict(name="norm_linear_train", op="norm_linear", rows=4096, cols=2048, out=16384, train=True),
        # SwiGLU and the down projection of the last tokens of a few answers
        dict(name="swiglu_linear_few", op="swiglu_linear", rows=24, cols=8192, out=2048, train=False),
        # the same in a training step of the larger model: all gradients
        dict(name="swiglu_linear_train", op="swiglu_linear", rows=8192, cols=11008, out=4096, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "swiglu", "linear", "norm_linear", "swiglu_linear"))
    while True:
        c = dict(op=op, rows=_log(rng, 1, 20000), cols=rng.choice((576, 2048, 4096, BLOCK * _log(rng, 6, 360), BLOCK * _log(rng, 6, 360))))
        if op in ("norm", "swiglu"):
            c["dtype"] = rng.choice(("bf16", "bf16", "fp32"))
            if op == "norm":
                c["residual"] = rng.random() < 0.7
        else:
            c["out"] = rng.choice((2048, 4096, 8 * _log(rng, 24, 2500), _log(rng, 200, 20000)))
            c["train"] = rng.random() < 0.5
        w = work(c)
        if w["flops"] < 1.6e12 and w["bytes"] < 1.6e9:
            return c


# ------------------------------------------------------------------------------------------------------- the states
def _activations(shape, g, dtype):
    """Normal values with a scale of its own for every channel, and now and then a channel that is far larger, as in a residual stream."""
    scale = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    scale = torch.where(torch.rand(shape[-1], generator=g, device="cuda") < 0.003, 12 * scale, scale)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, rows, cols, train = case, case["rows"], case["cols"], case.get("train", False)
    dtype = DTYPES[c.get("dtype", "bf16")]

    def normal(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case=case)
    if c["op"] in ("norm", "norm_linear"):
        s["x"] = _activations((rows, cols), g, dtype)
        s["residual"] = _activations((rows, cols), g, dtype) if c.get("residual", True) else None
        s["gamma"] = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    elif c["op"] == "linear":
        s["x"] = _activations((rows, cols), g, dtype)
    else:
        s["gate_up"] = normal(rows, 2 * cols, scale=1.5)
    if "out" in c:
        s["weight"] = normal(c["out"], cols, scale=cols ** -0.5)
        if train:
            s["dy"] = normal(rows, c["out"], scale=0.01)
            if c["op"] == "norm_linear":
                s["dh"] = normal(rows, cols, scale=0.01)
        elif own:   # a weight that is not trained is laid out once
            from picotron_amd import ops
            s["packed"] = ops.mx8_quantize(s["weight"])
        else:
            s["weight_values"] = _quantized(s["weight"].float())
    if c["op"] == "swiglu":
        s["dy"] = normal(rows, cols, scale=0.01)
    for name in ("x", "residual", "gamma", "gate_up", "weight") if train or c["op"] == "swiglu" else ():
        if s.get(name) is not None:
            s[name].requires_grad_()
    return s


def work(case):
    c, n, k, b = case, case["rows"], case["cols"], 4 if case.get("dtype") == "fp32" else 2
    held = 1 + 1 / BLOCK   # bytes of a value in the 8-bit form
    if c["op"] == "norm":   # x and the residual in, their sum out, the 8-bit form, and the values it stands for
        return {"bytes": n * k * (b * (3 if c["residual"] else 1) + held + 2) + k * b, "flops": 0}
    if c["op"] == "swiglu":   # gate and up in, their product out, the checkpoint out and in, the upstream gradient in, two gradients out
        return {"bytes": n * k * (2 * b + b + 2 * 2 * held + b + 2 * b), "flops": 0}
    m, train = c["out"], c["train"]
    weight = m * k * ((2 if train else held) + (2 if train else 0))   # in, and its gradient out
    inside = {"linear": 2 + (2 if train else 0), "norm_linear": 6 + (4 if train else 0), "swiglu_linear": 4 + (4 if train else 0)}[c["op"]]
    return {"bytes": n * k * inside + n * m * 2 * (2 if train else 1) + weight, "flops": 2.0 * n * m * k * (3 if train else 1)}


# ------------------------------------------------------------------------------------------------------- the plain form
def _power(e):
    """2^e of whole e in -126 .. 127."""
    return ((e + 127) << 23).to(torch.int32).view(F32)


def _quantized(v):
    """The values that the 8-bit form of v [rows, cols] stands for, fp32."""
    b = v.view(v.size(0), -1, BLOCK)
    part, e = torch.frexp(b.abs().amax(-1, keepdim=True))   # part in [1/2, 1): 448 is 7/8 of a power of two
    e = (e - 9 + (part > 0.875).to(e.dtype)).clamp(-126, 126)
    r = b * _power(-e)
    step = _power((torch.frexp(r.abs())[1] - 1).clamp(min=-6) - 3)
    return (torch.round(r / step) * step * _power(e)).view(v.shape)


def _silu(g):
    return g / (1 + torch.exp(-g))


def _swiglu_gradient(gate, up, dh):
    sig = 1 / (1 + torch.exp(-gate))
    return torch.cat((dh * up * sig * (1 + gate * (1 - sig)), dh * gate * sig), -1)


def _normalized(h):
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    return h * rstd, rstd


def _norm_gradient(h, gamma, dy, dh):
    n, rstd = _normalized(h)
    g = dy * gamma
    return rstd * (g - n * (g * n).mean(-1, keepdim=True)) + dh, (dy * n).sum(0)


@torch.no_grad()
def _plain(s):
    c = s["case"]
    op, train, f = c["op"], c.get("train", False), {k: v.float() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if op in ("norm", "norm_linear"):
        h = f["x"] + f["residual"] if s["residual"] is not None else f["x"]
        v = _quantized(_normalized(h)[0] * f["gamma"])
    if op == "norm":
        return (v.to(BF16),) + ((h.to(s["x"].dtype),) if s["residual"] is not None else ())
    if op in ("swiglu", "swiglu_linear"):
        gate, up = f["gate_up"].chunk(2, -1)
        v = _silu(gate) * up
    if op == "swiglu":
        gate, up = _quantized(f["gate_up"]).chunk(2, -1)
        return v.to(s["gate_up"].dtype), _swiglu_gradient(gate, up, f["dy"]).to(s["gate_up"].dtype)
    if op == "swiglu_linear":
        v = _quantized(v)
    if op == "linear":
        v = _quantized(f["x"])
    y = v @ (_quantized(f["weight"]) if train else s["weight_values"]).t()
    out = [y.to(BF16)] + ([h.to(BF16)] if op == "norm_linear" else [])
    if train:
        dv = f["dy"] @ f["weight"]
        if op == "linear":
            out += [dv, f["dy"].t() @ v]
        elif op == "norm_linear":
            out += [*_norm_gradient(h, f["gamma"], dv, f["dh"]), f["dy"].t() @ v]
        else:
            gate, up = _quantized(f["gate_up"]).chunk(2, -1)   # what the forward kept
            out += [_swiglu_gradient(gate, up, dv), f["dy"].t() @ (_silu(gate) * up)]
    return tuple(t.to(BF16) for t in out)


# ------------------------------------------------------------------------------------------------------- the package
def _own(s):
    from picotron_amd import functional, ops
    c = s["case"]
    op, train = c["op"], c.get("train", False)
    if op == "norm":
        packed, _, h = ops.rmsnorm_mx8_fwd(s["x"], s["gamma"], EPS, residual=s["residual"])
        return (packed.dequantize(BF16),) + ((h,) if s["residual"] is not None else ())
    if op == "swiglu":
        y = functional.swiglu_8bit(s["gate_up"])
        return (y, *torch.autograd.grad(y, s["gate_up"], s["dy"]))
    with torch.set_grad_enabled(train):
        if op == "linear":
            y, leaves = functional.linear_8bit(s["x"], s["weight"], packed=s.get("packed")), ("x", "weight")
        elif op == "norm_linear":
            y, h = functional.rms_norm_linear_8bit(s["x"], s["residual"], s["gamma"], EPS, s["weight"], packed=s.get("packed"))
            leaves = ("x", "gamma", "weight")
            if train:
                return (y, h, *torch.autograd.grad((y, h), [s[k] for k in leaves], (s["dy"], s["dh"])))
            return y, h
        else:
            y, leaves = functional.swiglu_linear_8bit(s["gate_up"], s["weight"], packed=s.get("packed")), ("gate_up", "weight")
    return (y, *torch.autograd.grad(y, [s[k] for k in leaves], s["dy"])) if train else (y,)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------- 64 bits
def _e4m3():
    """The values of e4m3 that are not negative, in order: the place of one in this list is its code."""
    return [(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8) if (e, m) != (15, 7)]


def _nearest(v):
    """The 8-bit form's values of v [rows, cols], fp64, by search among all of them."""
    values = torch.tensor(_e4m3(), dtype=F64, device=v.device)
    middles = (values[1:] + values[:-1]) / 2
    out = torch.empty_like(v)
    for first in range(0, v.size(0), 1024):
        b = v[first:first + 1024].reshape(-1, v.size(1) // BLOCK, BLOCK)
        largest = b.abs().amax(-1, keepdim=True)
        s = torch.exp2(torch.ceil(torch.log2(largest.clamp(min=1e-30) / 448)))
        r = (b.abs() / s).contiguous()
        below, above = torch.searchsorted(middles, r), torch.searchsorted(middles, r, right=True)   # (they differ where r is in the middle)
        code = torch.where(below % 2 == 0, below, above)
        out[first:first + 1024] = (torch.copysign(values[code], b) * s).view(-1, v.size(1))
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op, train = case["op"], case.get("train", False)
    x, r, gamma, gate_up, w, dy, dh = (None if s.get(k) is None else s[k].detach().to(F64) for k in ("x", "residual", "gamma", "gate_up", "weight", "dy", "dh"))
    if op.startswith("norm"):
        x = x if r is None else x + r
        rms = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.size(1) + EPS)
        a = _nearest(x / rms * gamma)
        if op == "norm":
            return (a,) if r is None else (a, x)
    elif op.startswith("swiglu"):
        half = case["cols"]
        a = gate_up[:, :half] * torch.sigmoid(gate_up[:, :half]) * gate_up[:, half:]
        if train or op == "swiglu":
            kept = _nearest(gate_up)
            kg, ku = kept[:, :half], kept[:, half:]
            sg = torch.sigmoid(kg)
            slope = sg + kg * sg * (1 - sg)
        if op == "swiglu":
            return a, torch.cat((dy * ku * slope, dy * kg * sg), 1)
        a = _nearest(a)
    else:
        a = _nearest(x)
    y = torch.mm(a, _nearest(w).t())
    head = (y, x) if op == "norm_linear" else (y,)
    if not train:
        return head
    da = torch.mm(dy, w)
    if op == "linear":
        return head + (da, torch.mm(dy.t(), a))
    if op == "norm_linear":
        n = x / rms
        inner = torch.sum(da * gamma * n, -1, keepdim=True) / x.size(1)
        return head + ((da * gamma - n * inner) / rms + dh, torch.sum(da * n, 0), torch.mm(dy.t(), a))
    return head + (torch.cat((da * ku * slope, da * kg * sg), 1), torch.mm(dy.t(), kg * sg * ku))
