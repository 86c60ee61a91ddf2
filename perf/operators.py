"""The operators on 8-bit activations, as cases that can be timed and compared.

A row is held in 8 bits as whole numbers q with one scale for the row (operands of products) or for every 64 of its
columns (what the backward pass reads again).  Of a group with the largest magnitude a:

    scale = a / 127        q = rint(x * (127 / a))        value = q * scale

``norm8``    residual add and norm of a forward pass that nothing differentiates, its output in 8 bits: h = res + delta as the
             residual stream stores it, y = h * rsqrt(mean(h^2) + eps) * w, rows of y in 8 bits.
``linear8``  a projection in 8 bits: rows of x in 8 bits, y[t, n] = sx[t] * sw[n] * sum_k xq[t, k] * wq[n, k].
``norm``     residual add and norm of a training step, forward and backward: the normalised rows xn = h * rsqrt(..) are kept in
             8 bits only; g = dy * w, dres = dh + rsqrt(..) * (g - xn * mean(g * xn)), dw = sum over rows of dy * xn.
``ffn``      the feed-forward part of a training step, forward and backward: gu = x w13^T, y = (silu(g) * u) w2^T; x and gu are kept
             in 8 bits, the activation not at all; the gradients are the formula's at the kept values.

``own`` false: the formulas in elementary torch operations, fp32 throughout; true: the framework's operators."""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
EPS = 1e-5
GROUP = 64          # columns that share a scale in what the backward pass reads


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a validator's norm in front of an 8-bit projection, 8B width, two sequences of 2048 tokens
        {"name": "norm8_8b", "op": "norm8", "tokens": 4096, "dim": 4096},
        # the smallest call: one token of the 1B model
        {"name": "norm8_token", "op": "norm8", "tokens": 1, "dim": 2048},
        # texts as they come: a token count and a width of no tile
        {"name": "norm8_ragged", "op": "norm8", "tokens": 1111, "dim": 1001},
        # the packed gate and up projection of the 1B model on a validator's batch of 4 x 2048 tokens
        {"name": "linear8_1b", "op": "linear8", "tokens": 8192, "dim": 2048, "out": 16384},
        # the down projection of the 8B model on one sequence of 1024 tokens: a long inner dimension
        {"name": "linear8_down_8b", "op": "linear8", "tokens": 1024, "dim": 14336, "out": 4096},
        # one token through the packed gate and up projection of the 1B model: the weight's bytes count
        {"name": "linear8_token", "op": "linear8", "tokens": 1, "dim": 2048, "out": 16384},
        # the next tokens of 24 texts through the packed query, key and value projection of the 8B model
        {"name": "linear8_few", "op": "linear8", "tokens": 24, "dim": 4096, "out": 6144},
        # every size odd
        {"name": "linear8_ragged", "op": "linear8", "tokens": 777, "dim": 1003, "out": 1111},
        # residual add and norm of the 1B model, forward and backward, on the benchmark's micro-batch of 8 x 2048 tokens
        {"name": "norm_1b", "op": "norm", "tokens": 16384, "dim": 2048},
        # the same of the 150M model on one sequence of 512 tokens
        {"name": "norm_150m", "op": "norm", "tokens": 512, "dim": 768},
        # the feed-forward part of a 1B block on the benchmark's micro-batch
        {"name": "ffn_1b", "op": "ffn", "tokens": 16384, "dim": 2048, "hidden": 8192},
        # a small model on a text as it comes
        {"name": "ffn_ragged", "op": "ffn", "tokens": 1999, "dim": 1024, "hidden": 2816},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Widths as models have them (whole groups of 64), one in four as it falls."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["norm8", "linear8", "linear8", "norm", "ffn"])
    if op in ("norm8", "norm"):
        return {"op": op, "tokens": _log(rng, 1, 16384), "dim": _width(rng, 256, 8192)}
    if op == "linear8":
        dim, out = _width(rng, 256, 16384), _width(rng, 256, 32768)
        return {"op": op, "tokens": _log(rng, 1, min(16384, 8192 * 2048 * 16384 // (dim * out))), "dim": dim, "out": out}
    # the bf16 products take rows of whole 16-byte pieces, so these widths are multiples of 8
    dim, hidden = rng.choice([(768, 2048), (1024, 2816), (1536, 4096), (2048, 8192), (1000, 2728), (4096, 14336)])
    return {"op": op, "tokens": _log(rng, 64, min(16384, 16384 * 2048 * 8192 // (dim * hidden))), "dim": dim, "hidden": hidden}


# ------------------------------------------------------------------------------------------ inputs
def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dtype)


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": c}
    T, D = c["tokens"], c["dim"]
    if c["op"] in ("norm8", "norm"):
        s["res"], s["delta"] = _normal(g, T, D, std=2.0), _normal(g, T, D)
        s["res"][:, ::97] *= 8                                             # channels that stand out, as trained models have them
        s["w"] = (1 + 0.1 * _normal(g, D, dtype=torch.float32)).to(torch.bfloat16)
    if c["op"] == "norm":
        s["dh"], s["dy"] = _normal(g, T, D, std=1e-3), _normal(g, T, D, std=1e-3)
        for k in ("res", "delta", "w"):
            s[k].requires_grad_()
    if c["op"] == "linear8":
        s["x"] = _normal(g, T, D)
        s["x"][:, ::89] *= 6
        # a weight in 8 bits as its owner keeps it: rows on 16-byte boundaries, one scale for each output channel
        rows = torch.zeros(c["out"], -(-D // 16) * 16, dtype=torch.int8, device=DEV)
        rows[:, :D] = torch.randint(-127, 128, (c["out"], D), generator=g, device=DEV, dtype=torch.int8)
        s["wq"] = rows[:, :D]
        s["ws"] = (1 + torch.rand(c["out"], generator=g, device=DEV)) * (D ** -0.5 / 127)
    if c["op"] == "ffn":
        F = c["hidden"]
        s["x"] = _normal(g, T, D).requires_grad_()
        s["w13"], s["w2"] = _normal(g, 2 * F, D, std=D ** -0.5).requires_grad_(), _normal(g, D, F, std=F ** -0.5).requires_grad_()
        s["dy"] = _normal(g, T, D, std=1e-3)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_own if own else _plain)(s, s["case"])


def _own(s, c):
    from templar_b200 import ops

    if c["op"] == "norm8":
        h, rows = ops.add_rmsnorm_q8(s["res"], s["delta"], s["w"], EPS)
        return {"h": h, "y": rows.dequantize()}
    if c["op"] == "linear8":
        return {"y": ops.linear_q8(s["x"], ops.QuantWeight(s["wq"], s["ws"]))}
    if c["op"] == "norm":
        h, y, _ = ops.add_rmsnorm_saved8(s["res"], s["delta"], s["w"], EPS)
        dres, ddelta, dw = torch.autograd.grad((h, y), (s["res"], s["delta"], s["w"]), (s["dh"], s["dy"]))
        return {"h": h.detach(), "y": y.detach(), "dres": dres, "ddelta": ddelta, "dw": dw}
    y = ops.feed_forward_saved8(s["x"], s["w13"], s["w2"])
    dx, dw13, dw2 = torch.autograd.grad(y, (s["x"], s["w13"], s["w2"]), s["dy"])
    return {"y": y.detach(), "dx": dx, "dw13": dw13, "dw2": dw2}


def _codes(x, group):
    """(q as fp32, scale) of rows of fp32, a scale for every ``group`` columns; scale has x's shape."""
    n = x.shape[-1]
    pad = -n % group
    xg = torch.cat((x, x.new_zeros(x.shape[0], pad)), dim=1).view(x.shape[0], -1, group)
    a = xg.abs().amax(-1, keepdim=True)
    q = torch.round(xg * (127 / a))
    wide = lambda t: t.expand_as(xg).reshape(x.shape[0], -1)[:, :n]  # noqa: E731
    return wide(q), wide(a / 127)


def _kept(x, group=GROUP):
    q, scale = _codes(x, group)
    return q * scale


def _plain(s, c):
    with torch.no_grad():
        if c["op"] == "linear8":
            q, scale = _codes(s["x"].float(), c["dim"])
            return {"y": ((q @ s["wq"].float().t()) * (scale[:, :1] * s["ws"])).to(torch.bfloat16)}
        if c["op"] == "ffn":
            return _plain_ffn(s)
        h = (s["res"].float() + s["delta"].float()).to(torch.bfloat16)
        x, w = h.float(), s["w"].float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        if c["op"] == "norm8":
            return {"h": h, "y": _kept(x * r * w, c["dim"]).to(torch.bfloat16)}
        y = (x * r * w).to(torch.bfloat16)
        xn, dy = _kept(x * r), s["dy"].float()
        g = dy * w
        dres = (s["dh"].float() + r * (g - xn * (g * xn).mean(-1, keepdim=True))).to(torch.bfloat16)
        return {"h": h, "y": y, "dres": dres, "ddelta": dres, "dw": (dy * xn).sum(0).to(torch.bfloat16)}


def _plain_ffn(s):
    x, w13, w2, dy = s["x"].float(), s["w13"].float(), s["w2"].float(), s["dy"].float()
    gu = x @ w13.t()
    gate, up = gu.chunk(2, dim=-1)
    y = ((gate * torch.sigmoid(gate) * up) @ w2.t()).to(torch.bfloat16)
    gate, up = _kept(gate), _kept(up)
    x = _kept(x)
    sg = torch.sigmoid(gate)
    dact = dy @ w2
    dw2 = (dy.t() @ (gate * sg * up)).to(torch.bfloat16)
    dgu = torch.cat((dact * up * sg * (1 + gate * (1 - sg)), dact * gate * sg), dim=-1)
    return {"y": y, "dx": (dgu @ w13).to(torch.bfloat16), "dw13": (dgu.t() @ x).to(torch.bfloat16), "dw2": dw2}


# ------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    T, D = float(c["tokens"]), float(c["dim"])
    if c["op"] == "norm8":
        return {"bytes": T * D * (2 + 2 + 2 + 2) + 2 * D, "flops": 0}              # res, delta; h, the values of y
    if c["op"] == "linear8":
        return {"bytes": 2 * T * D + D * c["out"] + 4 * c["out"] + 2 * T * c["out"], "flops": 2 * T * D * c["out"]}
    if c["op"] == "norm":
        return {"bytes": T * D * 2 * (4 + 3) + 4 * D, "flops": 0}                   # res, delta, dh, dy; h, y, the shared gradient
    F = c["hidden"]
    return {"bytes": 2 * T * D * 4 + 2 * 2 * 3 * D * F, "flops": 18 * T * D * F}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _held(x, width):
    """Rows of float64 with the values that 8 bits leave of them, group by group."""
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], width):
        part = x[:, at:at + width]
        top = part.abs().max(dim=1, keepdim=True).values
        out[:, at:at + width] = (part / top * 127).round() / 127 * top
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v)}
    D = c["dim"]
    if c["op"] == "linear8":
        return {"y": _held(f["x"], D) @ (f["wq"] * f["ws"][:, None]).t()}
    if c["op"] == "ffn":
        x, F = f["x"], c["hidden"]
        w1, w3, w2, dy = f["w13"][:F], f["w13"][F:], f["w2"], f["dy"]
        gate, up = x @ w1.t(), x @ w3.t()
        y = (torch.nn.functional.silu(gate) * up) @ w2.t()
        gate, up, x = _held(gate, GROUP), _held(up, GROUP), _held(x, GROUP)
        sig = 1 / (1 + torch.exp(-gate))
        act, slope = gate * sig, sig + gate * sig * (1 - sig)
        da = dy @ w2
        dg, du = da * up * slope, da * act
        return {"y": y, "dx": dg @ w1 + du @ w3, "dw13": torch.cat((dg.t() @ x, du.t() @ x)), "dw2": dy.t() @ (act * up)}
    h = (f["res"] + f["delta"]).to(torch.bfloat16).double()
    rms = (h.pow(2).sum(1, keepdim=True) / D + EPS).sqrt()
    if c["op"] == "norm8":
        return {"h": h, "y": _held(h / rms * f["w"], D)}
    xn = _held(h / rms, GROUP)
    g = f["dy"] * f["w"]
    dres = f["dh"] + (g - xn * (g * xn).sum(1, keepdim=True) / D) / rms
    return {"h": h, "y": h / rms * f["w"], "dres": dres, "ddelta": dres, "dw": (f["dy"] * xn).sum(0)}
