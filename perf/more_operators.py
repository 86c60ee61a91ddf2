"""The operators of a training step on packed documents, as cases that can be timed and compared.

Sequences hold several documents one behind the other.  A row s of a sequence has a ``start``: it belongs to the document that
begins there, its position is s - start, and it sees the keys start .. s.  Rows behind the last document see nothing.

``docs``    attention within documents on a packed projection [B, S, (H + 2 KV) hd] (query, key, value heads):
            p = softmax over the visible keys of q.k hd^-0.5, out = p v, zero for a row that sees nothing; with ``train`` the gradient
            dv = p^T dout, ds = p (dout v^T - sum(dout * out)) hd^-0.5, dq = ds k, dk = ds^T q.
``qknorm``  norm of every query and key head and the rotary embedding: z = x rsqrt(mean(x^2) + eps) w, the pairs (2i, 2i + 1) of z turned
            by the angle of the row's position, value heads as they are; with ``train`` the gradients of the rows and both weights.
``loss``    cross entropy of the products x w^T: with ``train`` its mean over the labels that are not ignored and the gradients of x and
            w, else the loss of every token, zero where the label is ignored.

``own`` false: the formulas in elementary torch operations, fp32 throughout; true: the framework's operators."""

from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda"
EPS = 1e-5
IGNORE = -100


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a 1B block's attention, forward and backward, on the benchmark's micro-batch of packed texts
        {"name": "docs_1b", "op": "docs", "train": True, "batch": 8, "seq": 2048, "heads": 16, "kv": 16, "hd": 128, "mean": 512, "pad": False},
        # one long sequence of long texts, grouped heads of the 8B model, forward and backward
        {"name": "docs_long", "op": "docs", "train": True, "batch": 1, "seq": 16384, "heads": 32, "kv": 8, "hd": 128, "mean": 4096, "pad": False},
        # the 150M model on short texts as they come, sequences filled up behind the last one
        {"name": "docs_ragged", "op": "docs", "train": True, "batch": 3, "seq": 1999, "heads": 12, "kv": 12, "hd": 64, "mean": 120, "pad": True},
        # scoring two short texts, 150M heads: the smallest call
        {"name": "docs_short", "op": "docs", "train": False, "batch": 1, "seq": 60, "heads": 12, "kv": 12, "hd": 64, "mean": 30, "pad": False},
        # query and key norms of a 1B block, forward and backward, on the benchmark's micro-batch
        {"name": "qknorm_1b", "op": "qknorm", "train": True, "batch": 8, "seq": 2048, "heads": 16, "kv": 16, "hd": 128, "mean": 512, "pad": False},
        # the same of the 8B model's grouped heads while scoring
        {"name": "qknorm_8b", "op": "qknorm", "train": False, "batch": 2, "seq": 4096, "heads": 32, "kv": 8, "hd": 128, "mean": 1024, "pad": False},
        # heads of 80 on texts as they come, forward and backward
        {"name": "qknorm_ragged", "op": "qknorm", "train": True, "batch": 3, "seq": 777, "heads": 10, "kv": 5, "hd": 80, "mean": 90, "pad": True},
        # one token
        {"name": "qknorm_token", "op": "qknorm", "train": False, "batch": 1, "seq": 1, "heads": 12, "kv": 12, "hd": 64, "mean": 1, "pad": False},
        # the 1B model's output projection and loss, forward and backward, on the benchmark's micro-batch
        {"name": "loss_1b", "op": "loss", "train": True, "tokens": 16384, "dim": 2048, "vocab": 32000},
        # scoring with the 8B model's vocabulary
        {"name": "loss_8b", "op": "loss", "train": False, "tokens": 4096, "dim": 4096, "vocab": 128256},
        # a vocabulary and a token count of no tile, forward and backward
        {"name": "loss_ragged", "op": "loss", "train": True, "tokens": 1111, "dim": 1000, "vocab": 50257},
        # the next token of a short text, 150M width
        {"name": "loss_few", "op": "loss", "train": False, "tokens": 30, "dim": 768, "vocab": 32000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["docs", "docs", "qknorm", "loss"])
    train = rng.random() < 0.6
    if op == "loss":
        dim = max(128, _log(rng, 128, 8192) // 8 * 8)
        vocab = _log(rng, 500, min(131072, 128256 * 4096 // dim))
        if rng.random() < 0.5:
            vocab = -(-vocab // 128) * 128
        top = min(16384, 4096 * 128256 // vocab, 16384 * 2048 * 32000 // (dim * vocab))
        return {"op": op, "train": train, "tokens": _log(rng, 1, top), "dim": dim, "vocab": vocab}
    kv = rng.choice([1, 2, 4, 5, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 2, 3, 4])
    hd = rng.choice([64, 128]) if op == "docs" else rng.choice([64, 80, 96, 128, 256])
    seq = _log(rng, 1, 16384)
    top = max(1, 32768 // seq)
    if op == "docs":
        heads, kv = (heads, kv) if heads <= 32 else (32, 8)
        top = max(1, min(top, 16384 * 16384 * 32 * 128 // (seq * seq * heads * hd)))
    batch = _log(rng, 1, min(16, top))
    return {"op": op, "train": train, "batch": batch, "seq": seq, "heads": heads, "kv": kv, "hd": hd,
            "mean": _log(rng, 1, 4 * seq), "pad": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------ inputs
def _documents(case, seed):
    """For each sequence the lengths of its documents and the rows left over behind them."""
    c, rng = case, random.Random(int(seed) * 7919 + c_hash(case))
    out = []
    for _ in range(c["batch"]):
        left = c["seq"]
        pad = int(left * rng.uniform(0.05, 0.4)) if c["pad"] else 0
        left -= pad
        lens = []
        while left > 0:
            n = min(left, max(1, int(rng.lognormvariate(math.log(c["mean"]) - 0.32, 0.8))))        # texts: many short ones, few long
            if not lens:
                n = max(1, int(n * rng.random()))              # the sequence begins inside a text
            lens.append(n)
            left -= n
        out.append((lens, pad))
    return out


def c_hash(case):
    return sum(ord(ch) * (i + 1) for i, ch in enumerate(repr(sorted((k, v) for k, v in case.items() if k != "name"))))


def _starts(case, seed):
    rows = []
    for lens, pad in _documents(case, seed):
        at, row = 0, []
        for n in lens:
            row += [at] * n
            at += n
        rows.append(row + [case["seq"]] * pad)
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dtype)


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": c}
    if c["op"] == "loss":
        T, D, V = c["tokens"], c["dim"], c["vocab"]
        s["w"] = _normal(g, V, D, std=2 * D ** -0.5)
        s["labels"] = torch.randint(0, V, (T,), generator=g, device=DEV)
        x = torch.randn(T, D, generator=g, device=DEV)
        # tokens that the model has learned: their own logit stands out by up to 12
        x += (3 * torch.rand(T, 1, generator=g, device=DEV)) * s["w"][s["labels"]].float()
        s["x"] = x.to(torch.bfloat16)
        s["labels"][torch.rand(T, generator=g, device=DEV) < 0.1] = IGNORE
        s["labels"][0] = V - 1
        if c["train"]:
            s["x"].requires_grad_()
            s["w"].requires_grad_()
        return s
    B, S, H, KV, hd = c["batch"], c["seq"], c["heads"], c["kv"], c["hd"]
    s["qkv"] = _normal(g, B, S, (H + 2 * KV) * hd, std=1.3)
    s["starts"] = _starts(c, seed)
    if c["op"] == "docs":
        s["dout"] = _normal(g, B, S, H * hd, std=1e-2)
    else:
        s["qkv"][..., 5::hd] *= 6                                          # a channel that stands out, as trained heads have
        s["wq"], s["wk"] = ((1 + 0.2 * _normal(g, hd, dtype=torch.float32)).to(torch.bfloat16) for _ in range(2))
        rows = torch.arange(S, device=DEV, dtype=torch.int32)
        s["positions"] = (rows - s["starts"]).clamp_(min=0)
        ang = torch.arange(S, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["dout"] = _normal(g, B, S, (H + 2 * KV) * hd, std=1e-2)
    if c["train"]:
        for k in ("qkv", "wq", "wk"):
            if k in s:
                s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_own if own else _plain)(s, s["case"])


def _own(s, c):
    from templar_b200 import ops

    with torch.set_grad_enabled(c["train"]):
        if c["op"] == "loss":
            if not c["train"]:
                return {"losses": ops.linear_cross_entropy(s["x"], s["w"], s["labels"], ignore_index=IGNORE, reduction="none")}
            loss = ops.linear_cross_entropy(s["x"], s["w"], s["labels"], ignore_index=IGNORE)
            dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]))
            return {"loss": loss.detach(), "dx": dx, "dw": dw}
        if c["op"] == "docs":
            out = ops.attention_documents(s["qkv"], s["starts"], c["heads"], c["kv"], c["hd"])
            if not c["train"]:
                return {"out": out}
            (dqkv,) = torch.autograd.grad(out, (s["qkv"],), s["dout"])
            return {"out": out.detach(), "dqkv": dqkv}
        out = ops.qk_norm_rope(s["qkv"], s["wq"], s["wk"], s["cos"], s["sin"], c["heads"], c["kv"], c["hd"], EPS, positions=s["positions"])
        if not c["train"]:
            return {"out": out}
        dqkv, dwq, dwk = torch.autograd.grad(out, (s["qkv"], s["wq"], s["wk"]), s["dout"])
        return {"out": out.detach(), "dqkv": dqkv, "dwq": dwq, "dwk": dwk}


def _plain(s, c):
    with torch.no_grad():
        return {"loss": _plain_loss, "docs": _plain_docs, "qknorm": _plain_qknorm}[c["op"]](s, c)


def _plain_loss(s, c):
    x, w, labels = s["x"].float(), s["w"].float(), s["labels"]
    logits = x @ w.t()
    valid = labels != IGNORE
    at = labels.clamp(min=0)[:, None]
    top = logits.amax(1, keepdim=True)
    target = logits.gather(1, at)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    losses = (total.log() + top - target)[:, 0] * valid
    if not c["train"]:
        return {"losses": losses}
    n = valid.sum()
    loss = losses.sum() / n
    d = e / total
    d.scatter_add_(1, at, torch.full_like(target, -1.0))
    d *= valid[:, None] / n
    return {"loss": loss, "dx": (d @ w).to(torch.bfloat16), "dw": (d.t() @ x).to(torch.bfloat16)}


def _plain_docs(s, c):
    B, S, H, KV, hd = c["batch"], c["seq"], c["heads"], c["kv"], c["hd"]
    G, scale = H // KV, c["hd"] ** -0.5
    out = s["qkv"].new_empty(B, S, H * hd)
    dqkv = torch.empty_like(s["qkv"])
    rows = torch.arange(S, device=DEV)
    for b in range(B):
        seen = (rows[None, :] <= rows[:, None]) & (rows[None, :] >= s["starts"][b][:, None])
        for kv in range(KV):
            col = slice(kv * G * hd, (kv + 1) * G * hd)
            kcol, vcol = slice((H + kv) * hd, (H + kv + 1) * hd), slice((H + KV + kv) * hd, (H + KV + kv + 1) * hd)
            q = s["qkv"][b, :, col].float().view(S, G, hd).transpose(0, 1)
            k, v = s["qkv"][b, :, kcol].float(), s["qkv"][b, :, vcol].float()
            p = torch.where(seen, (q @ k.t()) * scale, float("-inf"))
            top = p.amax(-1, keepdim=True)
            p = torch.exp(p - torch.where(torch.isinf(top), 0.0, top))
            total = p.sum(-1, keepdim=True)
            p /= torch.where(total == 0, 1.0, total)
            o = p @ v
            out[b, :, col] = o.transpose(0, 1).reshape(S, G * hd)
            if c["train"]:
                do = s["dout"][b, :, col].float().view(S, G, hd).transpose(0, 1)
                delta = (do * o).sum(-1, keepdim=True)
                dqkv[b, :, vcol] = (p.transpose(1, 2) @ do).sum(0).to(torch.bfloat16)
                ds = (do @ v.t()).sub_(delta).mul_(p).mul_(scale)
                dqkv[b, :, col] = (ds @ k).transpose(0, 1).reshape(S, G * hd).to(torch.bfloat16)
                dqkv[b, :, kcol] = (ds.transpose(1, 2) @ q).sum(0).to(torch.bfloat16)
    return {"out": out, "dqkv": dqkv} if c["train"] else {"out": out}


def _plain_qknorm(s, c):
    B, S, H, KV, hd = c["batch"], c["seq"], c["heads"], c["kv"], c["hd"]
    R = H + KV
    x = s["qkv"][..., :R * hd].float().reshape(B, S, R, hd)
    w = torch.cat((s["wq"].float().expand(H, hd), s["wk"].float().expand(KV, hd)))
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    z = x * r * w
    a, b = z[..., 0::2], z[..., 1::2]
    z = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).view(B, S, R * hd)
    out = torch.cat((z.to(torch.bfloat16), s["qkv"][..., R * hd:]), -1)
    if not c["train"]:
        return {"out": out}
    dy = s["dout"][..., :R * hd].float().view(B, S, R, hd)
    a, b = dy[..., 0::2], dy[..., 1::2]
    u = torch.stack((a * cos + b * sin, b * cos - a * sin), -1).view(B, S, R, hd)
    xh, g = x * r, u * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    dw = (u * xh).double().sum((0, 1))
    return {"out": out, "dqkv": torch.cat((dx.view(B, S, R * hd).to(torch.bfloat16), s["dout"][..., R * hd:]), -1),
            "dwq": dw[:H].sum(0).to(torch.bfloat16), "dwk": dw[H:].sum(0).to(torch.bfloat16)}


# ------------------------------------------------------------------------------------------ work
def work(case):
    c = case
    if c["op"] == "loss":
        T, D, V = float(c["tokens"]), float(c["dim"]), float(c["vocab"])
        both = 2 if c["train"] else 1                                      # x and w; dx and dw
        return {"bytes": both * 2 * (T * D + V * D) + 8 * T, "flops": (6 if c["train"] else 2) * T * D * V}
    tokens, H, KV, hd = float(c["batch"] * c["seq"]), c["heads"], c["kv"], c["hd"]
    C = (H + 2 * KV) * hd
    if c["op"] == "qknorm":
        return {"bytes": tokens * (2 * C * (4 if c["train"] else 2) + 4), "flops": 0}     # qkv, out; dout, dqkv
    pairs = sum(n * (n + 1) / 2 for lens, _ in _documents(c, 0) for n in lens)
    rows = tokens * (2 * C + 2 * H * hd + 4)                               # qkv, out, starts
    if c["train"]:
        rows += tokens * (2 * C + 2 * H * hd)                              # dout, dqkv
    return {"bytes": rows, "flops": (14 if c["train"] else 4) * pairs * H * hd}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    f = {k: v.detach().double() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if c["op"] == "loss":
        return _exact_loss(c, f, s["labels"])
    return (_exact_docs if c["op"] == "docs" else _exact_qknorm)(c, f, s, seed)


def _exact_loss(c, f, labels):
    x, w = f["x"], f["w"]
    keep = (labels != IGNORE).nonzero()[:, 0]
    z = x[keep] @ w.t()
    lse = torch.logsumexp(z, 1)
    pick = torch.arange(len(keep), device=DEV), labels[keep]
    losses = torch.zeros(len(x), dtype=torch.float64, device=DEV)
    losses[keep] = lse - z[pick]
    if not c["train"]:
        return {"losses": losses}
    z = z.sub_(lse[:, None]).exp_()
    z[pick] -= 1
    z /= len(keep)
    dx = torch.zeros_like(x)
    dx[keep] = z @ w
    return {"loss": losses.sum() / len(keep), "dx": dx, "dw": z.t() @ x[keep]}


def _exact_docs(c, f, s, seed):
    """Document by document, each as a causal attention of its own."""
    B, S, H, KV, hd = c["batch"], c["seq"], c["heads"], c["kv"], c["hd"]
    out = torch.zeros(B, S, H * hd, dtype=torch.float64, device=DEV)
    dqkv = torch.zeros(B, S, (H + 2 * KV) * hd, dtype=torch.float64, device=DEV)
    for b, (lens, _) in enumerate(_documents(c, seed)):
        at = 0
        for n in lens:
            part = slice(at, at + n)
            at += n
            q, k, v = (t.transpose(0, 1) for t in f["qkv"][b, part].view(n, H + 2 * KV, hd).split([H, KV, KV], dim=1))
            later = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
            step = max(1, min(H, 400_000_000 // (n * n)))                  # heads at a time
            for h0 in range(0, H, step):
                hs = torch.arange(h0, min(H, h0 + step), device=DEV)
                kh, vh, cols = k[hs // (H // KV)], v[hs // (H // KV)], slice(h0 * hd, (h0 + len(hs)) * hd)
                p = torch.softmax((q[hs] @ kh.transpose(1, 2) / math.sqrt(hd)).masked_fill_(later, -math.inf), dim=-1)
                o = p @ vh
                out[b, part, cols] = o.transpose(0, 1).reshape(n, -1)
                if c["train"]:
                    do = f["dout"][b, part, cols].view(n, len(hs), hd).transpose(0, 1)
                    ds = p * (do @ vh.transpose(1, 2) - (do * o).sum(2, keepdim=True)) / math.sqrt(hd)
                    dqkv[b, part, cols] = (ds @ kh).transpose(0, 1).reshape(n, -1)
                    for at_col, grad in ((H, ds.transpose(1, 2) @ q[hs]), (H + KV, p.transpose(1, 2) @ do)):
                        shared = dqkv[b, part].view(n, H + 2 * KV, hd)
                        shared.index_add_(1, at_col + hs // (H // KV), grad.transpose(0, 1))
    return {"out": out, "dqkv": dqkv} if c["train"] else {"out": out}


def _exact_qknorm(c, f, s, seed):
    """The rotation as a product of complex numbers; the gradient through the projection onto the row's complement."""
    B, S, H, KV, hd = c["batch"], c["seq"], c["heads"], c["kv"], c["hd"]
    at = s["positions"].long()
    turn = torch.complex(f["cos"][at], f["sin"][at])[:, :, None]
    q, k, v = f["qkv"].view(B, S, H + 2 * KV, hd).split([H, KV, KV], dim=2)
    dq, dk, dv = f["dout"].view(B, S, H + 2 * KV, hd).split([H, KV, KV], dim=2)
    outs, grads, dws = [], [], []
    for x, dy, w in ((q, dq, f["wq"]), (k, dk, f["wk"])):
        norm = (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
        unit = x / norm
        outs.append(torch.view_as_real(torch.view_as_complex((unit * w).view(*x.shape[:3], hd // 2, 2)) * turn).reshape(x.shape))
        if c["train"]:
            back = torch.view_as_real(torch.view_as_complex(dy.reshape(*x.shape[:3], hd // 2, 2)) * turn.conj()).reshape(x.shape)
            grads.append((back * w - unit * (back * w * unit).sum(-1, keepdim=True) / hd) / norm)
            dws.append((back * unit).sum((0, 1, 2)))
    out = {"out": torch.cat((*outs, v), dim=2).view(B, S, -1)}
    if c["train"]:
        out.update(dqkv=torch.cat((*grads, dv), dim=2).view(B, S, -1), dwq=dws[0], dwk=dws[1])
    return out
