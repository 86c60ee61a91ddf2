"""Attention within documents, norms of query and key heads, and the loss from the output projection on the GPU, against the formulas in
64 bits.  A tolerance is made of the roundings on the way: U is a bf16 rounding, half a step, relative to the value."""

import pytest
import torch

from templar_b200 import ops
from templar_b200.ops import documents as OD
from templar_b200.ops import functional as OF
from templar_b200.ops import native

pytestmark = pytest.mark.gpu
U = torch.finfo(torch.bfloat16).eps / 2
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def close(got, want, bound, what):
    got, bad = got.double(), (got.double() - want).abs() - bound
    assert torch.isfinite(got).all(), what
    assert bad.max() <= 0, f"{what}: {int((bad > 0).sum())} of {bad.numel()} off, worst by {bad.max().item():.3g} beyond {bound.flatten()[bad.argmax()].item():.3g}"


# ------------------------------------------------------------------------------------------ attention
def starts_of(kind, B, S, g):
    rows = torch.arange(S, device=DEV, dtype=torch.int32).expand(B, S)
    if kind == "whole":
        return torch.zeros(B, S, dtype=torch.int32, device=DEV)
    if kind == "single":                                       # every token a document
        return rows.clone()
    if kind == "window":
        return rows - 99                                       # negative at the front
    if kind == "nothing":
        return torch.full((B, S), S, dtype=torch.int32, device=DEV)
    if kind == "any":                                          # any numbers, also behind the row and below zero
        return torch.randint(-S, 2 * S, (B, S), generator=g, device=DEV, dtype=torch.int32)
    if kind == "extremes":
        return torch.where(torch.rand(B, S, generator=g, device=DEV) < 0.5, -2 ** 31, 2 ** 31 - 1).to(torch.int32)
    ends = torch.rand(B, S, generator=g, device=DEV) < (1 / 40 if kind == "docs" else 1 / 500)
    st = torch.where(torch.roll(ends, 1, 1), rows, 0).cummax(1).values.to(torch.int32)
    if kind == "padded":
        st[:, S - S // 3:] = S
    return st


def attention64(qkv, starts, H, KV, hd, dout):
    """(out, bound), (dqkv, bound) by the formulas."""
    B, S, C = qkv.shape
    G = H // KV
    q, k, v = qkv.double().split([H * hd, KV * hd, KV * hd], dim=2)
    q, k, v = (t.view(B, S, -1, hd).transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(G, 1) for t in (k, v))
    do = dout.double().view(B, S, H, hd).transpose(1, 2)
    rows = torch.arange(S, device=DEV)
    seen = ((rows[None, None] <= rows[None, :, None]) & (rows[None, None] >= starts.long()[:, :, None]))[:, None]
    sc = hd ** -0.5
    z = (q @ k.transpose(2, 3) * sc).masked_fill(~seen, float("-inf"))
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(torch.isinf(top), 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    near = 1e-4                                                # fp32 scores and exponentials, relative to the weights
    out = p @ v
    eo = (U + near) * (p @ v.abs()) + U * out.abs()            # rounded weights, rounded output
    delta = (do * out).sum(-1, keepdim=True)
    ed = (do.abs() * eo).sum(-1, keepdim=True)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - delta) * sc
    es = U * ds.abs() + p * (ed + near * (do.abs() @ v.abs().transpose(2, 3) + delta.abs())) * sc
    dq, eq = ds @ k, es @ k.abs()
    dk, ek = ds.transpose(2, 3) @ q, es.transpose(2, 3) @ q.abs()
    dv, ev = p.transpose(2, 3) @ do, (U + near) * (p.transpose(2, 3) @ do.abs())
    shared = lambda t: t.view(B, KV, G, S, hd).sum(2)          # noqa: E731
    rowsof = lambda *ts: torch.cat([t.transpose(1, 2).reshape(B, S, -1) for t in ts], -1)  # noqa: E731
    grad = rowsof(dq, shared(dk), shared(dv))
    bound = rowsof(eq, shared(ek), shared(ev)) * 1.01 + U * grad.abs() + 1e-6
    return (rowsof(out), rowsof(eo) * 1.01 + 1e-6), (grad, bound)


ATTENTION = [
    (1, 1, 1, 1, 64, "whole"), (1, 1, 2, 1, 128, "nothing"), (3, 2, 4, 2, 64, "single"), (1, 60, 12, 12, 64, "docs"),
    (2, 127, 4, 4, 128, "docs"), (2, 128, 4, 2, 128, "single"), (2, 129, 4, 1, 64, "docs"), (2, 300, 6, 2, 128, "padded"),
    (2, 511, 6, 2, 64, "padded"), (1, 640, 4, 4, 128, "any"), (2, 385, 4, 4, 64, "any"), (2, 700, 2, 2, 64, "window"),
    (1, 1024, 8, 2, 128, "window"), (2, 260, 4, 4, 128, "nothing"), (2, 260, 4, 2, 64, "nothing"), (1, 1999, 3, 3, 64, "long"),
    (1, 1536, 5, 5, 128, "long"), (2, 300, 4, 2, 128, "extremes"), (2, 300, 4, 2, 64, "extremes"), (16, 130, 32, 8, 128, "docs"),
]


@pytest.mark.parametrize("B,S,H,KV,hd,kind", ATTENTION)
def test_attention_documents(B, S, H, KV, hd, kind):
    g = gen(S * 31 + H)
    qkv = normal(g, B, S, (H + 2 * KV) * hd, std=1.3).requires_grad_()
    dout = normal(g, B, S, H * hd, std=0.3)
    starts = starts_of(kind, B, S, g)
    out = ops.attention_documents(qkv, starts, H, KV, hd)
    (grad,) = torch.autograd.grad(out, qkv, dout)
    with torch.no_grad():
        alone = ops.attention_documents(qkv, starts, H, KV, hd)
    assert torch.equal(alone, out)
    (want, bound), (wgrad, gbound) = attention64(qkv.detach(), starts, H, KV, hd, dout)
    close(out.detach(), want, bound, "out")
    close(grad, wgrad, gbound, "gradient")
    empty = starts.long() > torch.arange(S, device=DEV)
    assert not out[empty].any() and not grad[..., :H * hd][empty].any()
    assert int(OF.status_word(DEV).item()) == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_whole_sequences_match_the_causal_kernels(hd):
    g = gen(5)
    qkv = normal(g, 2, 515, 6 * hd).requires_grad_()
    dout = normal(g, 2, 515, 4 * hd)
    a = OF._AttentionPacked.apply(qkv, 4, 1, hd)
    b = ops.attention_documents(qkv, torch.zeros(2, 515, dtype=torch.int64, device=DEV), 4, 1, hd)
    (da,), (db,) = torch.autograd.grad(a, qkv, dout), torch.autograd.grad(b, qkv, dout)
    # each is within its roundings of the formulas; the kernels walk the keys in another order, so the roundings are not the same ones
    (_, eo), (_, eg) = attention64(qkv.detach(), torch.zeros(2, 515, device=DEV), 4, 1, hd, dout)
    close(a.detach(), b.detach().double(), 2 * eo, "out")
    close(da, db.double(), 2 * eg, "gradient")


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_documents_gives_the_same_bits_every_time(hd):
    g = gen(6)
    qkv = normal(g, 3, 1100, 16 * hd).requires_grad_()
    dout = normal(g, 3, 1100, 8 * hd)
    starts = starts_of("long", 3, 1100, g)
    runs = []
    for _ in range(12):                                        # more tiles than CTAs, each CTA's warps a step apart at times
        out = ops.attention_documents(qkv, starts, 8, 4, hd)
        runs.append((out.detach(), *torch.autograd.grad(out, qkv, dout)))
    assert all(torch.equal(x, y) for r in runs[1:] for x, y in zip(r, runs[0]))


def test_attention_gradient_twice_and_of_a_sum():
    """The same graph differentiated again, and with a gradient that has no memory of its own (an expanded number)."""
    g = gen(14)
    qkv = normal(g, 40, 260, 4 * 64).requires_grad_()          # 240 tiles: every CTA takes several
    out = ops.attention_documents(qkv, starts_of("docs", 40, 260, g), 2, 1, 64)
    one = torch.ones((), dtype=torch.bfloat16, device=DEV).expand_as(out)
    first = torch.autograd.grad(out, qkv, one, retain_graph=True)[0]
    second = torch.autograd.grad(out.sum(dtype=torch.float32), qkv, retain_graph=True)[0]
    third = torch.autograd.grad(out, qkv, one.contiguous() * 2)[0]
    assert torch.equal(first, second) and torch.equal(first * 2, third)


@pytest.mark.parametrize("hd", [64, 128])
def test_packed_documents_are_the_documents_alone(hd):
    """Documents that begin at whole blocks meet the same tiles as in a sequence of their own, so their outputs have the same bits."""
    g = gen(9)
    H, KV, lens = 4, 2, (128, 384, 50)
    qkv = normal(g, 1, sum(lens), (H + 2 * KV) * hd)
    starts = torch.cat([torch.full((n,), sum(lens[:i]), dtype=torch.int32) for i, n in enumerate(lens)])[None].to(DEV)
    out = ops.attention_documents(qkv, starts, H, KV, hd)
    at = 0
    for n in lens:
        one = ops.attention_documents(qkv[:, at:at + n], torch.zeros(1, n, dtype=torch.int32, device=DEV), H, KV, hd)
        assert torch.equal(out[:, at:at + n], one)
        at += n


def test_attention_takes_views():
    g = gen(3)
    H, KV, hd, B, S = 4, 2, 64, 2, 150
    C = (H + 2 * KV) * hd
    wide = normal(g, B, S, C + 24)
    dout = normal(g, S, B, H * hd).transpose(0, 1)
    starts = starts_of("docs", B, S, g)
    plain = wide[..., 16:16 + C].contiguous().requires_grad_()
    ref = ops.attention_documents(plain, starts, H, KV, hd)
    (dref,) = torch.autograd.grad(ref, plain, dout.contiguous())
    views = [wide[..., 16:16 + C], wide[..., 16:16 + C].transpose(0, 1).contiguous().transpose(0, 1)]
    odd = torch.empty(B * S * C + 3, dtype=torch.bfloat16, device=DEV)[3:].view(B, S, C)
    views.append(odd.copy_(plain.detach()))
    for v in views:
        v = v.detach().requires_grad_()
        out = ops.attention_documents(v, starts.long().t().contiguous().t(), H, KV, hd)
        assert torch.equal(out, ref)
        (d,) = torch.autograd.grad(out, v, dout)
        torch.testing.assert_close(d.float(), dref.float(), rtol=2 * U, atol=1e-6)
        assert torch.equal(d[..., H * hd:], dref[..., H * hd:])


# ------------------------------------------------------------------------------------------ norm of heads
def qknorm64(qkv, wq, wk, cos, sin, at, H, KV, hd, eps, dy):
    B, S, C = qkv.shape
    R = H + KV
    x, d = qkv.double()[..., :R * hd].reshape(B, S, R, hd), dy.double()[..., :R * hd].reshape(B, S, R, hd)
    w = torch.cat((wq.double().expand(H, hd), wk.double().expand(KV, hd)))
    c, s = cos.double()[at][:, :, None], sin.double()[at][:, :, None]
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    z = x * r * w
    turn = lambda t, s: torch.stack((t[..., 0::2] * c - t[..., 1::2] * s, t[..., 0::2] * s + t[..., 1::2] * c), -1).view(B, S, R, hd)  # noqa: E731
    size = lambda t: turn(t.abs(), 0 * s) * 0 + (t[..., 0::2].abs() + t[..., 1::2].abs()).repeat_interleave(2, -1)  # noqa: E731
    out, near = turn(z, s), 2e-6                               # a few fp32 steps
    u = turn(d, -s)
    gr, xh = u * w, x * r
    m = (gr * xh).mean(-1, keepdim=True)
    dx = r * (gr - xh * m)
    ex = near * r * (size(d) * w.abs() + xh.abs() * (size(d) * w.abs() * xh.abs()).mean(-1, keepdim=True))
    dw, ew = (u * xh).sum((0, 1)), (1e-5 * (size(d) * xh.abs())).sum((0, 1))       # a sum in fp32
    flat = lambda t: t.reshape(B, S, R * hd)                   # noqa: E731
    return (flat(out), U * flat(out).abs() + near * flat(size(z))), (flat(dx), U * flat(dx).abs() + 4 * flat(ex) + 1e-30), \
        [(dw[a:b].sum(0), U * dw[a:b].sum(0).abs() + ew[a:b].sum(0)) for a, b in ((0, H), (H, R))]


@pytest.mark.parametrize("B,S,H,KV,hd,pos", [
    (1, 1, 12, 12, 64, False), (1, 1, 1, 1, 8, True), (2, 7, 10, 5, 80, True), (3, 77, 3, 1, 128, False), (2, 130, 16, 16, 128, True),
    (1, 33, 5, 5, 256, True), (2, 19, 7, 7, 96, False), (1, 50, 9, 3, 40, True), (1, 3, 4, 2, 200, True), (5, 1, 32, 8, 128, True),
    (2, 700, 32, 8, 128, True), (1, 2500, 12, 12, 64, False)])
def test_qk_norm_rope(B, S, H, KV, hd, pos):
    g = gen(hd + S)
    qkv = normal(g, B, S, (H + 2 * KV) * hd)
    qkv[..., ::7] *= 9
    qkv[0, 0, :hd] = 0                                         # a head of zeros
    qkv.requires_grad_()
    wq, wk = (normal(g, hd).requires_grad_() for _ in range(2))
    cos, sin = ops.rope_tables(S + 9, hd, device=DEV)
    at = torch.randint(0, S + 9, (B, S), generator=g, device=DEV) if pos else torch.arange(S, device=DEV).expand(B, S)
    dy = normal(g, B, S, (H + 2 * KV) * hd)
    out = ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, 1e-5, positions=at.to(torch.int32) if pos else None)
    dx, dwq, dwk = torch.autograd.grad(out, (qkv, wq, wk), dy)
    R = (H + KV) * hd
    (w1, b1), (w2, b2), dws = qknorm64(qkv.detach(), wq.detach(), wk.detach(), cos, sin, at, H, KV, hd, 1e-5, dy)
    close(out.detach()[..., :R], w1, b1 + 1e-30, "out")
    close(dx[..., :R], w2, b2, "dx")
    for got, (want, bound), name in zip((dwq, dwk), dws, ("dwq", "dwk")):
        close(got, want, bound, name)
    assert torch.equal(out[..., R:], qkv[..., R:]) and torch.equal(dx[..., R:], dy[..., R:])
    with torch.no_grad():
        assert torch.equal(ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, 1e-5, positions=at if pos else None), out)
    again = torch.autograd.grad(ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, 1e-5, positions=at if pos else None), (qkv, wq, wk), dy)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dwq, dwk)))
    assert int(OF.status_word(DEV).item()) == 0


def test_qk_norm_rope_views_main_grad_and_bad_positions():
    g = gen(1)
    B, S, H, KV, hd = 2, 40, 4, 2, 64
    C = (H + 2 * KV) * hd
    wide = normal(g, B, S, C + 40)
    x = wide[..., 8:8 + C].detach().requires_grad_()
    dense = x.detach().contiguous().requires_grad_()
    wq, wk = (normal(g, hd).requires_grad_() for _ in range(2))
    cos, sin = ops.rope_tables(S, hd, device=DEV)
    dy = normal(g, S, B, C).transpose(0, 1)
    a, b = (ops.qk_norm_rope(t, wq, wk, cos, sin, H, KV, hd) for t in (x, dense))
    assert torch.equal(a, b)
    ga, gb = (torch.autograd.grad(o, (t, wq, wk), d) for o, t, d in ((a, x, dy), (b, dense, dy.contiguous())))
    assert all(torch.equal(s, t) for s, t in zip(ga, gb))
    mq, mk = torch.full((hd,), 3.0, device=DEV), torch.full((hd,), 5.0, device=DEV)
    out = ops.qk_norm_rope(dense, wq, wk, cos, sin, H, KV, hd, main_grad_q=mq, main_grad_k=mk)
    (dx,) = torch.autograd.grad(out, (dense,), dy, retain_graph=True)
    out.backward(dy)
    assert wq.grad is None and wk.grad is None
    torch.testing.assert_close(mq, 3 + 2 * gb[1].float(), rtol=2 * U, atol=1e-3)
    torch.testing.assert_close(mk, 5 + 2 * gb[2].float(), rtol=2 * U, atol=1e-3)
    word = OF.status_word(DEV)
    assert int(word.item()) == 0
    far = torch.full((B, S), S, dtype=torch.int32, device=DEV)
    far[0, 0] = -1
    edge = far.clamp(0, S - 1)
    try:
        with torch.no_grad():
            got = ops.qk_norm_rope(dense, wq, wk, cos, sin, H, KV, hd, positions=far)
            assert int(word.item()) == 1                       # TPLR_ST_BAD_INDEX
            assert torch.equal(got, ops.qk_norm_rope(dense, wq, wk, cos, sin, H, KV, hd, positions=edge))
    finally:
        word.zero_()


# ------------------------------------------------------------------------------------------ loss
def loss64(x, w, labels, ignore=-100):
    """(losses, bound), d logits of the sum, bound of d: by the formulas."""
    xd, wd = x.double(), w.double()
    V, D = wd.shape
    z = xd @ wd.t()
    # fp32 sums of products of 16 in the tensor cores: one step for each of them
    ez = (D / 16 + 2) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()).amax(1, keepdim=True)
    counts = ((labels != ignore) & (labels >= 0) & (labels < V))[:, None]
    at = labels.clamp(0, V - 1)[:, None]
    lse = torch.logsumexp(z, 1, keepdim=True)
    losses = torch.where(counts, lse - z.gather(1, at), 0.0)
    el = 2 * ez + 4 * 2.0 ** -23 * (lse.abs() + z.gather(1, at).abs() + 8)
    p = torch.exp(z - lse)
    d = p.scatter_add(1, at, -torch.ones_like(lse)) * counts
    # the products take every weight rounded, times a row of x times the row's factor, rounded: (1 + U)^2 - 1 < 2.02 U, in the label's
    # column too, whose weight is made from exp(z - lse) - 1 in fp32
    ed = (2.02 * U + 2 * ez + 1e-5) * p
    ed = ed.scatter(1, at, (2.02 * U * d.gather(1, at).abs() + (2 * ez + 1e-5) * p.gather(1, at) + 2.0 ** -22)) * counts
    return (losses[:, 0], (el * counts)[:, 0] + 1e-30), d, ed, counts.sum()


def rows_and_labels(g, T, D, V, ignored=0.1):
    w = normal(g, V, D, std=2 * D ** -0.5)
    labels = torch.randint(0, V, (T,), generator=g, device=DEV)
    x = torch.randn(T, D, generator=g, device=DEV) + 4 * torch.rand(T, 1, generator=g, device=DEV) * w[labels].float()
    labels[torch.rand(T, generator=g, device=DEV) < ignored] = -100
    return x.to(torch.bfloat16), w, labels


LOSS = [(1, 8, 1), (1, 64, 7), (3, 16, 8), (30, 768, 1000), (128, 64, 129), (129, 200, 513), (257, 128, 2000), (700, 256, 5003), (1111, 1000, 1237),
        (2048, 64, 640), (300, 512, 32000)]


def check_loss(x, w, labels, chunk=None):
    (want, el), d, ed, n = loss64(x.detach(), w.detach(), labels)
    n = n.clamp(min=1)
    loss = ops.linear_cross_entropy(x, w, labels)
    dx, dw = torch.autograd.grad(loss, (x, w))
    close(loss.detach()[None], want.sum()[None] / n, el.sum()[None] / n + 1e-12, "loss")
    xd, wd = x.detach().double(), w.detach().double()
    for got, ref, b in ((dx, d @ wd / n, ed @ wd.abs() / n), (dw, d.t() @ xd / n, ed.t() @ xd.abs() / n)):
        more = (ref.abs() + b) * 0 + 2.0 ** -18 * ((d.abs() @ wd.abs()) if got is dx else (d.abs().t() @ xd.abs())) / n      # fp32 sums
        close(got, ref, 1.02 * b + U * ref.abs() + more + 1e-30, "dx" if got is dx else "dw")
    with torch.no_grad():
        each = ops.linear_cross_entropy(x, w, labels, reduction="none")
        mean = ops.linear_cross_entropy(x, w, labels)
    close(each, want, el, "losses")
    close(mean[None], want.sum()[None] / n, el.sum()[None] / n + 1e-12, "loss alone")
    return dx, dw


@pytest.mark.parametrize("T,D,V", LOSS)
def test_linear_cross_entropy(T, D, V):
    g = gen(T + V)
    x, w, labels = rows_and_labels(g, T, D, V)
    labels[0] = V - 1
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = check_loss(x, w, labels)
    again = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), (x, w))
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    assert not dx[labels == -100].any()
    assert int(OF.status_word(DEV).item()) == 0


def test_loss_in_several_runs_of_tokens(monkeypatch):
    g = gen(8)
    x, w, labels = rows_and_labels(g, 1300, 128, 3001)
    x.requires_grad_()
    w.requires_grad_()
    monkeypatch.setattr(OD, "CHUNK_BYTES", 2 * 3001 * 300)
    assert len(OD._chunks(1300, 3001)) > 3
    check_loss(x, w, labels)


def test_loss_gradients_of_single_tokens():
    g = gen(4)
    T, D, V = 333, 264, 1501
    x, w, labels = rows_and_labels(g, T, D, V)
    x.requires_grad_()
    w.requires_grad_()
    by = torch.randn(9, 37, generator=g, device=DEV)
    each = ops.linear_cross_entropy(x.view(9, 37, D), w, labels.view(9, 37), reduction="none", grad_scale=2.0)
    assert each.shape == (9, 37)
    dx, dw = torch.autograd.grad(each, (x, w), by)
    _, d, ed, _ = loss64(x.detach(), w.detach(), labels)
    k = 2 * by.double().reshape(-1, 1)
    xd, wd = x.detach().double(), w.detach().double()
    d, ed = d * k, (ed + U * 0) * k.abs()
    close(dx, d @ wd, 1.02 * (ed @ wd.abs()) + U * (d @ wd).abs() + 2.0 ** -18 * (d.abs() @ wd.abs()), "dx")
    close(dw, d.t() @ xd, 1.02 * (ed.t() @ xd.abs()) + U * (d.t() @ xd).abs() + 2.0 ** -18 * (d.abs().t() @ xd.abs()), "dw")


def test_loss_scales_main_grad_and_graph_use():
    g = gen(6)
    x, w, labels = rows_and_labels(g, 200, 64, 777)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), (x, w))
    loss = ops.linear_cross_entropy(x, w, labels, grad_scale=4.0)
    d4 = torch.autograd.grad(loss * 0.5, (x, w), retain_graph=True)
    d8 = torch.autograd.grad(loss, (x, w))                     # a second time from the same graph
    for one, two, four in zip((dx, dw), d4, d8):
        assert torch.equal(one * 2, two) and torch.equal(one * 4, four)
    main = torch.full((777, 64), 0.25, device=DEV)
    loss = ops.linear_cross_entropy(x, w, labels, main_grad=main)
    assert (main == 0.25).all()                                # nothing is added before the backward pass
    loss.backward()
    assert w.grad is None
    torch.testing.assert_close(main - 0.25, dw.float(), rtol=2 * U, atol=1e-7)
    fixed = w.detach()
    (only,) = torch.autograd.grad(ops.linear_cross_entropy(x, fixed, labels), (x,))
    assert torch.equal(only, dx)
    (only,) = torch.autograd.grad(ops.linear_cross_entropy(x.detach(), w, labels), (w,))
    assert torch.equal(only, dw)


@pytest.mark.parametrize("chunk", [OD.CHUNK_BYTES, 2 * 777 * 300])          # dw in bf16, of several runs in fp32
def test_gradients_that_the_loss_made_belong_to_one_call(chunk, monkeypatch):
    monkeypatch.setattr(OD, "CHUNK_BYTES", chunk)
    g = gen(61)
    x, w, labels = rows_and_labels(g, 600, 64, 777)
    x.requires_grad_()
    w.requires_grad_()
    one = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), (x, w))
    kept = [t.clone() for t in one]
    loss = ops.linear_cross_entropy(x, w, labels)
    first = torch.autograd.grad(loss, (x, w), grad_outputs=loss.new_tensor(0.25), retain_graph=True)
    second = torch.autograd.grad(loss, (x, w), grad_outputs=loss.new_tensor(0.5), retain_graph=True)
    node = loss.grad_fn(loss.new_tensor(0.5))                  # called by hand: nothing says that the graph goes
    assert all(torch.equal(a, b) for a, b in zip(node[:2], second))
    third = torch.autograd.grad(loss, (x, w))
    for k, o, a, b, c in zip(kept, one, first, second, third):
        assert torch.equal(k, o) and torch.equal(a * 4, k) and torch.equal(b * 2, k) and torch.equal(c, k)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (x, w))                      # the graph is gone
    for times in (1, 2, 3):
        (2 * ops.linear_cross_entropy(x, w, labels)).backward()          # .grad gathers, and is nobody else's
        if times == 1:
            assert torch.equal(x.grad, 2 * kept[0]) and torch.equal(w.grad, 2 * kept[1])
    for t, k in ((x, kept[0]), (w, kept[1])):
        # two sums, rounded to bf16 each: 1 + U of 4 and of 6 times the gradient
        close(t.grad, 6 * k.double(), 2.01 * U * 6 * k.abs().double(), "grad")


def test_loss_without_labels_far_logits_and_bad_labels():
    g = gen(7)
    x, w, labels = rows_and_labels(g, 150, 64, 500)
    x.requires_grad_()
    w.requires_grad_()
    none = torch.full_like(labels, -100)
    loss = ops.linear_cross_entropy(x, w, none)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert loss.item() == 0 and not dx.any() and not dw.any()
    big = (x.detach() * 200).requires_grad_()                  # logits of thousands: all weights but a few are zero
    check_loss(big, w, labels)
    word = OF.status_word(DEV)
    assert int(word.item()) == 0
    bad = labels.clone()
    bad[5], bad[6] = 500, -7
    same = labels.clone()
    same[5] = same[6] = -100
    try:
        a, b = (torch.autograd.grad(ops.linear_cross_entropy(x, w, t), (x, w)) for t in (bad, same))
        assert int(word.item()) == 1                           # TPLR_ST_BAD_INDEX
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    finally:
        word.zero_()


@pytest.mark.parametrize("shift,some", [(100.0, False), (-100.0, False), (90.0, True), (-90.0, True)])
def test_loss_of_logits_far_from_zero(shift, some):
    """All logits, or every fifth run of 200 columns, moved far away: pieces of several references in a row."""
    g = gen(21)
    x, w, labels = rows_and_labels(g, 270, 72, 2000)
    x[:, 0] = 10
    far = torch.arange(2000, device=DEV) // 200 % 5 == 2 if some else torch.ones(2000, dtype=torch.bool, device=DEV)
    w[:, 0] = torch.where(far, shift / 10, 0.0)
    x.requires_grad_()
    w.requires_grad_()
    check_loss(x, w, labels)


@pytest.mark.parametrize("shift", [0.0, 95.0, -95.0])
@pytest.mark.parametrize("T,D,V", [(1, 8, 1), (1, 2048, 257), (2, 72, 31), (15, 64, 33), (17, 200, 32000), (33, 768, 255), (64, 128, 512), (80, 136, 3001), (97, 1000, 50257),
                                   (127, 64, 4097), (128, 264, 20000)])
def test_losses_of_few_tokens(T, D, V, shift):
    """Scoring without a gradient: up to 128 tokens take the product with the weight's rows along the tile."""
    g = gen(3 * T + V)
    x, w, labels = rows_and_labels(g, T, D, V)
    if T > 2:
        labels[0], labels[1], labels[2] = V - 1, 0, -100
    x[:, 0] = 10
    w[:, 0] = torch.where(torch.arange(V, device=DEV) // 40 % 3 == 1, shift / 10, 0.0)        # pieces of several references in a row
    (want, el), *_ = loss64(x, w, labels)
    each = ops.linear_cross_entropy(x, w, labels, reduction="none")
    close(each, want, el, "losses")
    assert torch.equal(each, ops.linear_cross_entropy(x.clone(), w, labels, reduction="none"))
    if T > 2:
        x[2] = float("nan")                                    # a token that does not count, and whose neighbours do
        assert torch.equal(each, ops.linear_cross_entropy(x, w, labels, reduction="none"))
        x[1] = float("nan")
        got = ops.linear_cross_entropy(x, w, labels, reduction="none")
        assert got[1].isnan() and torch.equal(got[2:], each[2:]) and torch.equal(got[:1], each[:1])
    assert int(OF.status_word(DEV).item()) == 0


def test_losses_in_runs_of_which_the_last_is_short(monkeypatch):
    g = gen(31)
    x, w, labels = rows_and_labels(g, 600, 64, 700)
    want = ops.linear_cross_entropy(x, w, labels, reduction="none")
    monkeypatch.setattr(OD, "CHUNK_BYTES", 1)                  # runs of 256, 256 and 88
    got = ops.linear_cross_entropy(x, w, labels, reduction="none")
    (_, el), *_ = loss64(x, w, labels)
    close(got, want.double(), 2 * el, "losses")


def test_rows_that_count_for_nothing_may_hold_anything():
    g = gen(22)
    x, w, labels = rows_and_labels(g, 140, 64, 900)
    labels[7] = labels[8] = -100
    nan = x.clone()
    nan[7], nan[8] = float("nan"), float("inf")
    got, want = [], []
    for t, out in ((nan, got), (x, want)):
        t.requires_grad_()
        w.requires_grad_()
        loss = ops.linear_cross_entropy(t, w, labels)
        out += [loss, *torch.autograd.grad(loss, (t, w)), ops.linear_cross_entropy(t, w, labels, reduction="none")]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_loss_of_one_row_and_of_a_class_that_is_ignored():
    g = gen(13)
    x, w, labels = rows_and_labels(g, 50, 64, 129, ignored=0)
    labels[::2] = 3
    one = ops.linear_cross_entropy(x[1], w, labels[1])         # a row without a batch, a label without a dimension
    assert one.shape == () and torch.equal(one, ops.linear_cross_entropy(x[1:2], w, labels[1:2]))
    assert torch.equal(ops.linear_cross_entropy(x[1], w, labels[1], reduction="none"), one)
    x.requires_grad_()
    w.requires_grad_()
    other = torch.where(labels == 3, -100, labels)
    for reduction in ("mean", "none"):
        a, b = ops.linear_cross_entropy(x, w, labels, ignore_index=3, reduction=reduction), ops.linear_cross_entropy(x, w, other, reduction=reduction)
        assert torch.equal(a, b)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(a.sum(), (x, w)), torch.autograd.grad(b.sum(), (x, w))))
    assert int(OF.status_word(DEV).item()) == 0


def test_loss_takes_views():
    g = gen(12)
    x, w, labels = rows_and_labels(g, 90, 72, 333)
    want = ops.linear_cross_entropy(x, w, labels, reduction="none")
    wide = torch.zeros(90, 100, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:77] = x
    for xv, wv in ((wide[:, 5:77], w), (x.t().contiguous().t(), w.t().contiguous().t()), (x[:, None].expand(90, 1, 72)[:, 0], w)):
        assert torch.equal(ops.linear_cross_entropy(xv, wv, labels.to(torch.int32), reduction="none"), want)


# ------------------------------------------------------------------------------------------ together, captured, on other streams
def training_step(qkv, starts, positions, wq, wk, cos, sin, w, labels, H, KV, hd):
    """The operators one behind the other, as a block and the model's end call them; gradients of everything."""
    q = ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, positions=positions)
    x = ops.attention_documents(q, starts, H, KV, hd)
    loss = ops.linear_cross_entropy(x, w, labels)
    grads = torch.autograd.grad(loss, (qkv, wq, wk, w))
    return (loss.detach(), *grads)       # no graph of these leaves is left alive when another one is captured


def step_inputs(seed, B=2, S=300, H=4, KV=2, hd=64, V=1003):
    g = gen(seed)
    cos, sin = ops.rope_tables(S, hd, device=DEV)
    starts = starts_of("docs", B, S, g)
    labels = torch.randint(0, V, (B, S), generator=g, device=DEV)
    labels[:, ::9] = -100
    t = dict(qkv=normal(g, B, S, (H + 2 * KV) * hd), wq=normal(g, hd), wk=normal(g, hd), w=normal(g, V, H * hd, std=0.1))
    return dict({k: v.requires_grad_() for k, v in t.items()}, starts=starts, positions=torch.arange(S, device=DEV, dtype=torch.int32) - starts,
                cos=cos, sin=sin, labels=labels), (H, KV, hd)


@pytest.mark.parametrize("H,KV,hd", [(4, 2, 64), (2, 1, 128)])
def test_the_operators_together(H, KV, hd):
    a, _ = step_inputs(31, H=H, KV=KV, hd=hd)
    got = training_step(**a, H=H, KV=KV, hd=hd)
    # the same in fp64 by the formulas that run where no kernel does
    b = {k: v.detach().double().requires_grad_(v.requires_grad) if v.is_floating_point() else v for k, v in a.items()}
    q = OD._qk_norm_rope_torch(b["qkv"], b["wq"], b["wk"], b["cos"], b["sin"], b["positions"], H, KV, hd, 1e-5)
    x = OD._attention_documents_torch(q, b["starts"], H, KV, hd)
    loss = OD._linear_cross_entropy_torch(x, b["w"], b["labels"].reshape(-1), 1.0, -100, "mean")
    want = (loss, *torch.autograd.grad(loss, (b["qkv"], b["wq"], b["wk"], b["w"])))
    torch.testing.assert_close(got[0].double(), want[0].double(), rtol=1e-3, atol=0)
    # roundings on the way to a gradient: the rotated rows, the outputs, the weights and products of three operators, ten of U / 2 at most on
    # average, added in squares
    for x, y in zip(got[1:], want[1:]):
        assert (x.double() - y.double()).norm() <= 10 ** 0.5 * U * y.double().norm()


def test_captured_and_replayed():
    a, (H, KV, hd) = step_inputs(41)
    other, _ = step_inputs(42)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            training_step(**a, H=H, KV=KV, hd=hd)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):                                         # two graphs with workspaces of their own
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(training_step(**a, H=H, KV=KV, hd=hd))
    for data in (other, a, other):
        with torch.no_grad():
            for k, v in data.items():
                a[k].copy_(v) if data is not a else None
        want = training_step(**a, H=H, KV=KV, hd=hd)
        for g in graphs + graphs:
            g.replay()
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_two_streams_at_once():
    a, (H, KV, hd) = step_inputs(51)
    b, _ = step_inputs(52, S=411)
    want = [training_step(**t, H=H, KV=KV, hd=hd) for t in (a, b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(5):
        for i, (s, t) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i] = training_step(**t, H=H, KV=KV, hd=hd)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_offsets_beyond_32_bits():
    """33 sequences of 8192 rows of 8192 columns: the last sequence as if it were alone."""
    B, S, H, KV, hd = 33, 8192, 32, 16, 128
    g = gen(61)
    qkv = torch.empty(B, S, (H + 2 * KV) * hd, dtype=torch.bfloat16, device=DEV).normal_(generator=g).requires_grad_()
    assert qkv.numel() > 2 ** 31
    starts = starts_of("long", B, S, g)
    wq, wk = (normal(g, hd).requires_grad_() for _ in range(2))
    cos, sin = ops.rope_tables(S, hd, device=DEV)
    dout = torch.empty(B, S, H * hd, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    rows = ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd)
    out = ops.attention_documents(rows, starts, H, KV, hd)
    (grad,) = torch.autograd.grad(out, qkv, dout)
    last = qkv.detach()[-1:].clone().requires_grad_()
    one = ops.attention_documents(ops.qk_norm_rope(last, wq, wk, cos, sin, H, KV, hd), starts[-1:], H, KV, hd)
    (gone,) = torch.autograd.grad(one, last, dout[-1:])
    assert torch.equal(out[-1:], one) and torch.equal(grad[-1:, :, :H * hd], gone[..., :H * hd])
    # alone its groups' heads may be split over tiles, whose parts are added in fp32: another order
    torch.testing.assert_close(grad[-1:].float(), gone.float(), rtol=2 * U, atol=2 * U * gone.float().abs().mean().item())


def test_nodes_in_python_and_in_cpp_make_the_same_bits(monkeypatch):
    """Without the host library the same operators run as nodes in Python."""
    g = gen(71)
    H, KV, hd, B, S = 4, 2, 64, 2, 300
    qkv = torch.randn(B, S, (H + 2 * KV) * hd, generator=g, device=DEV).to(torch.bfloat16).requires_grad_()
    wq, wk = (torch.rand(hd, generator=g, device=DEV).to(torch.bfloat16).requires_grad_() for _ in range(2))
    cos, sin = OF.rope_tables(512, hd, device=DEV)
    ends = torch.rand(B, S, generator=g, device=DEV) < 0.02
    starts = torch.where(ends, torch.arange(S, device=DEV, dtype=torch.int32), 0).cummax(1).values.to(torch.int32)
    do = torch.randn(B, S, H * hd, generator=g, device=DEV).to(torch.bfloat16)
    x, w, labels = rows_and_labels(g, 600, 64, 777)
    x.requires_grad_()
    w.requires_grad_()

    def everything():
        z = ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd)
        out = ops.attention_documents(z, starts, H, KV, hd)
        made = [out, *torch.autograd.grad(out, (qkv, wq, wk), do)]
        with torch.no_grad():
            made += [ops.attention_documents(z, starts, H, KV, hd)]
            made += [ops.linear_cross_entropy(x[:n], w, labels[:n], reduction=r) for n in (20, 600) for r in ("mean", "none")]
        for n in (20, 600):
            loss = ops.linear_cross_entropy(x[:n], w, labels[:n])
            made += [loss, *torch.autograd.grad(3 * loss, (x, w))]
            each = ops.linear_cross_entropy(x[:n], w, labels[:n], reduction="none")
            made += [each, *torch.autograd.grad(each.sum(), (x, w))]
        return made

    cpp = everything()
    monkeypatch.setattr(native, "host", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(everything(), cpp))
    assert int(OF.status_word(DEV).item()) == 0
