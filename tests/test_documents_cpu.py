"""Attention within documents, norms of query and key heads, the loss from the output projection and starts of documents on the CPU:
the formulas against other formulas and differences, and what is refused."""

import pytest
import torch
import torch.nn.functional as F

from templar_b200 import ops


def normal(seed, *shape, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float32).to(dtype)


STARTS = torch.tensor([[0, 0, 0, 3, 3, 5, 5, 5, 9], [-4, 0, 1, 2, 3, 4, 5, 9, 9]])


def by_hand(qkv, starts, H, KV, hd):
    """Row by row."""
    B, S, _ = qkv.shape
    q, k, v = qkv[..., :H * hd].view(B, S, H, hd), qkv[..., H * hd:(H + KV) * hd].view(B, S, KV, hd), qkv[..., (H + KV) * hd:].view(B, S, KV, hd)
    out = torch.zeros(B, S, H, hd, dtype=qkv.dtype)
    for b in range(B):
        for s in range(S):
            a = max(int(starts[b, s]), 0)
            if a > s:
                continue
            for h in range(H):
                z = k[b, a:s + 1, h // (H // KV)] @ q[b, s, h] / hd ** 0.5
                out[b, s, h] = torch.softmax(z, 0) @ v[b, a:s + 1, h // (H // KV)]
    return out.view(B, S, H * hd)


@pytest.mark.parametrize("H,KV,hd", [(2, 2, 4), (4, 2, 6), (3, 1, 5)])
def test_attention_documents_formula(H, KV, hd):
    qkv = normal(1, 2, 9, (H + 2 * KV) * hd, dtype=torch.float32)
    torch.testing.assert_close(ops.attention_documents(qkv, STARTS, H, KV, hd), by_hand(qkv, STARTS, H, KV, hd), rtol=1e-5, atol=1e-6)


def test_attention_documents_gradient():
    """Against the gradient of the same attention over each document alone, and zero where nothing is seen."""
    H, KV, hd = 2, 1, 4
    qkv = normal(2, 1, 9, (H + 2 * KV) * hd, dtype=torch.float32).requires_grad_()
    starts = torch.tensor([[0, 0, 0, 3, 3, 3, 3, 9, 9]], dtype=torch.int32)
    dout = normal(3, 1, 9, H * hd, dtype=torch.float32)
    (got,) = torch.autograd.grad(ops.attention_documents(qkv, starts, H, KV, hd), qkv, dout)
    want = torch.zeros_like(qkv)
    for a, b in ((0, 3), (3, 7)):
        part = qkv.detach()[:, a:b].clone().requires_grad_()
        q, k, v = part[..., :8].view(1, b - a, 2, 4), part[..., 8:12].view(1, b - a, 1, 4), part[..., 12:].view(1, b - a, 1, 4)
        o = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2).expand(1, 2, -1, -1), v.transpose(1, 2).expand(1, 2, -1, -1),
                                           is_causal=True).transpose(1, 2).reshape(1, b - a, 8)
        (want[:, a:b],) = torch.autograd.grad(o, part, dout[:, a:b])
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)


def test_attention_documents_refusals():
    qkv, st = torch.zeros(2, 5, 16), torch.zeros(2, 5, dtype=torch.int32)
    ops.attention_documents(qkv, st, 2, 1, 4)
    for bad in (lambda: ops.attention_documents(qkv, st, 2, 2, 4), lambda: ops.attention_documents(qkv, st, 3, 2, 4),
                lambda: ops.attention_documents(qkv[0], st, 2, 1, 4), lambda: ops.attention_documents(qkv, st[:1], 2, 1, 4),
                lambda: ops.attention_documents(qkv, st[:, :4], 2, 1, 4), lambda: ops.attention_documents(qkv, st.float(), 2, 1, 4),
                lambda: ops.attention_documents(qkv, st.bool(), 2, 1, 4), lambda: ops.attention_documents(qkv, st, 0, 1, 4),
                lambda: ops.attention_documents(qkv, st.to("meta"), 2, 1, 4), lambda: ops.attention_documents(qkv, st, 2, 0, 4)):
        with pytest.raises(ValueError):
            bad()
    assert ops.attention_documents(qkv[:, :0], st[:, :0], 2, 1, 4).shape == (2, 0, 8)


def test_document_starts():
    tokens = torch.tensor([[5, 6, 2, 7, 2, 2, 8, 9], [2, 1, 1, 1, 1, 1, 1, 2]])
    st = ops.document_starts(tokens, 2)
    assert st.dtype == torch.int32 and st.tolist() == [[0, 0, 0, 3, 3, 5, 6, 6], [0, 1, 1, 1, 1, 1, 1, 1]]
    assert ops.document_starts(tokens, 2, window=3).tolist() == [[0, 0, 0, 3, 3, 5, 6, 6], [0, 1, 1, 1, 2, 3, 4, 5]]
    assert ops.document_starts(tokens, 2, window=1).tolist() == [list(range(8))] * 2
    assert ops.document_starts(tokens[:, :1], 2).tolist() == [[0], [0]]
    assert ops.document_starts(tokens[:, :0], 2).shape == (2, 0)
    with pytest.raises(ValueError):
        ops.document_starts(tokens[0], 2)


@pytest.mark.parametrize("pos", [False, True])
def test_qk_norm_rope_formula_and_gradient(pos):
    H, KV, hd, B, S = 3, 1, 6, 2, 5
    qkv, wq, wk = normal(1, B, S, (H + 2 * KV) * hd, dtype=torch.float32), normal(2, hd, dtype=torch.float32), normal(3, hd, dtype=torch.float32)
    cos, sin = ops.rope_tables(11, hd)
    at = torch.tensor([[0, 1, 0, 1, 10], [3, 4, 5, 0, 1]], dtype=torch.int32) if pos else None
    # norm by norm, then the framework's own rotation on sequences of one token each
    for t in (qkv, wq, wk):
        t.requires_grad_()
    got = ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, 1e-3, positions=at)
    x = qkv.view(B, S, H + 2 * KV, hd)
    parts = [x[:, :, h] * (x[:, :, h].square().mean(-1, keepdim=True) + 1e-3).rsqrt() * (wq if h < H else wk) for h in range(H + KV)]
    flat = torch.cat((*parts, x[:, :, H + KV:].flatten(2)), -1)
    rows = at.long() if pos else torch.arange(S).expand(B, S)
    want = torch.stack([torch.cat([ops.rope(flat[b:b + 1, s:s + 1], cos[rows[b, s]][None], sin[rows[b, s]][None], H + KV, hd)
                                   for s in range(S)], 1)[0] for b in range(B)])
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
    d = normal(4, *got.shape, dtype=torch.float32)
    for a, b in zip(torch.autograd.grad(got, (qkv, wq, wk), d), torch.autograd.grad(want, (qkv, wq, wk), d)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def test_qk_norm_rope_main_grad_and_refusals():
    H, KV, hd, B, S = 2, 1, 4, 1, 3
    qkv = normal(1, B, S, (H + 2 * KV) * hd, dtype=torch.float32)
    wq, wk = (normal(i, hd, dtype=torch.float32).requires_grad_() for i in (2, 3))
    cos, sin = ops.rope_tables(S, hd)
    out = ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd)
    gq, gk = torch.autograd.grad(out.sum(), (wq, wk))
    wq.main_grad, mk = torch.ones(hd), torch.zeros(hd)
    ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, main_grad_k=mk).sum().backward()
    assert wq.grad is None and wk.grad is None
    torch.testing.assert_close(wq.main_grad, 1 + gq)
    torch.testing.assert_close(mk, gk)
    call = lambda **k: ops.qk_norm_rope(**{**dict(qkv=qkv, wq=wq, wk=wk, cos=cos, sin=sin, n_heads=H, n_kv=KV, hd=hd), **k})  # noqa: E731
    for bad in (dict(hd=3), dict(n_heads=3), dict(wq=wq[:2]), dict(wk=torch.ones(5)), dict(cos=cos[:2], sin=sin[:2]), dict(cos=cos[:, :1]),
                dict(positions=torch.zeros(1, 2, dtype=torch.int32)), dict(positions=torch.zeros(1, 3)), dict(qkv=qkv[0]), dict(wk=wk.to("meta")),
                dict(cos=cos[:0], sin=sin[:0], positions=torch.zeros(1, 3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(**bad)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_linear_cross_entropy_formula_and_gradient(reduction):
    x, w = normal(1, 2, 4, 6, dtype=torch.float32).requires_grad_(), normal(2, 9, 6, dtype=torch.float32).requires_grad_()
    labels = torch.tensor([[0, 8, -100, 3], [2, -100, 7, 7]])
    got = ops.linear_cross_entropy(x, w, labels, reduction=reduction)
    want = F.cross_entropy((x @ w.t()).flatten(0, 1), labels.flatten(), reduction=reduction)
    want = want if reduction == "mean" else want.view(2, 4)
    torch.testing.assert_close(got, want)
    d = torch.rand(got.shape, generator=torch.Generator().manual_seed(0))
    g3 = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels, grad_scale=3.0, reduction=reduction), (x, w), d)
    for a, b in zip(g3, torch.autograd.grad(want, (x, w), 3 * d)):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)
    main = torch.ones_like(w)
    ops.linear_cross_entropy(x.detach(), w, labels, main_grad=main, reduction=reduction).sum().backward()
    assert w.grad is None
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels, reduction=reduction).sum(), (w,))
    torch.testing.assert_close(main, 1 + dw)


def test_linear_cross_entropy_edges_and_refusals():
    x, w, labels = torch.randn(5, 4, requires_grad=True), torch.randn(7, 4, requires_grad=True), torch.tensor([1, 2, 3, 4, 5])
    for none in (torch.full((5,), -100), torch.full((5,), 99)):
        loss = ops.linear_cross_entropy(x, w, none)
        assert loss.item() == 0 and not any(g.any() for g in torch.autograd.grad(loss, (x, w)))
    assert ops.linear_cross_entropy(x[:0], w, labels[:0], reduction="none").shape == (0,)
    assert ops.linear_cross_entropy(x[:0], w, labels[:0]).item() == 0

    class Shards:
        def accumulate(self, *a):
            pass

    for bad in (lambda: ops.linear_cross_entropy(x, w, labels[:4]), lambda: ops.linear_cross_entropy(x, w[:, :3], labels),
                lambda: ops.linear_cross_entropy(x, w[0], labels), lambda: ops.linear_cross_entropy(x, w, labels.float()),
                lambda: ops.linear_cross_entropy(x, w, labels, reduction="sum"), lambda: ops.linear_cross_entropy(x, w, labels.to("meta")),
                lambda: ops.linear_cross_entropy(x, w, labels, main_grad=Shards()), lambda: ops.linear_cross_entropy(x, w[:0], labels)):
        with pytest.raises(ValueError):
            bad()
