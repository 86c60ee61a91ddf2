"""Operators on packed documents in uses that are easily got wrong: forward mode, one buffer for two weights, graphs walked more than once,
labels that the model is sure of.  On the CPU the formulas, on the GPU the kernels."""

import warnings

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from templar_b200 import ops
from templar_b200.ops import documents as OD
from templar_b200.ops import functional as OF
from templar_b200.ops import native

U = torch.finfo(torch.bfloat16).eps / 2
DEV = "cuda"


def normal(seed, *shape, std=1.0, device="cpu", dtype=torch.float32):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(device=device, dtype=dtype)


# ------------------------------------------------------------------------------------------ gradient buffers
@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
def test_buffers_that_are_not_the_weights_are_refused(device):
    """The kernels add by address: a buffer on another device or of another length must not reach them."""
    t = lambda seed, *shape: normal(seed, *shape, device=device, dtype=torch.bfloat16).requires_grad_()  # noqa: E731
    H, KV, hd, S, V, D = 2, 1, 64, 9, 300, 64
    elsewhere = "meta" if device == "cpu" else "cpu"
    qkv, wq, wk, x, w = t(1, 1, S, (H + 2 * KV) * hd), t(2, hd), t(3, hd), t(4, S, D), t(5, V, D)
    labels = torch.arange(S, device=device)
    cos, sin = ops.rope_tables(S, hd, device=device)
    norm = lambda **k: ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, **k)  # noqa: E731
    for bad in (torch.zeros(hd, device=elsewhere), torch.zeros(hd - 1, device=device), torch.zeros(2 * hd, device=device), torch.zeros(0, device=device),
                torch.zeros(hd, device=elsewhere, dtype=torch.bfloat16), type("Shards", (), {"accumulate": None})()):
        for name in ("main_grad_q", "main_grad_k"):
            with pytest.raises(ValueError, match="qk_norm_rope"):
                norm(**{name: bad})
        with torch.no_grad():                                  # nothing is added
            assert norm(main_grad_q=bad).shape == qkv.shape
    for bad in (torch.zeros(V, D, device=elsewhere), torch.zeros(V - 1, D, device=device), torch.zeros(V, D + 8, device=device),
                torch.zeros(0, device=device), torch.zeros(V, D, device=elsewhere, dtype=torch.bfloat16)):
        for reduction in ("mean", "none"):
            with pytest.raises(ValueError, match="main_grad"):
                ops.linear_cross_entropy(x, w, labels, main_grad=bad, reduction=reduction)
            with torch.no_grad():
                ops.linear_cross_entropy(x, w, labels, main_grad=bad, reduction=reduction)
            ops.linear_cross_entropy(x, w.detach(), labels, main_grad=bad, reduction=reduction).sum().backward()
    # of the weight's numbers in another shape or type is a buffer
    other, low = torch.zeros(D, V, device=device), torch.zeros(V, D, device=device, dtype=torch.bfloat16)
    (dw,) = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), w)
    for b in (other, low):
        ops.linear_cross_entropy(x.detach(), w, labels, main_grad=b).backward()
        torch.testing.assert_close(b.flatten().float(), dw.flatten().float(), rtol=2 * U, atol=1e-7)


def test_buffers_that_overlap_in_part_are_refused():
    H, KV, hd, S = 2, 1, 8, 5
    qkv, wq, wk = (normal(i, *s).requires_grad_() for i, s in ((1, (1, S, (H + 2 * KV) * hd)), (2, (hd,)), (3, (hd,))))
    cos, sin = ops.rope_tables(S, hd)
    long = torch.zeros(2 * hd)
    run = lambda a, b: ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, main_grad_q=a, main_grad_k=b)  # noqa: E731
    for i, j in ((0, 4), (1, 0), (7, 0)):
        with pytest.raises(ValueError, match="overlap"):
            run(long[i:i + hd], long[j:j + hd])
    run(long[:hd], long[hd:]).sum().backward()
    apart = long.clone()
    run(long[:hd], long[:hd]).sum().backward()
    torch.testing.assert_close(long[:hd], 2 * apart[:hd] + apart[hd:])


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
def test_buffers_in_each_others_gaps(device):
    H, KV, hd, S = 2, 1, 64, 90
    qkv, wq, wk = (normal(i, *s, device=device, dtype=torch.bfloat16).requires_grad_() for i, s in ((1, (1, S, (H + 2 * KV) * hd)), (2, (hd,)), (3, (hd,))))
    cos, sin = ops.rope_tables(S, hd, device=device)
    run = lambda **k: ops.qk_norm_rope(qkv, wq, wk, cos, sin, H, KV, hd, **k).float().square().sum()  # noqa: E731
    gq, gk = torch.autograd.grad(run(), (wq, wk))
    both = torch.zeros(hd, 2, device=device)
    run(main_grad_q=both[:, 0], main_grad_k=both[:, 1]).backward()
    assert torch.equal(both[:, 0].to(torch.bfloat16), gq) and torch.equal(both[:, 1].to(torch.bfloat16), gk)


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("B,S,H,KV,hd", [(1, 1, 1, 1, 8), (2, 700, 4, 2, 64), (1, 3000, 16, 4, 128), (1, 90, 5, 5, 256)])
def test_one_buffer_for_the_gradients_of_both_weights(B, S, H, KV, hd, host, monkeypatch):
    if not host:
        monkeypatch.setattr(native, "host", lambda: None)
    x = normal(1, B, S, (H + 2 * KV) * hd, device=DEV, dtype=torch.bfloat16).requires_grad_()
    w = normal(2, hd, device=DEV, dtype=torch.bfloat16).requires_grad_()
    cos, sin = ops.rope_tables(1, hd, device=DEV)
    at = torch.zeros(B, S, dtype=torch.int32, device=DEV)      # no angle, and gradients of the rows' own sign: every term of the sums is positive
    dy = torch.sign(x.detach())
    run = lambda wq, wk, mq, mk: ops.qk_norm_rope(x, wq, wk, cos, sin, H, KV, hd, positions=at, main_grad_q=mq, main_grad_k=mk).backward(dy)  # noqa: E731
    q, k = (torch.zeros(hd, device=DEV) for _ in range(2))
    other = w.detach().clone().requires_grad_()
    run(w, other, q, k)
    assert (q > 0).all() and (k > 0).all()
    first = None
    for _ in range(4):
        one, two = (torch.ones(hd, device=DEV) for _ in range(2))
        run(w, other, one, one)
        w.main_grad = two
        run(w, w, None, None)                                  # the buffer of one weight that serves both
        del w.main_grad
        assert torch.equal(one, two) and (first is None or torch.equal(one, first))
        first = one
    # both are sums of the same positive numbers, of less than 64 steps in fp32 for each thread and 32 behind them
    torch.testing.assert_close(first, 1 + q + k, rtol=96 * 2.0 ** -24, atol=0)
    (dw,) = torch.autograd.grad(ops.qk_norm_rope(x, w, w, cos, sin, H, KV, hd, positions=at), w, dy)
    torch.testing.assert_close(dw.float(), q + k, rtol=3 * U, atol=0)          # each of two gradients rounded, and their sum
    assert int(OF.status_word(DEV).item()) == 0


# ------------------------------------------------------------------------------------------ walks of one graph at the same time
@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("hd", [64, 128])
def test_walks_of_one_graph_that_overlap(hd, host, monkeypatch):
    """One kept graph of the attention walked on two streams at once, and by two captured backward passes replayed side by side: more tiles
    than CTAs, which each walk hands out by itself."""
    if not host:
        monkeypatch.setattr(native, "host", lambda: None)
    B, S, H, KV = 6, 900, 12, 4
    qkv = normal(1, B, S, (H + 2 * KV) * hd, device=DEV, dtype=torch.bfloat16).requires_grad_()
    starts = ops.document_starts(torch.randint(0, 200, (B, S), generator=torch.Generator().manual_seed(2)), 0).to(DEV)
    douts = [normal(3 + i, B, S, H * hd, device=DEV, dtype=torch.bfloat16) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        out = ops.attention_documents(qkv, starts, H, KV, hd)
        walk = lambda d: out.grad_fn(d) if callable(out.grad_fn) else out.grad_fn.apply(d)[0]  # noqa: E731
        want = [walk(d) for d in douts]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for s, d in zip(streams, douts):
            with torch.cuda.stream(s):
                got.append(walk(d))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)
    graphs, held = [], []
    for s, d in zip(streams, douts):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            held.append(walk(d))
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, w in zip(held, want):
            assert torch.equal(g, w)
    assert int(OF.status_word(DEV).item()) == 0


# ------------------------------------------------------------------------------------------ forward mode
def calls(device, dtype):
    """(operator of one operand, the operand) for every operand that has a derivative."""
    H, KV, hd, B, S, V = 4, 2, 64, 2, 70, 300
    t = lambda seed, *shape: normal(seed, *shape, std=0.5, device=device, dtype=dtype)  # noqa: E731
    qkv, wq, wk, x, w = t(1, B, S, (H + 2 * KV) * hd), t(2, hd), t(3, hd), t(4, B, S, 128), t(5, V, 128)
    starts = ops.document_starts(torch.randint(0, 9, (B, S), generator=torch.Generator().manual_seed(6)), 0).to(device)
    labels = torch.randint(0, V, (B, S), generator=torch.Generator().manual_seed(7)).to(device)
    cos, sin = ops.rope_tables(S, hd, device=device)
    norm = lambda **k: ops.qk_norm_rope(**{**dict(qkv=qkv, wq=wq, wk=wk, cos=cos, sin=sin, n_heads=H, n_kv=KV, hd=hd), **k})  # noqa: E731
    return {"attention": (lambda a: ops.attention_documents(a, starts, H, KV, hd), qkv),
            "norm of qkv": (lambda a: norm(qkv=a), qkv), "norm, wq": (lambda a: norm(wq=a), wq), "norm, wk": (lambda a: norm(wk=a), wk),
            "norm, tables": (lambda a: norm(cos=a), cos),
            "loss of x": (lambda a: ops.linear_cross_entropy(a, w, labels), x), "loss, w": (lambda a: ops.linear_cross_entropy(x, a, labels), w),
            "losses of x": (lambda a: ops.linear_cross_entropy(a, w, labels, reduction="none"), x),
            "losses, w": (lambda a: ops.linear_cross_entropy(x, a, labels, reduction="none"), w)}


NAMES = ["attention", "norm of qkv", "norm, wq", "norm, wk", "norm, tables", "loss of x", "loss, w", "losses of x", "losses, w"]


@pytest.mark.parametrize("name", NAMES)
def test_the_formulas_carry_a_tangent(name):
    op, a = calls("cpu", torch.float32)[name]
    v = normal(8, *a.shape)
    with fwAD.dual_level():
        tangent = fwAD.unpack_dual(op(fwAD.make_dual(a, v))).tangent
    a = a.clone().requires_grad_()
    out = op(a)
    d = normal(9, *out.shape)
    (g,) = torch.autograd.grad(out, a, d)
    # <d, J v> = <J^T d, v>: two sums in fp32, each off relative to the sizes of its terms
    torch.testing.assert_close((tangent * d).sum(), (g * v).sum(), rtol=1e-3, atol=1e-5 * float((tangent * d).abs().sum() + (g * v).abs().sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_the_kernels_refuse_a_tangent(name, host, monkeypatch):
    """A result without a tangent would read as a derivative of zero."""
    if not host:
        monkeypatch.setattr(native, "host", lambda: None)
    op, a = calls(DEV, torch.bfloat16)[name]
    plain = op(a)
    with fwAD.dual_level():
        dual = fwAD.make_dual(a, torch.ones_like(a))
        with pytest.raises(NotImplementedError, match="forward"):
            op(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
            op(dual)
        assert torch.equal(op(a), plain)                       # inside a level, of plain tensors
    other, b = calls(DEV, torch.float32)[name]                 # no kernel's type: the formulas
    with fwAD.dual_level():
        assert fwAD.unpack_dual(other(fwAD.make_dual(b, torch.ones_like(b)))).tangent is not None


# ------------------------------------------------------------------------------------------ graphs walked more than once
@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [OD.CHUNK_BYTES, 2 * 500 * 300])          # dw in bf16, of several runs in fp32
def test_a_captured_backward_pass_replayed_twice(chunk, monkeypatch):
    """The forward pass in one CUDA graph, the backward pass in another, as graphed callables have them: every replay of the second gives the
    gradient of the first's last replay."""
    monkeypatch.setattr(OD, "CHUNK_BYTES", chunk)
    x, w = (normal(i, n, 64, device=DEV, dtype=torch.bfloat16).requires_grad_() for i, n in ((1, 600), (2, 500)))
    labels = torch.randint(0, 500, (600,), generator=torch.Generator().manual_seed(3)).to(DEV)
    by = torch.full((), 0.5, device=DEV)
    want = [t.clone() for t in torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), (x, w), by)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), (x, w), by)
    side.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=side):
        loss = ops.linear_cross_entropy(x, w, labels)
    with torch.cuda.graph(backward, stream=side, pool=forward.pool()):
        got = torch.autograd.grad(loss, (x, w), by)
    del loss
    for _ in range(2):
        forward.replay()
        for _ in range(3):
            backward.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------ weights of one row
@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
def test_norm_weights_may_have_any_shape_of_their_numbers(host, monkeypatch):
    if not host:
        monkeypatch.setattr(native, "host", lambda: None)
    H, KV, hd, B, S = 4, 2, 64, 2, 70
    qkv, wq, wk = (normal(i, *s, device=DEV, dtype=torch.bfloat16).requires_grad_() for i, s in ((1, (B, S, (H + 2 * KV) * hd)), (2, (hd,)), (3, (hd,))))
    cos, sin = ops.rope_tables(S, hd, device=DEV)
    run = lambda a, b: torch.autograd.grad(ops.qk_norm_rope(qkv, a, b, cos, sin, H, KV, hd).float().square().sum(), (qkv, a, b))  # noqa: E731
    want = run(wq, wk)
    row, grid = wq.detach().view(1, hd).requires_grad_(), wk.detach().view(8, 8).requires_grad_()
    got = run(row, grid)
    assert got[1].shape == (1, hd) and got[2].shape == (8, 8)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------ labels that the model is sure of
def sure(T, D, V, far, seed=0):
    """x, w, labels: rows whose label has probabilities of one half to 1 - 1e-9; far: all logits moved by as much."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g)
    labels = torch.randint(0, V, (T,), generator=g)
    w = w / w.norm(dim=1, keepdim=True)
    x = w[labels] * torch.linspace(9, 36, T)[:, None]
    x[:, 0], w[:, 0] = 10, far / 10
    return x.to(DEV, torch.bfloat16), w.to(DEV, torch.bfloat16), labels.to(DEV)


def sure64(x, w, labels):
    """(losses, bound), d logits of their sum, its bound.  What is off is relative to 1 - p in the label's column, as to p in the others, so
    that the gradient of a label that is nearly certain has digits: 1 - p is formed in 64 bits from the other columns."""
    xd, wd = x.detach().double(), w.detach().double()
    z, at, D = xd @ wd.t(), labels[:, None], x.shape[1]
    # fp32 sums of products of 16 in the tensor cores, one step for each; exponents below 128 rounded to fp32, 128 ln 2 2^-24, and the exponential's own
    ez = (D / 16 + 2) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()).amax(1, keepdim=True)
    e = 2 * ez + 1e-5
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    others = z.scatter(1, at, float("-inf"))
    rest = torch.exp(torch.logsumexp(others, 1, keepdim=True) - lse)       # 1 - p of the label
    losses = torch.log1p(rest / p.gather(1, at))
    d = p.scatter(1, at, -rest)
    ed = (2.02 * U + e) * d.abs()                              # a weight rounded, a row times its factor rounded
    return (losses[:, 0], (e * rest + 2.0 ** -21 * losses)[:, 0]), d, ed, rest


@pytest.mark.gpu
@pytest.mark.parametrize("far", [0.0, 30.0, -30.0, 300.0, -1000.0])
@pytest.mark.parametrize("T,D,V", [(100, 64, 1000), (300, 128, 5003)])
def test_gradients_of_labels_that_are_nearly_certain(T, D, V, far):
    x, w, labels = sure(T, D, V, far)
    (want, el), d, ed, rest = sure64(x, w, labels)
    if far == 0:
        assert rest.min() < 1e-7 and rest.max() > 0.1
    x.requires_grad_()
    w.requires_grad_()
    xd, wd = x.detach().double(), w.detach().double()
    with torch.no_grad():
        each = ops.linear_cross_entropy(x, w, labels, reduction="none").double()
    assert ((each - want).abs() <= el).all(), ((each - want).abs() / el).max().item()
    # a row at a time: its label's column of dw is -(1 - p) x, whatever the others are
    for t in range(0, T, 7):
        loss = ops.linear_cross_entropy(x[t:t + 1], w, labels[t:t + 1])
        (dw,) = torch.autograd.grad(loss, w)
        assert (loss.double() - want[t]).abs() <= el[t] + 2.0 ** -23 * want[t]
        ref = d[t, :, None] * xd[t]
        off = (dw.double() - ref).abs() - (1.02 * ed[t, :, None] * xd[t].abs() + U * ref.abs() + 1e-30)
        assert off.max() <= 0, (t, rest[t].item(), off.max().item())
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, labels), (x, w))
    for got, ref, b, size in ((dx, d @ wd, ed @ wd.abs(), d.abs() @ wd.abs()), (dw, d.t() @ xd, ed.t() @ xd.abs(), d.abs().t() @ xd.abs())):
        off = (got.double() * T - ref).abs() - (1.02 * b + U * ref.abs() + 2.0 ** -18 * size + 1e-30)
        assert off.max() <= 0


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e3, 1e6, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("T", [40, 200])
def test_logits_of_any_size(T, size):
    """The largest logit's exponent ends at zero, however coarse fp32 is at its size: the loss is the distance of two logits."""
    x, w = normal(1, T, 64, std=size ** 0.5, device=DEV, dtype=torch.bfloat16), normal(2, 300, 64, std=size ** 0.5, device=DEV, dtype=torch.bfloat16)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    ez = (64 / 16 + 2) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()).amax(1)
    labels = z.argmax(1)
    labels[::2] = (labels[::2] + 1) % 300
    want = torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]
    got = ops.linear_cross_entropy(x, w, labels, reduction="none").double()
    bound = 2 * ez + 2.0 ** -21 * want + 2e-5                  # and whole references of logits: as the logits themselves
    assert ((got - want).abs() <= bound + 2.0 ** -22 * z.abs().amax(1)).all()
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, labels)
    assert (loss.double() - want.mean()).abs() <= (bound + 2.0 ** -22 * z.abs().amax(1)).mean()
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.isfinite().all() and dw.isfinite().all()
    top2 = z.topk(2, 1).values
    if size > 1e3 and ((top2[:, 0] - top2[:, 1]) > 4 * ez + 200).all():        # one column has all the weight
        d = torch.nn.functional.one_hot(z.argmax(1), 300).double() - torch.nn.functional.one_hot(labels, 300)
        ref = d @ wd / T
        assert ((dx.double() - ref).abs() <= 4 * U * (d.abs() @ wd.abs()) / T).all()


# ------------------------------------------------------------------------------------------ the formulas
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_rows_without_a_label_may_hold_anything_in_the_formulas_too(what, reduction):
    x, w, labels = normal(1, 6, 8), normal(2, 11, 8), torch.tensor([3, -100, 10, 99, 0, -100])
    results = []
    for fill in (0.5, what):
        a, b = x.clone(), w.clone().requires_grad_()
        a[1], a[3] = fill, fill                                # ignored, and no column
        a.requires_grad_()
        loss = ops.linear_cross_entropy(a, b, labels, reduction=reduction)
        results.append((loss, *torch.autograd.grad(loss.sum(), (a, b))))
    assert all(torch.equal(p, q) for p, q in zip(*results))


@pytest.mark.parametrize("window", [8, 9, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 5, 2 ** 40, 2 ** 70])
def test_windows_longer_than_the_sequence_leave_the_documents_whole(window):
    tokens = torch.tensor([[5, 6, 2, 7, 2, 2, 8, 9]])
    assert torch.equal(ops.document_starts(tokens, 2, window=window), ops.document_starts(tokens, 2))
    assert ops.document_starts(tokens[:, :0], 2, window=window).shape == (1, 0)


@pytest.mark.parametrize("device", ["cpu", pytest.param(DEV, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.uint32, torch.int64])
def test_starts_of_every_whole_type(dtype, device):
    H, KV, hd, S = 2, 1, 64, 140
    qkv = normal(1, 1, S, (H + 2 * KV) * hd, device=device, dtype=torch.bfloat16)
    starts = torch.arange(S, dtype=torch.int64)[None] // 10 * 10
    starts[:, 125:] = torch.iinfo(dtype).max                   # as behind the row as the type can say
    want = ops.attention_documents(qkv, starts.clamp(max=2 ** 31 - 1).to(torch.int32).to(device), H, KV, hd)
    got = ops.attention_documents(qkv, starts.to(dtype).to(device), H, KV, hd)
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        ops.attention_documents(qkv, starts.to(torch.uint64).to(device), H, KV, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,dtype", [(80, torch.bfloat16), (64, torch.float32)])
def test_attention_outside_the_kernels_is_said_once(hd, dtype, monkeypatch):
    monkeypatch.setattr(OD, "_fallback_seen", set())
    qkv, starts = normal(1, 2, 30, 4 * hd, device=DEV, dtype=dtype), torch.zeros(2, 30, dtype=torch.int32, device=DEV)
    with pytest.warns(UserWarning, match=f"attention_documents: heads of {hd}"):
        ops.attention_documents(qkv, starts, 2, 1, hd)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        ops.attention_documents(qkv, starts, 2, 1, hd)
        ops.attention_documents(qkv[:, :0], starts[:, :0], 2, 1, hd)
        own = normal(2, 2, 30, 4 * 64, device=DEV, dtype=torch.bfloat16)
        ops.attention_documents(own, starts, 2, 1, 64)
        ops.attention_documents(own.cpu(), starts.cpu(), 2, 1, 64)


# ------------------------------------------------------------------------------------------ a buffer and several runs of tokens
@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_buffer_takes_the_sum_of_several_runs(reduction, host, monkeypatch):
    if not host:
        monkeypatch.setattr(native, "host", lambda: None)
    T, D, V = 900, 72, 777
    monkeypatch.setattr(OD, "CHUNK_BYTES", 2 * V * 300)
    assert len(OD._chunks(T, V)) == 4
    x, w = (normal(i, n, D, std=0.4, device=DEV, dtype=torch.bfloat16).requires_grad_() for i, n in ((1, T), (2, V)))
    labels = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(3)).to(DEV)
    labels[::11] = -100
    run = lambda b: ops.linear_cross_entropy(x, w, labels, main_grad=b, reduction=reduction).sum()  # noqa: E731
    dx, dw = torch.autograd.grad(run(None), (x, w))
    main = torch.zeros(V, D, device=DEV)
    (gx,) = torch.autograd.grad(run(main), (x,))
    assert torch.equal(main.to(torch.bfloat16), dw) and torch.equal(gx, dx)        # the same sum in fp32, rounded by the caller
    once = main.clone()
    loss = run(main)
    (0.5 * loss).backward(retain_graph=True)
    loss.backward()
    # two additions in fp32, and a product with a half, which is exact
    torch.testing.assert_close(main, 2.5 * once, rtol=3 * 2.0 ** -24, atol=0)
    assert w.grad is None and torch.equal(x.grad, (0.5 * dx.float()).to(torch.bfloat16) + dx)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,V", [(32, 8, 33), (33, 400, 1003), (33, 392, 1003), (64, 768, 4097), (64, 760, 4097), (96, 1152, 5003), (96, 1144, 5003),
                                   (128, 1536, 20000), (128, 1528, 20000), (128, 4096, 1000)])
def test_losses_of_few_tokens_on_both_sides_of_the_rule(T, D, V):
    """The product with the weight's rows along the tile, and the next width that takes the tokens along it."""
    x, w, labels = sure(T, D, V, 0.0, seed=T + D)
    labels[1::3] = torch.randint(0, V, (len(labels[1::3]),), generator=torch.Generator().manual_seed(1)).to(DEV)
    labels[0] = V - 1
    (want, el), *_ = sure64(x, w, labels)
    each = ops.linear_cross_entropy(x, w, labels, reduction="none")
    off = (each.double() - want).abs() - el
    assert off.max() <= 0
    part = ops.linear_cross_entropy(x[:31], w, labels[:31], reduction="none").double()
    assert ((part - want[:31]).abs() <= el[:31]).all()
    assert int(OF.status_word(DEV).item()) == 0
