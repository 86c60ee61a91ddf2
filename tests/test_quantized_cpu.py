"""Activations in 8 bits (ops/quantized.py) on the CPU: format, formulas, refusals, and the model paths that use them."""

from types import SimpleNamespace

import pytest
import torch
import torch.autograd.graph as ag

from templar_b200 import model_factory as mf
from templar_b200 import ops
from templar_b200.models.llama import ModelArgs, build_model
from templar_b200.models.llama_int8 import Int8Llama
from templar_b200.models.llama_tp import TPLlamaModel
from templar_b200.parallel.window_engine import EngineConfig, WindowEngine

ARGS = ModelArgs(dim=128, n_layers=3, n_heads=2, n_kv_heads=1, vocab_size=256, intermediate_size=192, max_seq_len=32)


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def kept(x, group):
    """What 8 bits leave of rows, in 64 bits."""
    out = torch.empty_like(x, dtype=torch.float64)
    for i in range(0, x.shape[1], group):
        part = x[:, i:i + group].double()
        a = part.abs().amax(1, keepdim=True)
        out[:, i:i + group] = torch.where(a > 0, torch.round(part / torch.where(a > 0, a, 1) * 127) * a / 127, 0)
    return out


@pytest.mark.parametrize("T,D", [(0, 8), (1, 1), (3, 63), (2, 64), (5, 65), (4, 200)])
@pytest.mark.parametrize("group", [0, 64])
def test_rows_keep_their_values_to_half_a_step(T, D, group):
    x = rand(T, D)
    r = ops.quantize_rows(x, group)
    assert r.q.dtype == torch.int8 and r.q.shape[1] % 16 == 0 and not r.q[:, D:].any()
    assert r.scale.shape == (T, -(-D // group) if group else 1)
    step = r.scale.repeat_interleave(group or D, dim=1)[:, :D]
    assert ((r.dequantize(torch.float32) - x).abs() <= step * 0.50001).all()
    if T:
        assert r.q.abs().amax() == 127


@pytest.mark.parametrize("group", [0, 64])
def test_rows_of_zeros_tiny_values_and_values_that_are_not_finite(group):
    x = rand(6, 70)
    x[1] = 0
    x[2] *= 1e-38                                              # 127 / a would overflow
    x[3, 3], x[4, 69], x[5, 0] = float("nan"), float("inf"), -float("inf")
    r = ops.quantize_rows(x, group)
    v = r.dequantize(torch.float32)
    assert (v[1:3] == 0).all() and (r.scale[1:3] == 0).all()
    assert not r.q[3, :64 if group else 70].any() and v[3, :64].isnan().all()
    assert v[4, 64:].isnan().all() and v[5, :64].isnan().all()
    assert v[4, :64].isnan().all() == (group == 0) and v[0].isfinite().all()


def test_leading_shapes_views_and_weights_of_the_columns():
    x = rand(2, 3, 40).transpose(0, 1)
    w = rand(40, seed=1)
    r = ops.quantize_rows(x, 64)
    assert r.shape == x.shape and r.dequantize().shape == x.shape and r.dequantize().dtype == torch.bfloat16
    assert torch.equal(ops.dequantize_rows(r, torch.float32, w), r.dequantize(torch.float32) * w)


def test_row_codes_off_a_16_byte_boundary_are_copied():
    buf = torch.randint(-127, 128, (3 * 32 + 1,), dtype=torch.int8, generator=torch.Generator().manual_seed(0))
    for at in (0, 1):
        q = buf[at:at + 96].view(3, 32)
        r = ops.QuantRows(q, torch.ones(3, 1), 0, (3, 20))
        assert r.q.equal(q) and r.q.data_ptr() % 16 == 0 and (r.q.data_ptr() == q.data_ptr()) == (q.data_ptr() % 16 == 0)


def test_weights_of_the_columns_in_any_shape():
    x, w = rand(40, 40), rand(40, seed=1)                      # as many rows as columns: a column of weights would multiply the rows
    r = ops.quantize_rows(x, 64)
    want = r.dequantize(torch.float32) * w
    for shape in ((40,), (40, 1), (1, 40), (1, 40, 1)):
        assert torch.equal(ops.dequantize_rows(r, torch.float32, w.view(shape)), want)
        assert torch.equal(r.dequantize(weight=w.view(shape)), want.to(torch.bfloat16))
    with pytest.raises(ValueError, match="weights for 40 columns"):
        ops.dequantize_rows(r, torch.float32, w[:39])


@pytest.mark.parametrize("T,K,N", [(1, 1, 1), (3, 17, 5), (8, 128, 64)])
def test_product_is_the_one_of_the_kept_values(T, K, N):
    x, w = rand(T, K), rand(N, K, seed=1)
    qw = ops.quantize_weight(w)
    y = ops.linear_q8(x, qw)
    want = kept(x, K) @ kept(w, K).t()
    # three roundings of the product and its scales, and the scales' own
    assert ((y.double() - want).abs() <= 6 * 2.0 ** -24 * (kept(x, K).abs() @ kept(w, K).abs().t()) + 1e-30).all()
    assert ops.linear_q8(ops.quantize_rows(x), qw, torch.float32).equal(y)
    assert (qw.dequantize(torch.float32) - w).abs().max() <= qw.scale.max() * 0.50001


# (rows' scale, channels' scale): products of the two below and above the normal numbers, whose results are normal, tiny or zero
@pytest.mark.parametrize("sx,sw", [(2.0 ** -73, 2.0 ** -60), (2.0 ** -87, 2.0 ** -64), (2.0 ** -107, 2.0 ** -40), (2.0 ** -107, 2.0 ** 121),
                                   (2.0 ** 90, 2.0 ** 60), (2.0 ** 121, 2.0 ** -140)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_products_whose_scales_multiply_out_of_range(sx, sw, out):
    T, K, N = 4, 4096, 6
    g = torch.Generator().manual_seed(0)
    q = torch.randint(64, 128, (T, K), dtype=torch.int8, generator=g)
    wq = torch.randint(64, 128, (N, K), dtype=torch.int8, generator=g)
    wq[1] = 0
    rows = ops.QuantRows(q, torch.full((T, 1), sx) * torch.tensor([[1.0], [1.3], [0.0], [float("nan")]]), 0, (T, K))
    y = ops.linear_q8(rows, ops.QuantWeight(wq, torch.full((N,), sw) * 1.7), out)
    want = (q.double() @ wq.double().t()) * rows.scale.double() * torch.full((N,), sw).mul(1.7).double()
    assert y[3].isnan().all() and (y[2] == 0).all() and (y[:3, 1] == 0).all()
    # one rounding to 24 or 8 bits after three of 24, and half a step of the smallest numbers at each
    rel, tiny = (2.0 ** -22, 2.0 ** -148) if out == torch.float32 else (2.0 ** -8, 2.0 ** -132)
    far = want[:3].abs() > 2.0 ** 128
    assert y[:3][far].isinf().all() and ((y[:3].double() - want[:3]).abs() <= want[:3].abs() * rel + tiny)[~far].all()


def test_forward_operators_against_their_formulas():
    res, delta, w = rand(5, 96), rand(5, 96, seed=1), rand(96, seed=2)
    h, rows = ops.add_rmsnorm_q8(res, delta, w)
    y = ((res + delta) * torch.rsqrt((res + delta).pow(2).mean(-1, keepdim=True) + 1e-5) * w).double()
    assert h.equal(res + delta) and ((rows.dequantize(torch.float32).double() - y).abs() <= rows.scale * 0.501).all()
    h, rows = ops.add_rmsnorm_q8(res, None, w)
    assert h is res
    gu = rand(5, 96, seed=3)
    act = torch.nn.functional.silu(gu[:, :48].double()) * gu[:, 48:].double()
    rows = ops.swiglu_q8(gu)
    assert rows.shape == (5, 48) and ((rows.dequantize(torch.float32).double() - act).abs() <= rows.scale * 0.501).all()


def _grads(fn, *leaves, dy):
    outs = fn()
    return torch.autograd.grad(outs, leaves, dy)


@pytest.mark.parametrize("T,D", [(1, 64), (4, 100)])
def test_norm_gradient_is_the_formula_at_the_kept_rows(T, D):
    res, delta, w = (rand(*s, seed=i).requires_grad_() for i, s in enumerate([(T, D), (T, D), (D,)]))
    dh, dy = rand(T, D, seed=5), rand(T, D, seed=6)
    h, y, rows = ops.add_rmsnorm_saved8(res, delta, w)
    got = torch.autograd.grad((h, y), (res, delta, w), (dh, dy))
    hd = (res + delta).detach().double()
    r = torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5)
    xn = rows.dequantize(torch.float32).double()
    assert ((xn - hd * r).abs() <= rows.scale.repeat_interleave(64, 1)[:, :D] * 0.501).all()
    g = dy.double() * w.detach().double()
    dx = dh + r * (g - xn * (g * xn).mean(-1, keepdim=True))
    for a, b in zip(got, (dx, dx, (dy.double() * xn).sum(0))):
        assert torch.allclose(a.double(), b, rtol=1e-5, atol=1e-5)
    # only the sum is used
    h, y, _ = ops.add_rmsnorm_saved8(res, delta, w)
    assert torch.autograd.grad(h, res, dh)[0].equal(dh)


def test_feed_forward_gradient_is_the_formula_at_the_kept_values_and_near_the_differences():
    T, D, Fd = 6, 48, 72
    x, w13, w2 = (rand(*s, seed=i).mul(0.3).requires_grad_() for i, s in enumerate([(T, D), (2 * Fd, D), (D, Fd)]))
    dy = rand(T, D, seed=9)
    y = ops.feed_forward_saved8(x, w13, w2)
    got = torch.autograd.grad(y, (x, w13, w2), dy)
    xd, w13d, w2d, dyd = (t.detach().double() for t in (x, w13, w2, dy))

    def f(x, w13, w2):
        g, u = (x @ w13.t()).chunk(2, -1)
        return torch.nn.functional.silu(g) * u @ w2.t()

    assert torch.allclose(y.double(), f(xd, w13d, w2d), rtol=1e-5, atol=1e-5)
    gate, up = (t.requires_grad_() for t in (kept(p, 64) for p in (xd @ w13d.t()).chunk(2, -1)))
    act = torch.nn.functional.silu(gate) * up
    dg, du = torch.autograd.grad(act, (gate, up), dyd @ w2d)
    dgu = torch.cat((dg, du), -1)
    # codes of the fp32 and the 64-bit projection may differ by a step at a tie, which no element here is near
    for a, b in zip(got, (dgu @ w13d, dgu.t() @ kept(xd, 64), dyd.t() @ act.detach())):
        assert torch.allclose(a.double(), b, rtol=1e-4, atol=1e-5)
    # along the gradient itself: kept values are off by 1/254 of a group's largest at most, about 1 % of its spread
    for i, g in enumerate(got):
        eps, args = 1e-5, [xd, w13d, w2d]
        ends = []
        for s in (1, -1):
            moved = list(args)
            moved[i] = moved[i] + s * eps * g.double()
            ends.append((f(*moved) * dyd).sum())
        slope = (ends[0] - ends[1]) / (2 * eps)
        assert abs(slope / g.double().pow(2).sum() - 1) < 0.03


def test_feed_forward_keeps_a_third_of_the_bytes_and_takes_the_norms_rows():
    T, D, Fd = 64, 64, 256
    x, w13, w2, wn = rand(T, D).requires_grad_(), rand(2 * Fd, D, seed=1).requires_grad_(), rand(D, Fd, seed=2).requires_grad_(), rand(D, seed=3)
    _, y, rows = ops.add_rmsnorm_saved8(x, None, wn)

    def stored(fn):
        n = [0]

        def pack(t):
            if t.data_ptr() not in (w13.data_ptr(), w2.data_ptr()):                  # activations, not weights
                n[0] += t.numel() * t.element_size()
            return t
        with ag.saved_tensors_hooks(pack, lambda t: t):
            out = fn()
        return out, n[0]
    from templar_b200.ops import functional as OF
    out0, b0 = stored(lambda: OF.feed_forward(y, w13, w2))
    out1, b1 = stored(lambda: ops.feed_forward_saved8(y, w13, w2, rows, wn))
    assert torch.allclose(out0, out1, rtol=1e-5, atol=1e-4) and b1 < b0 / 3
    (dw,) = torch.autograd.grad(out1, w13, torch.ones_like(out1), retain_graph=True)
    (dw0,) = torch.autograd.grad(ops.feed_forward_saved8(y, w13, w2), w13, torch.ones_like(out1))
    assert (dw - dw0).norm() < 0.02 * dw0.norm()


def test_no_tokens():
    w13, w2, wn = rand(16, 8).requires_grad_(), rand(8, 8).requires_grad_(), rand(8).requires_grad_()
    x = rand(0, 8).requires_grad_()
    h, y, rows = ops.add_rmsnorm_saved8(x, None, wn)
    out = ops.feed_forward_saved8(y, w13, w2, rows, wn)
    assert out.shape == (0, 8)
    for g in torch.autograd.grad(out.sum() + ops.linear_saved8(y, w13).sum(), (w13, w2, wn)):
        assert not g.any()


def test_refusals():
    x, w = rand(4, 32), ops.quantize_weight(rand(8, 32, seed=1))
    with pytest.raises(ValueError, match="inner dimensions"):
        ops.linear_q8(rand(4, 31), w)
    with pytest.raises(ValueError, match="inner dimensions"):
        ops.linear_q8(ops.quantize_rows(rand(4, 31)), w)
    with pytest.raises(ValueError, match="one scale each"):
        ops.linear_q8(ops.quantize_rows(x, 64), w)
    with pytest.raises(ValueError, match="no backward"):
        ops.linear_q8(x.clone().requires_grad_(), w)
    with pytest.raises(ValueError, match="no backward"):
        ops.add_rmsnorm_q8(x, None, torch.ones(32, requires_grad=True))
    with pytest.raises(ValueError, match="group"):
        ops.quantize_rows(x, 32)
    with pytest.raises(ValueError, match="no elements"):
        ops.quantize_rows(torch.empty(3, 0))
    with pytest.raises(ValueError, match="weights for rows"):
        ops.add_rmsnorm_q8(x, None, torch.ones(31))
    with pytest.raises(ValueError, match="differ"):
        ops.add_rmsnorm_saved8(x, rand(3, 32), torch.ones(32))
    with pytest.raises(ValueError, match="halves"):
        ops.swiglu_q8(rand(2, 7))
    with pytest.raises(ValueError, match="int8 codes"):
        ops.QuantWeight(torch.zeros(3, 4), torch.zeros(3))
    with pytest.raises(ValueError, match="fp32 scales"):
        ops.QuantWeight(torch.zeros(3, 4, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(ValueError, match="leave 32 bits"):
        ops.QuantWeight(torch.zeros(1, 131088, dtype=torch.int8), torch.zeros(1))
    with pytest.raises(ValueError, match="dense int8 codes"):
        ops.QuantRows(torch.zeros(3, 20, dtype=torch.int8), torch.zeros(3, 1), 0, (3, 20))
    with pytest.raises(ValueError, match="3 rows of codes"):
        ops.QuantRows(torch.zeros(3, 32, dtype=torch.int8), torch.zeros(3, 1), 0, (4, 20))
    with pytest.raises(ValueError, match="fp32 scales"):
        ops.QuantRows(torch.zeros(3, 80, dtype=torch.int8), torch.zeros(3, 1), 64, (3, 80))
    with pytest.raises(ValueError, match="do not fit"):
        ops.feed_forward_saved8(x, rand(16, 32), rand(32, 9))
    with pytest.raises(ValueError, match="weights on"):
        ops.feed_forward_saved8(x, rand(16, 32), rand(32, 8), ops.quantize_rows(x, 64), torch.ones(31))
    with pytest.raises(ValueError, match="by 64 columns"):
        ops.feed_forward_saved8(x, rand(16, 32), rand(32, 8), ops.quantize_rows(x))


def test_weight_codes_that_end_with_their_storage_are_copied():
    q = torch.randint(-127, 128, (3 * 20,), dtype=torch.int8)[:57].view(3, 19)       # rows off 16-byte boundaries
    w = ops.QuantWeight(q, torch.ones(3))
    assert w.q.equal(q) and w.q.stride(0) == 32
    q = torch.zeros(3 * 32 - 8, dtype=torch.int8).as_strided((3, 20), (32, 1))       # the last piece would leave the storage
    assert ops.QuantWeight(q, torch.ones(3)).q.data_ptr() != q.data_ptr()
    q = torch.zeros(3, 32, dtype=torch.int8)[:, :20]
    assert ops.QuantWeight(q, torch.ones(3)).q.data_ptr() == q.data_ptr()


# codes stored by input channel, a column of a wider matrix, one channel for all: of inner dimensions that are whole 16-byte pieces and not
@pytest.mark.parametrize("K", [16, 19, 48, 64])
def test_weight_codes_in_every_layout_become_dense_rows(K):
    q = torch.randint(-127, 128, (24, K), dtype=torch.int8, generator=torch.Generator().manual_seed(K))
    wide = torch.zeros(24, K, 5, dtype=torch.int8)
    wide[:, :, 2] = q
    for view in (q.t().contiguous().t(), wide[:, :, 2], q[:1].expand(24, K), q.flip(0)[::2]):
        w = ops.QuantWeight(view, torch.ones(view.shape[0]))
        assert w.q.equal(view) and w.q.stride(1) == 1 and w.q.stride(0) % 16 == 0 and w.q.stride(0) >= K
        assert w.q.data_ptr() % 16 == 0 and w.q.untyped_storage().nbytes() >= (w.q.shape[0] - 1) * w.q.stride(0) + -(-K // 16) * 16


def _step(mode, packed=True, shard=False):
    m = build_model(ARGS, seed=3)
    m.activation_checkpointing = mode
    eng = WindowEngine(m, EngineConfig(shard_params=shard), device="cpu") if packed else None
    tok = torch.randint(0, 256, (3, 33), generator=torch.Generator().manual_seed(0))
    stored = [0]

    def pack(t):
        stored[0] += t.numel() * t.element_size()
        return t
    with ag.saved_tensors_hooks(pack, lambda t: t):
        loss = m.loss(tok[:, :-1], tok[:, 1:])
    loss.backward()
    if shard:
        return float(loss.detach()), eng.store.stage.clone(), stored[0]
    return float(loss.detach()), eng.store.grad.clone() if packed else torch.cat([p.grad.flatten() for p in m.parameters()]), stored[0]


@pytest.mark.parametrize("packed,shard", [(True, False), (False, False), (True, True)])
def test_a_training_step_with_saved_activations_in_8_bits(packed, shard):
    l0, g0, b0 = _step("none", packed, shard)
    l1, g1, b1 = _step("int8", packed, shard)
    # the forward pass computes the same thing; gradients are off by what 8 bits leave out
    assert abs(l1 - l0) < 1e-5 and (g1 - g0).norm() < 0.02 * g0.norm() and b1 < b0


def test_model_factory_reads_the_mode():
    hp = SimpleNamespace(model_size="tiny", sequence_length=32,
                         model_config=SimpleNamespace(vocab_size=256, hidden_size=128, num_hidden_layers=2, num_attention_heads=2,
                                                      num_key_value_heads=2, intermediate_size=256, rms_norm_eps=1e-5, rope_theta=10000.0),
                         torchtitan=SimpleNamespace(activation_checkpoint={"mode": "int8"}))
    assert mf.initialize_torchtitan_model(hp, role="miner", device="cpu", world_size=1).activation_checkpointing == "int8"


def test_scoring_refuses_sharded_weights():
    m = build_model(ARGS, seed=3)
    WindowEngine(m, EngineConfig(shard_params=True), device="cpu")
    with pytest.raises(ValueError, match="sharded"):
        Int8Llama(m)


# two ranks; one rank whose vocabulary is padded, so that its logits have columns of no entry
@pytest.mark.parametrize("world,vocab", [(2, 256), (1, 200)])
def test_scoring_refuses_one_ranks_part_of_a_model(world, vocab):
    args = ModelArgs(dim=128, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=vocab, intermediate_size=256, max_seq_len=32)
    full = build_model(args, seed=3)
    m = TPLlamaModel(args, 0, world)
    m.freqs_cis = full.freqs_cis
    m.load_from_full(full)
    with pytest.raises(ValueError, match="one rank's part"):
        Int8Llama(m)


def test_scoring_in_8_bits_is_near_the_model():
    m = build_model(ARGS, seed=3)
    tok = torch.randint(0, 256, (2, 33), generator=torch.Generator().manual_seed(1))
    q = Int8Llama(m)
    with torch.no_grad():
        want, got = m(tok[:, :-1]), q(tok[:, :-1])
        loss = m.loss(tok[:, :-1], tok[:, 1:])
    assert (got - want).norm() < 0.03 * want.norm()
    assert abs(float(q.loss(tok[:, :-1], tok[:, 1:])) - float(loss)) < 0.02
    assert q(tok[:1, :1]).shape == (1, 1, 256)
