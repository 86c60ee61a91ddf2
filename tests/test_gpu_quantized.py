"""Activations in 8 bits on the kernels, against plain formulas in 64 bits.

Codes come from fp32 products with one rounding each, so those of given bf16 rows are compared exactly.  Where an fp32 value is
quantised (a norm's row, a projection's sums), it is off by ``NOISE`` of its size at most and the code by half a step."""

import pytest
import torch
import torch.nn.functional as F

from templar_b200 import ops
from templar_b200.models.llama import ModelArgs, build_model
from templar_b200.models.llama_int8 import Int8Llama
from templar_b200.ops import functional as OF
from templar_b200.ops import native
from templar_b200.ops import quantized as OQ
from templar_b200.parallel.window_engine import EngineConfig, WindowEngine

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8               # one rounding to bf16: at most 2^-9 of the value, twice that where the sum before it was off a little
NOISE = 3e-6                   # an fp32 norm or product chain: a few dozen roundings of 2^-24, and sums of up to 4096 terms in parts
EPS = 1e-5


def bf(*shape, std=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * len(shape))
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def wide(scale, group, n):
    return scale.repeat_interleave(group, dim=1)[:, :n] if group else scale


def kept(x, group):
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for i in range(0, x.shape[1], group):
        part = x[:, i:i + group].double()
        a = part.abs().amax(1, keepdim=True)
        out[:, i:i + group] = torch.where(a > 0, torch.round(part / torch.where(a > 0, a, 1) * 127) * a / 127, 0)
    return out


def healthy():
    assert int(OF.status_word(DEV).item()) == 0


WIDTHS = [(600, 384), (40, 1536), (9, 2560), (5, 6144), (1, 1), (3, 63), (5, 64), (2, 65), (1, 72), (9, 136), (7, 768), (4, 1001), (300, 2048), (65, 4096), (33, 8192), (3, 28672), (2, 40001)]


@pytest.mark.parametrize("T,D", WIDTHS)
@pytest.mark.parametrize("group", [0, 64])
def test_rows(T, D, group):
    x = bf(T, D)
    x[0] *= 0
    r = ops.quantize_rows(x, group)
    q, scale = OQ._codes(x.float(), group or D)
    assert r.q[:, :D].equal(q) and r.scale.equal(scale) and not r.q[:, D:].any()
    want = q.double() * wide(scale, group, D).double()
    assert ((r.dequantize().double() - want).abs() <= want.abs() * HALF).all()
    w = bf(D, seed=1)
    assert ((r.dequantize(weight=w).double() - want * w.double()).abs() <= (want * w.double()).abs() * HALF).all()


@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("D", [70, 1024])
def test_rows_of_zeros_tiny_values_and_values_that_are_not_finite(D, group):
    x = bf(6, D)
    x[1] = 0
    x[2] *= 1e-38
    x[3, 3], x[4, D - 1], x[5, 0] = float("nan"), float("inf"), -float("inf")
    r = ops.quantize_rows(x, group)
    q, scale = OQ._codes(x.float(), group or D)
    assert r.q[:, :D].equal(q) and r.scale.equal(scale) | (torch.equal(r.scale.isnan(), scale.isnan()) and torch.equal(r.scale.nan_to_num(), scale.nan_to_num()))
    v = r.dequantize()
    assert (v[1:3] == 0).all() and v[3, :64].isnan().all() and v[4, -6:].isnan().all() and v[5, :64].isnan().all() and v[0].isfinite().all()


def test_rows_without_tokens_views_and_other_streams():
    for f in (lambda x: ops.quantize_rows(x), lambda x: ops.quantize_rows(x, 64), lambda x: ops.add_rmsnorm_q8(x, x, bf(64))[1],
              lambda x: ops.swiglu_q8(torch.cat((x, x), -1))):
        r = f(bf(0, 64))
        assert r.q.shape == (0, 64) and r.dequantize().shape == (0, 64)
    assert ops.linear_q8(bf(2, 0, 64), ops.quantize_weight(bf(8, 64))).shape == (2, 0, 8)
    big = bf(40, 200)
    for x in (big[:, 8:136], big[:, 3:131], big[::2, 64:192], big.t()[:128], big[:24, :128].view(2, 12, -1)):
        r = ops.quantize_rows(x, 64)
        q, scale = OQ._codes(x.float().reshape(-1, x.shape[-1]), 64)
        assert r.q[:, :x.shape[-1]].equal(q) and r.scale.equal(scale) and r.shape == x.shape
    side = torch.cuda.Stream()
    x, w = bf(100, 512), ops.quantize_weight(bf(96, 512))
    want = ops.linear_q8(x, w)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_q8(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert got.equal(want)


@pytest.mark.parametrize("group", [0, 64])
def test_rows_beyond_32_bit_offsets(group):
    T, D = 65552, 32768                                    # 2^31 elements and 16 rows more
    x = torch.zeros(T, D, dtype=torch.bfloat16, device=DEV)
    x[-16:] = bf(16, D)
    r = ops.quantize_rows(x, group)
    q, scale = OQ._codes(x[-16:].float(), group or D)
    assert r.q[-16:].equal(q) and r.scale[-16:].equal(scale) and not r.q[:16].any()
    del x
    v = r.dequantize()
    assert v[-16:].equal(ops.QuantRows(r.q[-16:].clone(), r.scale[-16:].clone(), group, (16, D)).dequantize())


def test_products_beyond_32_bit_offsets():
    T, K, N = 65552, 64, 32768
    rows, w = ops.quantize_rows(bf(T, K)), ops.quantize_weight(bf(N, K, seed=1))
    y = ops.linear_q8(rows, w)
    want = (rows.q[-16:].double() @ w.q.double().t()) * rows.scale[-16:].double() * w.scale.double()
    assert ((y[-16:].double() - want).abs() <= want.abs() * HALF).all()


def norm64(res, delta):
    h = res if delta is None else (res.float() + delta.float()).to(torch.bfloat16)
    hd = h.double()
    return h, hd, torch.rsqrt(hd.pow(2).mean(-1, keepdim=True) + EPS)


@pytest.mark.parametrize("T,D", WIDTHS)
@pytest.mark.parametrize("add", [True, False])
def test_norm_in_8_bits(T, D, add):
    res, delta, w = bf(T, D, std=2.0), bf(T, D, seed=1) if add else None, bf(D, seed=2)
    h, rows = ops.add_rmsnorm_q8(res, delta, w, EPS)
    want_h, hd, r = norm64(res, delta)
    y = hd * r * w.double()
    assert h.equal(want_h)
    v = rows.q[:, :D].double() * rows.scale.double()
    assert ((v - y).abs() <= rows.scale.double() / 2 + y.abs().amax(-1, keepdim=True) * NOISE).all()
    assert torch.allclose(rows.scale.double(), y.abs().amax(-1, keepdim=True) / 127, rtol=NOISE)
    assert not rows.q[:, D:].any()


@pytest.mark.parametrize("T,D", WIDTHS)
@pytest.mark.parametrize("add", [True, False])
def test_saved_norm_and_its_gradient(T, D, add):
    res, delta, w = bf(T, D, std=2.0).requires_grad_(), bf(T, D, seed=1).requires_grad_() if add else None, bf(D, seed=2).requires_grad_()
    dh, dy = bf(T, D, seed=3), bf(T, D, seed=4)
    h, y, rows = ops.add_rmsnorm_saved8(res, delta, w, EPS)
    want_h, hd, r = norm64(res.detach(), delta.detach() if add else None)
    assert h.equal(want_h)
    yd = hd * r * w.detach().double()
    assert ((y.double() - yd).abs() <= yd.abs() * HALF).all()
    step = wide(rows.scale, 64, D).double()
    xn = rows.q[:, :D].double() * step
    assert ((xn - hd * r).abs() <= step / 2 + (hd * r).abs().amax(-1, keepdim=True) * NOISE).all()
    outs, dys = ((h, y), (dh, dy)) if add else ((y,), (dy,))
    leaves = (res, delta, w) if add else (res, w)
    got = torch.autograd.grad(outs, leaves, dys, retain_graph=True)
    g = dy.double() * w.detach().double()
    dx = r * (g - xn * (g * xn).mean(-1, keepdim=True)) + (dh.double() if add else 0)
    # rstd and the mean are sums of D terms in fp32; their errors enter at the size of the row's largest terms
    atol = NOISE * r * (g.abs().amax(-1, keepdim=True) + xn.abs().amax(-1, keepdim=True) * (g * xn).abs().mean(-1, keepdim=True))
    assert ((got[0].double() - dx).abs() <= dx.abs() * HALF + atol + 1e-30).all()
    if add:
        assert got[1].equal(got[0])
    dw = (dy.double() * xn).sum(0)
    assert ((got[-1].double() - dw).abs() <= dw.abs() * HALF + (dy.double() * xn).abs().sum(0) * NOISE).all()
    again = torch.autograd.grad(outs, leaves, dys, retain_graph=True)
    assert all(a.equal(b) for a, b in zip(got, again))                     # the same bits on every run
    mg = torch.ones(D, device=DEV)
    w.main_grad = mg
    h, y, _ = ops.add_rmsnorm_saved8(res, delta, w, EPS)
    torch.autograd.backward((h, y) if add else (y,), (dh, dy) if add else (dy,), inputs=[res, w])
    assert ((mg.double() - 1 - dw).abs() <= (dy.double() * xn).abs().sum(0) * NOISE + (1 + dw.abs()) * 2.0 ** -23).all()


# many rows: CTAs that stay and take several in turn, the last turn with fewer; more than 2^20 * 28 values
@pytest.mark.parametrize("T,D", [(2501, 2008), (1201, 4096), (5003, 768), (700, 8192), (14401, 2048)])
def test_many_rows(T, D):
    for group in (0, 64):
        test_rows(T, D, group)
    for add in (True, False):
        test_norm_in_8_bits(T, D, add)
        test_saved_norm_and_its_gradient(T, D, add)
    x = bf(T, D)
    want = ops.quantize_rows(x)
    x[T // 2, D - 1] = float("inf")
    got = ops.quantize_rows(x)
    rest = torch.arange(T, device=DEV) != T // 2
    assert got.scale[T // 2].isnan().all() and not got.q[T // 2].any()
    assert got.q[rest].equal(want.q[rest]) and got.scale[rest].equal(want.scale[rest])


@pytest.mark.parametrize("T,Fd", [(1, 1), (3, 100), (5, 64), (4, 1001), (200, 2816), (17, 8192), (2, 28672), (1, 40000)])
def test_activation_in_8_bits(T, Fd):
    gu = bf(T, 2 * Fd)
    rows = ops.swiglu_q8(gu)
    y = F.silu(gu[:, :Fd].double()) * gu[:, Fd:].double()
    v = rows.q[:, :Fd].double() * rows.scale.double()
    assert ((v - y).abs() <= rows.scale.double() / 2 + y.abs().amax(-1, keepdim=True) * NOISE).all()
    strided = torch.cat((gu, gu), 1)[:, :2 * Fd]
    assert ops.swiglu_q8(strided).q.equal(rows.q)


# (9 to 64 tokens: inner dimensions of 3, 5 and 9 blocks of 128 make clusters of 3 and 5; 8 tokens: both sides of an inner dimension of 8192)
PRODUCTS = [(24, 1152, 100), (64, 640, 130), (9, 384, 1000), (40, 1100, 17), (128, 8192, 136), (8, 8192, 40), (8, 8208, 40), (1, 1, 1), (1, 16, 8), (1, 8, 3), (1, 16384, 40), (1, 16392, 40), (3, 5456, 100), (5, 2040, 48), (7, 2336, 17), (8, 2056, 33), (2, 8192, 512), (3, 1003, 65), (8, 2048, 1111), (9, 4096, 640), (17, 100, 24), (24, 4096, 1544), (31, 777, 33),
            (32, 14336, 256), (33, 256, 512), (64, 2048, 640), (65, 2048, 2048), (100, 1000, 1000), (129, 384, 257), (256, 4096, 256), (300, 72, 5000),
            (777, 1003, 1111), (1500, 2048, 1024), (2049, 128, 96)]


@pytest.mark.parametrize("T,K,N", PRODUCTS)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product(T, K, N, out):
    x, w = bf(T, K), ops.quantize_weight(bf(N, K, seed=1))
    rows = ops.quantize_rows(x)
    y = ops.linear_q8(rows, w, out)
    sums = rows.q[:, :K].double() @ w.q.double().t()                        # exact: below 2^53
    want = sums * rows.scale.double() * w.scale.double()
    assert ((y.double() - want).abs() <= want.abs() * (HALF if out == torch.bfloat16 else 2.0 ** -22)).all()
    assert ops.linear_q8(x.view(1, T, K), w, out).equal(y.view(1, T, N))
    healthy()


# 340 tiles of 256 x 256, with and without TMA stores: each pair has several in turn, the last turn not all of them
@pytest.mark.parametrize("T,K,N", [(5003, 640, 4104), (5003, 333, 4101), (2900, 128, 9000)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_of_several_tiles_a_pair(T, K, N, out):
    test_product(T, K, N, out)


# inner dimensions that are cut into parts (4, 4, 8, 4, 6, 8 of them, the last of fewer blocks), rows that do not end with a plane's last box of 32
@pytest.mark.parametrize("T,K,N", [(256, 8192, 2048), (333, 5001, 1004), (100, 4096, 768), (130, 14336, 4096), (65, 6000, 1536), (65, 131072, 12)])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_product_with_the_inner_dimension_in_parts(T, K, N, out):
    L = native.lib()
    assert L.tplr_gemm_q8_workspace(T, N, K) > 0 and L.tplr_gemm_q8_workspace(T, N - 1, K) == 0
    x, w = bf(T, K), ops.quantize_weight(bf(N, K, seed=1))
    x[T - 2] = 0
    rows = ops.quantize_rows(x)
    y = ops.linear_q8(rows, w, out)
    want = (rows.q[:, :K].double() @ w.q.double().t()) * rows.scale.double() * w.scale.double()
    assert ((y.double() - want).abs() <= want.abs() * (HALF if out == torch.bfloat16 else 2.0 ** -22)).all()
    assert ops.linear_q8(x, w, out).equal(y)
    less = ops.linear_q8(rows, ops.QuantWeight(w.q[:N - 1], w.scale[:N - 1]), out)       # whole: channels that make no 16-byte pieces
    assert less.equal(y[:, :N - 1])
    x[3, 5] = float("nan")
    z = ops.linear_q8(x, w, out)
    assert z[3].isnan().all() and z[:3].equal(y[:3]) and z[4:].equal(y[4:])
    healthy()


@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_longest_sums_are_exact(T):
    K, N = OQ.MAX_INNER, 40
    q = torch.full((N, K), -127, dtype=torch.int8, device=DEV)
    q[1], q[2, ::2] = 127, 0
    w = ops.QuantWeight(q, torch.ones(N, device=DEV))
    rows = ops.QuantRows(torch.full((T, K), 127, dtype=torch.int8, device=DEV), torch.ones(T, 1, device=DEV), 0, (T, K))
    y = ops.linear_q8(rows, w, torch.float32)
    top = 127.0 * 127 * K
    assert (y[:, 0] == -top).all() and (y[:, 1] == top).all() and (y[:, 2] == -top / 2).all()


@pytest.mark.parametrize("T", [3, 70, 700])
def test_a_row_that_is_not_finite_spoils_itself_alone(T):
    x, w = bf(T, 256), ops.quantize_weight(bf(320, 256, seed=1))
    clean = ops.linear_q8(x, w)
    x[T - 1, 7] = float("inf")
    y = ops.linear_q8(x, w)
    assert y[T - 1].isnan().all() and y[:T - 1].equal(clean[:T - 1])


@pytest.mark.parametrize("T", [1, 20, 200])
def test_weight_codes_as_a_view_and_what_lies_behind_them(T):
    K, N = 1003, 264
    full = torch.randint(-127, 128, (N, 1008), device=DEV, dtype=torch.int8)        # codes behind column K are not zeros
    w = ops.QuantWeight(full[:, :K], torch.rand(N, device=DEV))
    assert w.q.data_ptr() == full.data_ptr()
    rows = ops.quantize_rows(bf(T, K))
    want = (rows.q[:, :K].double() @ full[:, :K].double().t()) * rows.scale.double() * w.scale.double()
    assert ((ops.linear_q8(rows, w, torch.float32).double() - want).abs() <= want.abs() * 2.0 ** -22).all()


# a few tokens, streamed in one CTA a block and in clusters, on CTA pairs with and without TMA stores, the inner dimension in parts
@pytest.mark.parametrize("T,K,N", [(3, 256, 40), (20, 256, 40), (40, 4096, 130), (200, 256, 320), (200, 256, 333), (100, 4096, 768)])
@pytest.mark.parametrize("sx,sw", [(2.0 ** -73, 2.0 ** -60), (2.0 ** -87, 2.0 ** -64), (2.0 ** -107, 2.0 ** -40), (2.0 ** -107, 2.0 ** 121),
                                   (2.0 ** 90, 2.0 ** 60), (2.0 ** 121, 2.0 ** -140)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_products_whose_scales_multiply_out_of_range(T, K, N, sx, sw, out):
    g = torch.Generator(device=DEV).manual_seed(0)
    q, wq = (torch.randint(64, 128, (n, K), dtype=torch.int8, generator=g, device=DEV) for n in (T, N))
    wq[1] = 0
    spread = lambda n: torch.linspace(1, 2, n, device=DEV)  # noqa: E731
    rows = ops.QuantRows(q, (sx * spread(T))[:, None].contiguous(), 0, (T, K))
    rows.scale[0], rows.scale[T - 1] = 0, float("nan")
    w = ops.QuantWeight(wq, sw * spread(N))
    y = ops.linear_q8(rows, w, out)
    want = (q.double() @ wq.double().t()) * rows.scale.double() * w.scale.double()
    assert y[T - 1].isnan().all() and (y[0] == 0).all() and (y[:T - 1, 1] == 0).all()
    rel, tiny = (2.0 ** -22, 2.0 ** -148) if out == torch.float32 else (HALF, 2.0 ** -132)
    y, want = y[:T - 1].double(), want[:T - 1]
    far = want.abs() > 2.0 ** 128
    assert y[far].isinf().all() and ((y - want).abs() <= want.abs() * rel + tiny)[~far].all()
    # scales of both kinds side by side: a result does not depend on its neighbours
    near = ops.QuantRows(q, rows.scale.clone(), 0, (T, K))
    near.scale[1::2], wn = 1.0, w.scale.clone()
    wn[::2] = 0.5
    z = ops.linear_q8(near, ops.QuantWeight(wq, wn), out)
    assert z[2:T - 1:2, 1::2].double().equal(y[2::2, 1::2])
    assert z[1::2, ::2].equal(ops.linear_q8(ops.QuantRows(q, torch.ones(T, 1, device=DEV), 0, (T, K)), ops.QuantWeight(wq, torch.full((N,), 0.5, device=DEV)), out)[1::2, ::2])
    healthy()


@pytest.mark.parametrize("T", [1, 20, 200])
@pytest.mark.parametrize("K", [1003, 1024])
def test_weight_codes_stored_by_input_channel(T, K):
    codes = torch.randint(-127, 128, (K, 264), device=DEV, dtype=torch.int8)
    w = ops.QuantWeight(codes.t(), torch.rand(264, device=DEV))
    rows = ops.quantize_rows(bf(T, K))
    want = (rows.q[:, :K].double() @ codes.double()) * rows.scale.double() * w.scale.double()
    assert ((ops.linear_q8(rows, w, torch.float32).double() - want).abs() <= want.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("T", [1, 8, 20, 200])
@pytest.mark.parametrize("K", [1, 100, 1003, 2047])
def test_codes_behind_the_last_column_are_not_looked_at(T, K):
    g = torch.Generator(device=DEV).manual_seed(K)
    q, full = (torch.randint(-127, 128, (n, -(-K // 16) * 16), generator=g, device=DEV, dtype=torch.int8) for n in (T, 40))
    w, scale = ops.QuantWeight(full[:, :K], torch.rand(40, device=DEV)), torch.rand(T, 1, device=DEV)
    assert w.q.data_ptr() == full.data_ptr()
    want = (q[:, :K].double() @ full[:, :K].double().t()) * scale.double() * w.scale.double()
    got = ops.linear_q8(ops.QuantRows(q, scale, 0, (T, K)), w, torch.float32)
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("T", [2, 20, 200])
def test_row_codes_off_a_16_byte_boundary(T):
    buf = torch.randint(-127, 128, (T * 64 + 1,), device=DEV, dtype=torch.int8)
    w = ops.quantize_weight(bf(40, 64))
    rows = [ops.QuantRows(q, torch.ones(T, 1, device=DEV), 0, (T, 64)) for q in (buf[1:].view(T, 64), buf[1:].clone().view(T, 64))]
    assert ops.linear_q8(rows[0], w).equal(ops.linear_q8(rows[1], w)) and rows[0].dequantize().equal(rows[1].dequantize())


@pytest.mark.parametrize("group", [32, 48, 100, 128])
def test_rows_of_a_callers_own_groups(group):
    T, D = 5, 112
    q = torch.randint(-127, 128, (T, D), device=DEV, dtype=torch.int8)
    scale, w = torch.rand(T, -(-D // group), device=DEV), bf(D)
    want = q.double() * wide(scale, group, D).double()
    rows = ops.QuantRows(q, scale, group, (T, D))
    assert ((rows.dequantize().double() - want).abs() <= want.abs() * HALF).all()
    assert ((rows.dequantize(weight=w).double() - want * w.double()).abs() <= (want * w.double()).abs() * HALF).all()


def ffn64(x, w13, w2, dy):
    """(y, dx, dw13, dw2) in 64 bits with x and the projection held in 8 bits for the gradients."""
    x, w13, w2, dy = (t.detach().double() for t in (x, w13, w2, dy))
    g, u = (x @ w13.t()).chunk(2, -1)
    y = F.silu(g) * u @ w2.t()
    g, u = kept(g, 64).requires_grad_(), kept(u, 64).requires_grad_()
    act = F.silu(g) * u
    dg, du = torch.autograd.grad(act, (g, u), dy @ w2)
    dgu = torch.cat((dg, du), -1)
    return y, dgu @ w13, dgu.t() @ kept(x, 64), dy.t() @ act.detach()


def test_no_tokens():
    w13, w2, wn = bf(256, 64).requires_grad_(), bf(64, 128).requires_grad_(), bf(64).requires_grad_()
    x = bf(0, 64).requires_grad_()
    for res, delta in ((x, None), (x, bf(0, 64))):
        h, y, rows = ops.add_rmsnorm_saved8(res, delta, wn)
        out = ops.feed_forward_saved8(y, w13, w2, rows, wn)
        grads = torch.autograd.grad(out.sum() + ops.linear_saved8(y, w13).sum() + y.sum(), (w13, w2, wn))
        assert out.shape == (0, 64) and not any(g.any() for g in grads)


def test_fp32_rows_take_the_formulas():
    x, w = torch.randn(5, 48, device=DEV), ops.quantize_weight(torch.randn(7, 48, device=DEV))
    rows = ops.quantize_rows(x)
    y = ops.linear_q8(x, w)
    want = (rows.q[:, :48].double() @ w.q.double().t()) * rows.scale.double() * w.scale.double()
    assert y.dtype == torch.float32 and ((y.double() - want).abs() <= want.abs() * 2.0 ** -22).all()
    assert ((rows.dequantize(torch.float32) - x).abs() <= rows.scale * 0.501).all()
    h, y, _ = ops.add_rmsnorm_saved8(x, x, torch.ones(48, device=DEV))
    assert h.dtype == torch.float32 and y.dtype == torch.float32


FFN = [(1, 64, 128), (5, 72, 40), (100, 128, 256), (130, 256, 384), (257, 200, 136), (300, 1024, 2816), (513, 512, 1000), (1000, 768, 2048)]


@pytest.mark.parametrize("T,D,Fd", FFN)
def test_feed_forward(T, D, Fd):
    x, w13, w2 = bf(T, D).requires_grad_(), bf(2 * Fd, D, std=D ** -0.5, seed=1).requires_grad_(), bf(D, Fd, std=Fd ** -0.5, seed=2).requires_grad_()
    dy = bf(T, D, seed=3)
    y = ops.feed_forward_saved8(x, w13, w2)
    got = (y, *torch.autograd.grad(y, (x, w13, w2), dy, retain_graph=True))
    # In norm: results rounded once (2^-9 / sqrt 3 = 0.0012), products of up to three factors that were rounded to bf16 (the same each), and
    # codes that fall the other way at a tie of the fp32 sums (a step of 1/127 of the largest for one value in some thousands): 0.003
    for a, b in zip(got, ffn64(x, w13, w2, dy)):
        assert (a.double() - b).norm() <= 4e-3 * b.norm()
    again = torch.autograd.grad(y, (x, w13, w2), dy)
    assert all(a.equal(b) for a, b in zip(got[1:], again))
    mg13, mg2 = torch.ones_like(w13, dtype=torch.float32), torch.ones_like(w2, dtype=torch.float32)
    y = ops.feed_forward_saved8(x, w13, w2, main_grad13=mg13, main_grad2=mg2)
    dx, = torch.autograd.grad(y, (x,), dy)
    assert dx.equal(got[1])
    for m, a in ((mg13, got[2]), (mg2, got[3])):
        assert ((m - 1 - a.float()).abs() <= a.float().abs() * HALF + 2.0 ** -18 * (1 + a.float().abs())).all()
    healthy()


# 320 and 160 tiles of 256 x 256 for half as many pairs as there are SMs, or more of narrower ones: each pair has several in turn, the last turn
# not all of them, the last rows of tiles are cut off; with fewer hidden units than a tile's columns in the last one
@pytest.mark.parametrize("T,D,Fd", [(5003, 256, 2048), (4390, 128, 2944)])
def test_feed_forward_of_several_tiles_a_pair(T, D, Fd):
    test_feed_forward(T, D, Fd)
    x, w13, w2 = bf(T, D).requires_grad_(), bf(2 * Fd, D, std=D ** -0.5, seed=1).requires_grad_(), bf(D, Fd, std=Fd ** -0.5, seed=2).requires_grad_()
    dy = bf(T, D, seed=3)
    y = ops.feed_forward_saved8(x, w13, w2)
    got = (y, *torch.autograd.grad(y, (x, w13, w2), dy))
    # by token and by hidden unit, so that one box of 32 x 64 cannot hide: 0.003 in norm each, up to four times that where a row is short
    for a, b, dim in zip(got, ffn64(x, w13, w2, dy), (1, 1, 1, 0)):
        assert ((a.double() - b).norm(dim=dim) <= 0.012 * b.norm(dim=dim)).all()
    healthy()


# rows of the kernels' kind, rows off their 16-byte boundary, widths that make no 16-byte pieces
@pytest.mark.parametrize("D,Fd,off", [(256, 72, 0), (256, 72, 1), (256, 128, 3), (100, 72, 0), (256, 100, 0), (129, 65, 0)])
def test_feed_forward_keeps_codes_of_fp32_sums(D, Fd, off):
    T = 200
    x = bf(T * D + 8)[off:off + T * D].view(T, D).requires_grad_()
    w13, w2 = bf(2 * Fd, D, std=D ** -0.5, seed=1).requires_grad_(), bf(D, Fd, std=Fd ** -0.5, seed=2).requires_grad_()
    codes = []

    def pack(t):
        if t.dtype == torch.int8 and t.shape[1] >= 2 * Fd:
            codes.append(t)
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = ops.feed_forward_saved8(x, w13, w2)
    g, u = (x.detach().double() @ w13.detach().double().t()).chunk(2, -1)
    want = torch.cat([OQ._codes(t.float(), 64)[0] for t in (g, u)], dim=1)
    # sums of D products in fp32 are 2^-24 sqrt(D) of a group's largest off or less, a code 127 times that from its neighbour: one in 5000 at
    # D = 256; sums rounded to bf16 (2^-9) change one in five
    assert len(codes) >= 1 and (codes[-1][:, :2 * Fd] != want).double().mean() < 1e-3
    assert ((y.double() - (F.silu(g) * u).to(torch.bfloat16).double() @ w2.detach().double().t()).norm() <= 2.5e-3 * y.double().norm())
    dy = bf(T, D, seed=3)
    got = torch.autograd.grad(y, (x, w13, w2), dy)
    for a, b in zip(got, ffn64(x, w13, w2, dy)[1:]):
        assert (a.double() - b).norm() <= 3.3e-3 * b.norm()        # three roundings to bf16 of 0.0017 each, 0.0029


@pytest.mark.parametrize("stride", [1, 0, 259])
def test_feed_forward_of_a_single_row_whatever_its_stride(stride):
    D, Fd = 256, 384
    w13, w2 = bf(2 * Fd, D, std=D ** -0.5, seed=1).requires_grad_(), bf(D, Fd, std=Fd ** -0.5, seed=2).requires_grad_()

    def run(f):
        x = f(bf(1, D)).requires_grad_()
        y = ops.feed_forward_saved8(x, w13, w2)
        return y, *torch.autograd.grad(y, (x, w13, w2), f(bf(1, D, seed=3)))
    for a, b in zip(run(lambda t: torch.as_strided(t, t.shape, (stride, 1))), run(lambda t: t)):
        assert a.equal(b)


def test_feed_forward_with_the_norms_rows_a_frozen_part_and_one_row_that_is_not_finite():
    T, D, Fd = 200, 256, 512
    x, wn = bf(T, D).requires_grad_(), (1 + 0.1 * bf(D, seed=5).float()).to(torch.bfloat16)
    w13, w2 = bf(2 * Fd, D, std=D ** -0.5, seed=1).requires_grad_(), bf(D, Fd, std=Fd ** -0.5, seed=2).requires_grad_()
    dy = bf(T, D, seed=3)
    _, y, rows = ops.add_rmsnorm_saved8(x, None, wn)
    y = y.detach().requires_grad_()
    out = ops.feed_forward_saved8(y, w13, w2, rows, wn)
    dw, = torch.autograd.grad(out, (w13,), dy)
    ref = ffn64(y, w13, w2, dy)
    assert out.equal(ops.feed_forward_saved8(y, w13, w2)) and (dw.double() - ref[2]).norm() <= 0.02 * ref[2].norm()
    frozen = w13.detach()
    a, b = torch.autograd.grad(ops.feed_forward_saved8(y, frozen, w2, rows, wn), (y, w2), dy)
    assert (a.double() - ref[1]).norm() <= 4e-3 * ref[1].norm() and (b.double() - ref[3]).norm() <= 4e-3 * ref[3].norm()
    bad = y.detach().clone()
    bad[3, 5] = float("nan")
    bad.requires_grad_()
    out2 = ops.feed_forward_saved8(bad, w13, w2)
    dbad, dw13 = torch.autograd.grad(out2, (bad, w13), dy)
    assert out2[3].isnan().all() and out2[4:].equal(out[4:]) and dbad[3].isnan().all() and dbad[4:].isfinite().all() and dw13.isnan().any()


@pytest.mark.parametrize("B,S,H,KV,hd", [(2, 128, 2, 1, 128), (1, 100, 4, 2, 64)])
def test_attention_block(B, S, H, KV, hd):
    D = H * hd
    x = bf(B, S, D).requires_grad_()
    wqkv, wo = bf((H + 2 * KV) * hd, D, std=D ** -0.5, seed=1).requires_grad_(), bf(D, D, std=D ** -0.5, seed=2).requires_grad_()
    cos, sin = (t.contiguous() for t in OF.rope_tables(S, hd, 10000.0, DEV))
    dy = bf(B, S, D, seed=3)
    y = ops.attention_block_saved8(x, wqkv, wo, cos, sin, H, KV, hd)
    want = OF.attention_block(x, wqkv, wo, cos, sin, H, KV, hd)
    assert y.equal(want)
    got, ref = (torch.autograd.grad(o, (x, wqkv, wo), dy) for o in (y, want))
    assert got[0].equal(ref[0]) and got[2].equal(ref[2])                    # the kept input enters its weight's gradient alone
    assert (got[1].float() - ref[1].float()).norm() <= 0.02 * ref[1].float().norm()


ARGS = ModelArgs(dim=256, n_layers=3, n_heads=2, n_kv_heads=1, vocab_size=512, intermediate_size=384, max_seq_len=128)


def test_a_training_step_with_saved_activations_in_8_bits():
    tok = torch.randint(0, 512, (4, 129), generator=torch.Generator().manual_seed(0)).to(DEV)

    def step(mode, shard=False):
        m = build_model(ARGS, device=DEV, dtype=torch.bfloat16, seed=3)
        m.activation_checkpointing = mode
        eng = WindowEngine(m, EngineConfig(shard_params=shard), device=DEV)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        loss = m.loss(tok[:, :-1], tok[:, 1:])
        held = torch.cuda.memory_allocated() - base
        loss.backward()
        return float(loss.detach()), (eng.store.grad_shard if shard else eng.store.grad).clone(), held
    l0, g0, b0 = step("none")
    l1, g1, b1 = step("int8")
    assert abs(l1 - l0) < 5e-3 and (g1 - g0).norm() < 0.03 * g0.norm() and b1 < 0.75 * b0
    l0, g0, _ = step("none", True)                                         # gradient targets with a method of their own: the Python nodes
    l1, g1, _ = step("int8", True)
    assert abs(l1 - l0) < 5e-3 and (g1 - g0).norm() < 0.03 * g0.norm()
    healthy()


def test_scoring_in_8_bits_is_near_the_model():
    # initial values in fp32 and then rounded, as a node makes them: drawn in bf16, a truncated normal has values 100 deviations out,
    # and 8 bits with one scale a channel leave little of the others
    m = build_model(ARGS, device=DEV, seed=3)
    m = m._apply(lambda t: t.to(torch.bfloat16) if t.is_floating_point() else t)
    q = Int8Llama(m)
    tok = torch.randint(0, 512, (2, 129), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        want = m(tok[:, :-1]).float()
        loss = float(m.loss(tok[:, :-1], tok[:, 1:]))
    assert (q(tok[:, :-1]).float() - want).norm() < 0.04 * want.norm()
    assert abs(float(q.loss(tok[:, :-1], tok[:, 1:])) - loss) < 0.02
    one = q(tok[:1, :1]).float()
    assert (one - want[:1, :1]).norm() < 0.06 * want[:1, :1].norm()
    healthy()


@pytest.mark.parametrize("T,D,Fd", [(5, 72, 40), (300, 256, 384)])
def test_the_python_nodes_give_the_bits_of_those_in_cpp(T, D, Fd, monkeypatch):
    res, delta, wn = bf(T, D).requires_grad_(), bf(T, D, seed=1).requires_grad_(), bf(D, seed=2).requires_grad_()
    w13, w2 = bf(2 * Fd, D, std=D ** -0.5, seed=3).requires_grad_(), bf(D, Fd, std=Fd ** -0.5, seed=4).requires_grad_()
    dh, dy = bf(T, D, seed=5), bf(T, D, seed=6)
    qw = ops.quantize_weight(w13)

    def everything():
        out = []
        for d in (delta, None):
            h, y, rows = ops.add_rmsnorm_saved8(res, d, wn)
            z = ops.feed_forward_saved8(y, w13, w2, rows, wn)
            out += [h, y, rows.q, rows.scale, z, *torch.autograd.grad((h, z), (res, wn, w13, w2), (dh, dy))]
            out += torch.autograd.grad(ops.feed_forward_saved8(res, w13, w2), (res, w13), dy)
            with torch.no_grad():
                h, rows = ops.add_rmsnorm_q8(res, d, wn)
                gu = ops.linear_q8(rows, qw)
                out += [h, rows.q, rows.scale, gu, ops.linear_q8(res, qw), rows.dequantize(weight=wn), ops.swiglu_q8(gu).q]
        out += [ops.quantize_rows(res, g).q for g in (0, 64)]
        return out

    want = everything()
    assert native.host()
    monkeypatch.setattr(native, "host", lambda: None)
    got = everything()
    assert len(got) == len(want) and all(a.equal(b) for a, b in zip(got, want))
