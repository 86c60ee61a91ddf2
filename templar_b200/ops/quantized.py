"""Activations in 8 bits: operands of forward passes that nothing differentiates, and what a training step keeps for its
backward pass.

A group of a row with the largest magnitude ``a`` is held as whole numbers ``q = rint(x * (127 / a))`` and one fp32 scale
``a / 127``; its values are ``q * scale``.  A group is the whole row (:func:`quantize_rows`, :func:`add_rmsnorm_q8`,
:func:`swiglu_q8`: what :func:`linear_q8` multiplies) or 64 columns of it (the ``*_saved8`` operators).  A group whose largest
magnitude is below 2^-100 is zero with scale zero; one with a member that is not finite has scale NaN, so that everything made
of it is NaN.

bf16 CUDA tensors go to the kernels of ``csrc/quant.cu``, ``csrc/gemm_2sm.cu`` and ``csrc/gemm_q8_stream.cu``, everything else to the
same formulas in PyTorch, as in :mod:`templar_b200.ops.functional`.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import functional as OF
from . import native

GROUP = 64                      # columns that share a scale in what a backward pass reads
MAX_INNER = 131072              # inner dimension of an 8-bit product: 127 * 128 * 131072 is below 2^31


def _padded(n: int) -> int:
    """Bytes from one row of codes to the next: whole 16-byte pieces, as the products' copies take them."""
    return -(-n // 16) * 16


def _native_rows(*ts) -> bool:
    for t in ts:
        if t is not None and not (t.is_cuda and t.dtype == torch.bfloat16):
            return False
    return True


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"rows of no elements: shape {tuple(x.shape)}")
    return x.reshape(-1, x.shape[-1])


def _codes(x: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(int8 codes [T, n], scales [T, G]) of fp32 rows, in PyTorch."""
    T, n = x.shape
    G = -(-n // group)
    xg = F.pad(x, (0, -n % group)).view(T, G, group)
    a = xg.abs().amax(-1, keepdim=True)                       # NaN where a member is NaN
    ok = torch.isfinite(a) & (a >= 2.0 ** -100)
    top = torch.full_like(a, 127.0)                           # a tensor: PyTorch multiplies by the reciprocal of a number
    q = torch.where(ok, torch.round(xg * (top / torch.where(ok, a, 1.0))), 0.0)
    scale = torch.where(torch.isfinite(a), torch.where(ok, a / top, 0.0), float("nan"))
    return q.to(torch.int8).view(T, G * group)[:, :n], scale.squeeze(-1)


class QuantRows:
    """Rows in 8 bits.  ``q``: int8 [T, columns rounded up to 16], of which nothing behind the last column counts (copied from a
    place that is not on a 16-byte boundary); ``scale``: fp32 [T, G] (any
    strides), one for the whole row (``group`` 0) or for every ``group`` columns; ``shape``: the rows' own shape."""

    __slots__ = ("q", "scale", "group", "shape")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, group: int, shape):
        D = shape[-1]
        if q.dtype != torch.int8 or q.dim() != 2 or q.shape[1] != _padded(D) or q.stride() != (q.shape[1], 1):
            raise ValueError(f"QuantRows: dense int8 codes [T, {_padded(D)}] expected, got {q.dtype} {tuple(q.shape)}, strides {q.stride()}")
        if math.prod(shape[:-1]) != q.shape[0]:
            raise ValueError(f"QuantRows: {q.shape[0]} rows of codes for the shape {tuple(shape)}")
        if scale.dtype != torch.float32 or scale.shape != (q.shape[0], -(-D // group) if group else 1) or scale.device != q.device:
            raise ValueError(f"QuantRows: fp32 scales [{q.shape[0]}, {-(-D // group) if group else 1}] on {q.device} expected, got "
                             f"{scale.dtype} {tuple(scale.shape)} on {scale.device}")
        if q.data_ptr() % 16:
            q = q.clone()
        self.q, self.scale, self.group, self.shape = q, scale, int(group), torch.Size(shape)

    @classmethod
    def _of(cls, q, scale, group: int, shape):
        """From the operators themselves, whose codes and scales need no look."""
        r = cls.__new__(cls)
        r.q, r.scale, r.group, r.shape = q, scale, group, shape
        return r

    @property
    def width(self) -> int:
        return self.shape[-1]

    def dequantize(self, dtype: torch.dtype = torch.bfloat16, weight: torch.Tensor | None = None) -> torch.Tensor:
        """:func:`dequantize_rows`."""
        if weight is not None:
            return dequantize_rows(self, dtype, weight)
        return _values(self.q, self.scale, self.group, self.shape, dtype)


def _empty_rows(shape, group: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    T, D = shape
    return (torch.empty(T, _padded(D), dtype=torch.int8, device=device),
            torch.empty(T, -(-D // group) if group else 1, dtype=torch.float32, device=device))


def _plain_rows(x32: torch.Tensor, group: int) -> tuple[torch.Tensor, torch.Tensor]:
    D = x32.shape[1]
    q, scale = _codes(x32, group or D)
    return F.pad(q, (0, _padded(D) - D)), scale


def quantize_rows(x: torch.Tensor, group: int = 0) -> QuantRows:
    """Rows of ``x`` in 8 bits, one scale a row (``group`` 0) or for every 64 columns (``group`` 64)."""
    if group not in (0, GROUP):
        raise ValueError(f"quantize_rows: group is 0 (the row) or {GROUP}, got {group}")
    x2 = _rows_of(x.detach())
    if not _native_rows(x2):
        return QuantRows._of(*_plain_rows(x2.float(), group), group, x.shape)
    if host := native.host():
        return QuantRows._of(*host.quantize_rows(x2, group), group, x.shape)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    T, D = x2.shape
    q, scale = _empty_rows((T, D), group, x.device)
    native.check(native.lib().tplr_quantize_rows(x2.data_ptr(), x2.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0),
                                                 scale.stride(1), T, D, group, native.stream_ptr()), "quantize_rows")
    return QuantRows._of(q, scale, group, x.shape)


def dequantize_rows(rows: QuantRows, dtype: torch.dtype = torch.bfloat16, weight: torch.Tensor | None = None) -> torch.Tensor:
    """The values ``q * scale``, times ``weight`` [columns] where one is given."""
    if weight is not None and weight.numel() != rows.width:
        raise ValueError(f"dequantize_rows: {weight.numel()} weights for {rows.width} columns")
    return _values(rows.q, rows.scale, rows.group, rows.shape, dtype, weight)


def _values(q, scale, group: int, shape, dtype, weight=None):
    T, D = q.shape[0], shape[-1]
    if q.is_cuda and dtype == torch.bfloat16 and (group in (0, GROUP) or group >= D) and _native_rows(weight):
        if host := native.host():
            return host.dequantize_rows(q, scale, group, shape, None if weight is None else weight.detach())
        y = torch.empty(shape, dtype=dtype, device=q.device)
        w = None if weight is None else weight.detach().contiguous()
        native.check(native.lib().tplr_dequantize_rows(q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0),
                                                       scale.stride(1) if group else 0, group or D, native.ptr(w),
                                                       y.data_ptr(), T, D, native.stream_ptr()), "dequantize_rows")
        return y
    wide = scale if not group else scale.repeat_interleave(group, dim=1)[:, :D]
    v = q[:, :D].float() * wide
    if weight is not None:
        v = v * weight.detach().reshape(-1).float()
    return v.to(dtype).view(shape)


# --------------------------------------------------------------------------- #
# Forward passes in 8 bits
# --------------------------------------------------------------------------- #
class QuantWeight:
    """A projection's weight in 8 bits: codes ``q`` [N, K] (int8, rows on 16-byte boundaries) and one fp32 ``scale`` for each
    output channel.  Codes in another layout are copied once, here."""

    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        if q.is_cuda and (host := native.host()) and host.weight_as_it_is(q, scale):
            self.q, self.scale = q, scale
            return
        if q.dim() != 2 or q.dtype != torch.int8 or q.shape[1] == 0:
            raise ValueError(f"QuantWeight: int8 codes [N, K] expected, got {q.dtype} {tuple(q.shape)}")
        if q.shape[1] > MAX_INNER:
            raise ValueError(f"QuantWeight: inner dimension {q.shape[1]} above {MAX_INNER}: the sums would leave 32 bits")
        if scale.shape != (q.shape[0],) or scale.dtype != torch.float32 or scale.device != q.device:
            raise ValueError(f"QuantWeight: fp32 scales [{q.shape[0]}] on {q.device} expected, got {scale.dtype} {tuple(scale.shape)} "
                             f"on {scale.device}")
        wide = _padded(q.shape[1])
        behind = q.storage_offset() + (q.shape[0] - 1) * q.stride(0) + wide       # the last row's last 16-byte piece
        if q.stride(1) != 1 or q.stride(0) % 16 or q.stride(0) < wide or q.data_ptr() % 16 or behind > q.untyped_storage().nbytes():
            rows = q.new_zeros(q.shape[0], wide)             # F.pad by nothing would keep the strides of a transposed matrix
            rows[:, :q.shape[1]] = q
            q = rows[:, :q.shape[1]]
        self.q, self.scale = q, OF._dense(scale)

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return (self.q.float() * self.scale[:, None]).to(dtype)


@torch.no_grad()
def quantize_weight(w: torch.Tensor) -> QuantWeight:
    """A weight [N, K] in 8 bits with one scale for each output channel (row)."""
    if w.dim() != 2:
        raise ValueError(f"quantize_weight: a matrix expected, got {tuple(w.shape)}")
    if w.shape[1] > MAX_INNER:
        raise ValueError(f"quantize_weight: inner dimension {w.shape[1]} above {MAX_INNER}: the sums would leave 32 bits")
    r = quantize_rows(w)
    return QuantWeight(r.q[:, :w.shape[1]], r.scale[:, 0].contiguous())


def _no_grad_asked(what: str, *ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad() (training uses the *_saved8 operators)")


def add_rmsnorm_q8(res: torch.Tensor, delta: torch.Tensor | None, w: torch.Tensor, eps: float = 1e-5) -> tuple[torch.Tensor, QuantRows]:
    """``(res + delta, rmsnorm(res + delta) * w)``, the second in 8 bits with one scale a row (``delta`` None: of ``res``)."""
    if res.is_cuda and (host := native.host()) and (made := host.add_rmsnorm_q8(res, delta, w, eps)) is not None:
        return (res if delta is None else made[0]), QuantRows._of(made[1], made[2], 0, res.shape)
    _no_grad_asked("add_rmsnorm_q8", res, delta, w)
    _norm_args("add_rmsnorm_q8", res, delta, w)
    if not _native_rows(res, delta, w):
        h = res if delta is None else res + delta
        hf = _rows_of(h.float())
        y = hf * torch.rsqrt(hf.pow(2).mean(-1, keepdim=True) + eps) * w.float()
        return h, QuantRows._of(*_plain_rows(y, 0), 0, res.shape)
    x2, w = _rows_of(res).contiguous(), w.contiguous()
    T, D = x2.shape
    d2 = None if delta is None else delta.contiguous()
    h = res if delta is None else torch.empty(res.shape, dtype=res.dtype, device=res.device)
    q, scale = _empty_rows((T, D), 0, res.device)
    native.check(native.lib().tplr_add_rmsnorm_q8(x2.data_ptr(), native.ptr(d2), w.data_ptr(), h.data_ptr(), q.data_ptr(), q.stride(0),
                                                  scale.data_ptr(), T, D, eps, native.stream_ptr()), "add_rmsnorm_q8")
    return h, QuantRows._of(q, scale, 0, res.shape)


def _norm_args(what: str, res, delta, w) -> None:
    if res.dim() == 0 or res.shape[-1] == 0:
        raise ValueError(f"{what}: rows of no elements: shape {tuple(res.shape)}")
    if w.dim() != 1 or w.shape[0] != res.shape[-1]:
        raise ValueError(f"{what}: {tuple(w.shape)} weights for rows of {res.shape[-1]}")
    if delta is not None and delta.shape != res.shape:
        raise ValueError(f"{what}: shapes {tuple(res.shape)} and {tuple(delta.shape)} differ")


def swiglu_q8(gu: torch.Tensor) -> QuantRows:
    """``silu(gate) * up`` of a packed projection [.., 2F] = [gate | up], in 8 bits with one scale a row."""
    _no_grad_asked("swiglu_q8", gu)
    if gu.shape[-1] % 2:
        raise ValueError(f"swiglu_q8: gate and up halves expected, got {gu.shape[-1]} columns")
    g2 = _rows_of(gu)
    T, Fd = g2.shape[0], g2.shape[1] // 2
    shape = (*gu.shape[:-1], Fd)
    if not _native_rows(gu):
        return QuantRows._of(*_plain_rows(F.silu(g2[:, :Fd].float()) * g2[:, Fd:].float(), 0), 0, torch.Size(shape))
    if g2.stride(1) != 1:
        g2 = g2.contiguous()
    q, scale = _empty_rows((T, Fd), 0, gu.device)
    native.check(native.lib().tplr_swiglu_q8(g2.data_ptr(), g2.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(), T, Fd,
                                             native.stream_ptr()), "swiglu_q8")
    return QuantRows._of(q, scale, 0, torch.Size(shape))


def linear_q8(x: torch.Tensor | QuantRows, w: QuantWeight, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ w.T`` from 8-bit rows and an 8-bit weight: exact sums in 32-bit integers, times one scale for each row and one for each
    channel in fp32 (the sum, the scales' product and the result are rounded to 24 bits; no step leaves the range where the result
    does not), rounded to ``out_dtype`` (bf16 or fp32; default: that of ``x``, bf16 for rows in 8 bits).  A tensor ``x`` is
    quantised first, by rows.  Forward passes only."""
    out_dtype = out_dtype or (torch.bfloat16 if isinstance(x, QuantRows) else x.dtype)
    if not isinstance(x, QuantRows):
        _no_grad_asked("linear_q8", x)
        if x.dim() == 0 or x.shape[-1] != w.q.shape[1]:
            raise ValueError(f"linear_q8: inner dimensions of {tuple(x.shape)} and {tuple(w.shape)} differ")
        if x.device != w.q.device:
            raise ValueError(f"linear_q8: rows on {x.device}, weight on {w.q.device}")
        if out_dtype is torch.bfloat16 and _native_rows(x) and (host := native.host()):
            return host.linear_q8(x, w.q, w.scale, OF.status_word(x.device))
        x = quantize_rows(x)
    if x.group:
        raise ValueError("linear_q8: rows with one scale each are multiplied, got rows with a scale for every "
                         f"{x.group} columns")
    if x.width != w.shape[1]:
        raise ValueError(f"linear_q8: inner dimensions {x.width} and {w.shape[1]} differ")
    if x.q.device != w.q.device:
        raise ValueError(f"linear_q8: rows on {x.q.device}, weight on {w.q.device}")
    if out_dtype is torch.bfloat16 and x.q.is_cuda and (host := native.host()):
        return host.linear_q8_rows(x.q, x.scale.contiguous(), x.shape, w.q, w.scale, OF.status_word(x.q.device))
    T, N, K = x.q.shape[0], w.shape[0], w.shape[1]
    if x.q.is_cuda and out_dtype in (torch.bfloat16, torch.float32):
        y = torch.empty(*x.shape[:-1], N, dtype=out_dtype, device=x.q.device)
        sx, L = x.scale.contiguous(), native.lib()
        n = L.tplr_gemm_q8_workspace(T, N, K)                 # parts of a long inner dimension
        ws = torch.empty(n, dtype=torch.int32, device=y.device) if n else None
        native.check(L.tplr_gemm_q8(x.q.data_ptr(), w.q.data_ptr(), sx.data_ptr(), w.scale.data_ptr(), y.data_ptr(), native.ptr(ws), T, N, K,
                                    x.q.stride(0), w.q.stride(0), N, int(out_dtype == torch.float32), OF.status_word(y.device).data_ptr(),
                                    native.stream_ptr()), "gemm_q8")
        return y
    y = (x.q[:, :K].double() @ w.q.double().t()) * x.scale.double() * w.scale.double()       # 64 bits: the scales may multiply out of 32
    return y.to(out_dtype).view(*x.shape[:-1], N)


# --------------------------------------------------------------------------- #
# Training steps that keep their activations in 8 bits
# --------------------------------------------------------------------------- #
class _AddRMSNormSaved8(torch.autograd.Function):
    """``(h, y)`` of :func:`functional.add_rmsnorm`; kept: the normalised rows ``xn = h * rstd`` in 8 bits by 64 columns, and
    rstd.  Backward: ``g = dy * w``, ``dx = dh + rstd * (g - xn * mean(g * xn))``, ``dw = sum(dy * xn)`` over the rows."""

    @staticmethod
    def forward(ctx, res, delta, w, eps, main_grad):
        ctx.set_materialize_grads(False)
        ctx.main_grad = main_grad
        ctx.native = _native_rows(res, delta, w)
        x2 = _rows_of(res)
        T, D = x2.shape
        if ctx.native:
            x2, w = x2.contiguous(), w.contiguous()
            d2 = None if delta is None else delta.contiguous()
            h = None if delta is None else torch.empty(res.shape, dtype=res.dtype, device=res.device)
            y = torch.empty(res.shape, dtype=res.dtype, device=res.device)
            q, scale = _empty_rows((T, D), GROUP, res.device)
            rstd = torch.empty(T, dtype=torch.float32, device=res.device)
            native.check(native.lib().tplr_add_rmsnorm_saved8(x2.data_ptr(), native.ptr(d2), w.data_ptr(), native.ptr(h), y.data_ptr(),
                                                              q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0),
                                                              scale.stride(1), rstd.data_ptr(), T, D, eps, native.stream_ptr()),
                         "add_rmsnorm_saved8")
        else:
            h = None if delta is None else res + delta
            hf = (res if h is None else h).float().reshape(T, D)
            rstd = torch.rsqrt(hf.pow(2).mean(-1) + eps)
            xn = hf * rstd[:, None]
            y = (xn * w.float()).to(res.dtype).view(res.shape)
            q, scale = _plain_rows(xn, GROUP)
        ctx.save_for_backward(q, scale, rstd, w)
        ctx.mark_non_differentiable(q, scale)
        return h, y, q, scale

    @staticmethod
    def backward(ctx, dh, dy, _dq, _dscale):
        q, scale, rstd, w = ctx.saved_tensors
        mg, D = ctx.main_grad, w.shape[0]
        if dy is None:                                        # only the sum was used
            return dh, dh if ctx.needs_input_grad[1] else None, None, None, None
        shape = dy.shape
        want = mg is not None or ctx.needs_input_grad[2]
        if ctx.native:
            dyc = dy.contiguous()
            dhc = None if dh is None else dh.contiguous()
            T = q.shape[0]
            L = native.lib()
            dx = torch.empty(shape, dtype=dy.dtype, device=dy.device)
            part = torch.empty(L.tplr_rmsnorm_saved8_parts(T, D) * D, dtype=torch.float32, device=dy.device)
            add = out = None
            if mg is not None:
                add = mg if mg.dtype == torch.float32 and mg.is_contiguous() and mg.numel() == D else \
                    torch.zeros(D, dtype=torch.float32, device=dy.device)
            elif want:
                out = torch.zeros_like(w) if T == 0 else torch.empty_like(w)
            native.check(L.tplr_rmsnorm_saved8_bwd(dyc.data_ptr(), q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0),
                                                   scale.stride(1), rstd.data_ptr(), w.data_ptr(), native.ptr(dhc), dx.data_ptr(),
                                                   part.data_ptr(), native.ptr(add), native.ptr(out), T, D, native.stream_ptr()),
                         "rmsnorm_saved8_bwd")
            if add is not None and add is not mg:
                mg.add_(add.view(mg.shape).to(mg.dtype))
            return dx, dx if ctx.needs_input_grad[1] else None, out, None, None
        xn = _values(q, scale, GROUP, (q.shape[0], D), torch.float32)
        d = dy.float().reshape(-1, D)
        g = d * w.float()
        dx = (rstd[:, None] * (g - xn * (g * xn).mean(-1, keepdim=True))).view(shape)
        if dh is not None:
            dx = dx + dh.float()
        dw = None
        if want:
            dw = (d * xn).sum(0)
            if mg is not None:
                mg.add_(dw.view(mg.shape).to(mg.dtype))
                dw = None
            else:
                dw = dw.to(w.dtype)
        dx = dx.to(dy.dtype)
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None, None


def add_rmsnorm_saved8(res: torch.Tensor, delta: torch.Tensor | None, w: torch.Tensor, eps: float = 1e-5,
                       main_grad: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, QuantRows]:
    """``(res + delta, rmsnorm(res + delta) * w, rows)`` (``delta`` None: of ``res``).  Kept for the backward pass are the
    normalised rows in 8 bits, which the third result holds for the projection behind the norm (its input is ``rows`` times
    ``w``) to keep as well instead of its input."""
    if main_grad is None:
        main_grad = getattr(w, "main_grad", None)
    _norm_args("add_rmsnorm_saved8", res, delta, w)
    if _native_rows(res, delta, w) and OF._buffers_ok((main_grad, w)) and (host := native.host()):
        if delta is None:
            h, (y, q, scale) = res, host.rmsnorm_saved8(res, w, main_grad, eps)
        else:
            h, y, q, scale = host.add_rmsnorm_saved8(res, delta, w, main_grad, eps)
        return h, y, QuantRows._of(q, scale, GROUP, res.shape)
    h, y, q, scale = _AddRMSNormSaved8.apply(res, delta, w, eps, main_grad)
    return (res if delta is None else h), y, QuantRows._of(q, scale, GROUP, res.shape)


def _kept_input(x, rows: QuantRows | None, weight):
    """(codes, scales, weight) that stand for ``x`` until the backward pass."""
    if rows is None:
        rows, weight = quantize_rows(x, GROUP), None
    if rows.group != GROUP or rows.shape != x.shape or rows.q.device != x.device:
        raise ValueError(f"rows by {GROUP} columns in the shape {tuple(x.shape)} of the input on {x.device} expected, got "
                         f"{tuple(rows.shape)} by {rows.group or 'row'} on {rows.q.device}")
    if weight is not None and (weight.shape != x.shape[-1:] or weight.device != x.device):
        raise ValueError(f"{tuple(weight.shape)} weights on {weight.device} for rows of {x.shape[-1]} on {x.device}")
    return rows.q, rows.scale, None if weight is None else weight.detach()


def _input_again(q, scale, weight, shape, dtype):
    """The rows that a projection multiplied, from what was kept of them: [T, K].  In the type that the product for the weight's
    gradient takes, so values of codes in bf16 are rounded once more: 2^-9 beside the 0.006 in norm that the codes leave."""
    return _values(q, scale, GROUP, (q.shape[0], shape[-1]), dtype, weight)


def _linear_of_nothing(x, w, main_grad):
    """A projection of no rows; the weight's gradient is zero, so a gradient buffer stays as it is."""
    return F.linear(x, w if main_grad is None else w.detach())


class _LinearSaved8(torch.autograd.Function):
    """``y = x W^T``; ``x`` is kept in 8 bits for the weight's gradient."""

    @staticmethod
    def forward(ctx, x, w, main_grad, q, scale, weight):
        ctx.save_for_backward(q, scale, weight, w)
        ctx.main_grad, ctx.shape, ctx.dtype = main_grad, x.shape, x.dtype
        y = torch.empty(*x.shape[:-1], w.shape[0], dtype=x.dtype, device=x.device)
        OF.gemm(x.reshape(-1, x.shape[-1]), w, out=y.view(-1, w.shape[0]))
        return y

    @staticmethod
    def backward(ctx, dy):
        q, scale, weight, w = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        dw = None
        if ctx.main_grad is not None or ctx.needs_input_grad[1]:
            dw = OF._weight_grad(ctx.main_grad, dy2, _input_again(q, scale, weight, ctx.shape, ctx.dtype), w, ctx.needs_input_grad[1])
        dx = OF.gemm(dy2, w, b_mn=True).view(ctx.shape) if ctx.needs_input_grad[0] else None
        return dx, dw, None, None, None, None


def linear_saved8(x, w, rows: QuantRows | None = None, weight=None, main_grad=None):
    """``x @ w.T`` whose input is kept in 8 bits.  ``rows`` (by 64 columns, times ``weight``): codes of ``x`` that are kept
    already, as :func:`add_rmsnorm_saved8` returns them; else ``x`` is quantised here."""
    if main_grad is None:
        main_grad = getattr(w, "main_grad", None)
    if not torch.is_grad_enabled():
        return OF.linear(x, w, main_grad)
    if x.numel() == 0:
        return _linear_of_nothing(x, w, main_grad)
    return _LinearSaved8.apply(x, w, main_grad, *_kept_input(x, rows, weight))


def _sums32(a: torch.Tensor, b: torch.Tensor, b_mn: bool = False) -> torch.Tensor:
    """``a b^T`` (``a b`` with ``b_mn``) with its sums left in fp32.  Operands that the own kernels do not take are copied to where they
    do; rows of no whole 16-byte pieces are multiplied in fp32, since a library product of bf16 operands rounds its sums to bf16."""
    if _native_rows(a, b) and OF._GEMM_BACKEND != "cublas":
        if a.shape[1] % 8 == 0 and b.shape[1] % 8 == 0:
            a, b = (t if t.stride(1) == 1 and t.stride(0) % 8 == 0 and OF._aligned(t) else OF._dense(t) for t in (a, b))
            return OF.gemm(a, b, b_mn=b_mn, out_dtype=torch.float32)
        OF._library_gemm_fallback(a, b)
    return a.float() @ (b.float() if b_mn else b.float().t())


class _FeedForwardSaved8(torch.autograd.Function):
    """``(silu(x w1^T) * (x w3^T)) w2^T``; kept: ``x`` and the projection [gate | up] in 8 bits, quantised from its fp32 sums.
    The backward pass forms the activation again from the kept projection."""

    @staticmethod
    def forward(ctx, x, w13, w2, mg13, mg2, xq, xscale, weight):
        x2 = x.reshape(-1, x.shape[-1])
        T, Fd = x2.shape[0], w13.shape[0] // 2
        ctx.native = _native_rows(x, w13, w2)
        ctx.fused = OF._feed_forward_fused(x2, w13, w2)
        gu = None
        if not ctx.fused:
            gu = _sums32(x2, w13)
        if ctx.fused:                 # activation and codes in the projection's epilogue
            act = torch.empty(T, Fd, dtype=x.dtype, device=x.device)
            q, scale = _empty_halves(T, Fd, x.device)
            native.check(native.lib().tplr_gemm2_swiglu_saved8(x2.data_ptr(), w13.data_ptr(), q.data_ptr(), scale.data_ptr(), act.data_ptr(),
                                                               T, Fd, x2.shape[1], x2.stride(0), w13.stride(0), q.stride(0),
                                                               scale.stride(1), Fd, OF.status_word(x.device).data_ptr(),
                                                               native.stream_ptr()), "gemm2_swiglu_saved8")
        elif ctx.native:
            act = torch.empty(T, Fd, dtype=x.dtype, device=x.device)
            q, scale = _empty_halves(T, Fd, x.device)
            native.check(native.lib().tplr_swiglu_saved8(gu.data_ptr(), act.data_ptr(), q.data_ptr(), q.stride(0), scale.data_ptr(),
                                                         scale.stride(0), scale.stride(1), T, Fd, native.stream_ptr()), "swiglu_saved8")
        else:
            g, u = gu[:, :Fd], gu[:, Fd:]
            act = (F.silu(g) * u).to(x.dtype)
            halves = [_codes(t, GROUP) for t in (g, u)]
            q, scale = (torch.cat(t, dim=1) for t in zip(*halves))
        y = torch.empty(*x.shape[:-1], w2.shape[0], dtype=x.dtype, device=x.device)
        OF.gemm(act, w2, out=y.view(-1, w2.shape[0]))
        ctx.save_for_backward(xq, xscale, weight, w13, w2, q, scale)
        ctx.mg, ctx.shape, ctx.dtype = (mg13, mg2), x.shape, x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        xq, xscale, weight, w13, w2, q, scale = ctx.saved_tensors
        mg13, mg2 = ctx.mg
        dy2 = dy.reshape(-1, dy.shape[-1]).contiguous()
        T, Fd = dy2.shape[0], w13.shape[0] // 2
        dact = None
        if not ctx.fused:
            dact = _sums32(dy2, w2, b_mn=True)
        if ctx.fused:
            dy2 = OF._dense(dy2)
            dgu = torch.empty(T, 2 * Fd, dtype=dy.dtype, device=dy.device)
            act = torch.empty(T, Fd, dtype=dy.dtype, device=dy.device)
            native.check(native.lib().tplr_gemm2_swiglu_bwd_saved8(dy2.data_ptr(), w2.data_ptr(), q.data_ptr(), scale.data_ptr(), dgu.data_ptr(),
                                                                   act.data_ptr(), T, Fd, dy2.shape[1], dy2.stride(0), w2.stride(0),
                                                                   q.stride(0), scale.stride(1), 2 * Fd, Fd,
                                                                   OF.status_word(dy.device).data_ptr(), native.stream_ptr()),
                         "gemm2_swiglu_bwd_saved8")
        elif ctx.native:
            dgu = torch.empty(T, 2 * Fd, dtype=dy.dtype, device=dy.device)
            act = torch.empty(T, Fd, dtype=dy.dtype, device=dy.device)
            native.check(native.lib().tplr_swiglu_saved8_bwd(dact.data_ptr(), q.data_ptr(), q.stride(0), scale.data_ptr(), scale.stride(0),
                                                             scale.stride(1), dgu.data_ptr(), act.data_ptr(), T, Fd, native.stream_ptr()),
                         "swiglu_saved8_bwd")
        else:
            G = scale.shape[1] // 2
            g, u = (_values(q[:, i * Fd:(i + 1) * Fd], scale[:, i * G:(i + 1) * G], GROUP, (T, Fd), torch.float32) for i in (0, 1))
            sg = torch.sigmoid(g)
            silu = g * sg
            dgu = torch.cat((dact * u * (sg + silu * (1 - sg)), dact * silu), dim=1).to(ctx.dtype)
            act = (silu * u).to(ctx.dtype)
        del dact
        dw2 = OF._weight_grad(mg2, dy2, act, w2, ctx.needs_input_grad[2])
        del act
        dx = OF.gemm(dgu, w13, b_mn=True).view(ctx.shape) if ctx.needs_input_grad[0] else None
        dw13 = None
        if mg13 is not None or ctx.needs_input_grad[1]:
            dw13 = OF._weight_grad(mg13, dgu, _input_again(xq, xscale, weight, ctx.shape, ctx.dtype), w13, ctx.needs_input_grad[1])
        return dx, dw13, dw2, None, None, None, None, None


def _empty_halves(T: int, Fd: int, device):
    """Codes [T, 2F] and scales of a packed [gate | up] projection, whose halves have groups of their own.  The scales of a group
    lie side by side for consecutive rows, the order in which a GEMM's epilogue meets them."""
    groups = 2 * -(-Fd // GROUP)
    return (torch.empty(T, _padded(2 * Fd), dtype=torch.int8, device=device),
            torch.empty(groups, T, dtype=torch.float32, device=device).t())


def feed_forward_saved8(x, w13, w2, rows: QuantRows | None = None, weight=None, main_grad13=None, main_grad2=None):
    """:func:`functional.feed_forward` with its activations kept in 8 bits: the input (``rows`` and ``weight`` as in
    :func:`linear_saved8`) and the packed projection; the activation is formed again in the backward pass."""
    if main_grad13 is None:
        main_grad13 = getattr(w13, "main_grad", None)
    if main_grad2 is None:
        main_grad2 = getattr(w2, "main_grad", None)
    if w13.shape[0] % 2 or w13.shape[1] != x.shape[-1] or w2.shape[1] != w13.shape[0] // 2:
        raise ValueError(f"feed_forward_saved8: weights {tuple(w13.shape)} and {tuple(w2.shape)} do not fit rows of {x.shape[-1]}")
    if not torch.is_grad_enabled():
        return OF.feed_forward(x, w13, w2, main_grad13, main_grad2)
    if x.numel() == 0:
        gu = _linear_of_nothing(x, w13, main_grad13)
        return _linear_of_nothing(F.silu(gu[..., :w2.shape[1]]) * gu[..., w2.shape[1]:], w2, main_grad2)
    if (OF._feed_forward_fused(x.reshape(-1, x.shape[-1]), w13, w2) and OF._buffers_ok((main_grad13, w13), (main_grad2, w2))
            and _native_rows(weight) and (host := native.host())):
        q, scale, weight = (None, None, None) if rows is None else _kept_input(x, rows, weight)
        return host.feed_forward_saved8(x, w13, w2, main_grad13, main_grad2, OF.status_word(x.device), q, scale, weight)
    return _FeedForwardSaved8.apply(x, w13, w2, main_grad13, main_grad2, *_kept_input(x, rows, weight))


class _AttentionBlockSaved8(torch.autograd.Function):
    """:class:`functional._AttentionBlock` with its input kept in 8 bits.  The rotated projection and the attention's output
    stay in bf16: the backward pass forms the probabilities again from the kept row statistics, which belong to exactly those
    values."""

    @staticmethod
    def forward(ctx, x, wqkv, wo, mg_qkv, mg_wo, cos, sin, n_heads, n_kv, hd, q, scale, weight):
        inner = OF._NoCtx()
        y = OF._AttentionBlock.forward(inner, x, wqkv, wo, mg_qkv, mg_wo, cos, sin, n_heads, n_kv, hd)
        ctx.mg, ctx.dims, ctx.shape, ctx.dtype = inner.mg, inner.dims, x.shape, x.dtype
        ctx.save_for_backward(q, scale, weight, *inner.saved[1:])
        return y

    @staticmethod
    def backward(ctx, dy):
        q, scale, weight, *rest = ctx.saved_tensors
        inner = OF._NoCtx()
        inner.saved_tensors = (_input_again(q, scale, weight, ctx.shape, ctx.dtype).view(ctx.shape), *rest)
        inner.mg, inner.dims, inner.needs_input_grad = ctx.mg, ctx.dims, ctx.needs_input_grad
        return (*OF._AttentionBlock.backward(inner, dy), None, None, None)


def attention_block_saved8(x, wqkv, wo, cos, sin, n_heads: int, n_kv: int, hd: int, rows: QuantRows | None = None, weight=None,
                           main_grad_qkv=None, main_grad_wo=None):
    """:func:`functional.attention_block` with its input kept in 8 bits (``rows`` and ``weight`` as in :func:`linear_saved8`)."""
    if main_grad_qkv is None:
        main_grad_qkv = getattr(wqkv, "main_grad", None)
    if main_grad_wo is None:
        main_grad_wo = getattr(wo, "main_grad", None)
    if not torch.is_grad_enabled():
        return OF.attention_block(x, wqkv, wo, cos, sin, n_heads, n_kv, hd, main_grad_qkv, main_grad_wo)
    if OF._attention_block_fused(x, wqkv, wo, cos, sin, n_heads, n_kv, hd):
        return _AttentionBlockSaved8.apply(x, wqkv, wo, main_grad_qkv, main_grad_wo, cos, sin, n_heads, n_kv, hd,
                                           *_kept_input(x, rows, weight))
    qkv = OF.rope(linear_saved8(x, wqkv, rows, weight, main_grad_qkv), cos, sin, n_heads + n_kv, hd)
    return OF.linear(OF.attention_packed(qkv, n_heads, n_kv, hd), wo, main_grad_wo)
