"""Operators of a training step, or of scoring, on sequences that hold several documents one behind the other.

Every row ``s`` of a sequence has a ``start``: it sees the keys ``max(start, 0) .. s``, so a document's rows have the row their
document begins at, a window of ``n`` keys is a start of ``s - n + 1``, and a row whose start lies behind it (one that fills up a
sequence) sees nothing.  :func:`document_starts` makes them from the tokens.

bf16 CUDA tensors go to the kernels of ``csrc/attention.cu``, ``csrc/qk_norm.cu``, ``csrc/gemm_2sm.cu`` and ``csrc/vocab_loss.cu``, everything else
to the same formulas in PyTorch, as in :mod:`templar_b200.ops.functional`.
"""

from __future__ import annotations

import contextlib
import warnings

import torch
import torch.autograd.forward_ad as fwAD

from . import functional as OF
from . import native

# Of the weights exp(logit) that are there at a time.  Every run of tokens reads the whole weight and, where there are several, adds onto the whole
# fp32 gradient: 16384 x 4096 x 128256 is eight runs of 2048 tokens, 4 GB each beside 4.7 ms of products.
CHUNK_BYTES = 512 << 20


def _on(t: torch.Tensor):
    """The kernels are launched on the current device's stream: makes the tensor's device the current one where it is not."""
    if not t.is_cuda or t.device.index == torch._C._cuda_getDevice():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _word(t: torch.Tensor) -> torch.Tensor:
    return OF._status_words.get(t.get_device()) if t.get_device() in OF._status_words else OF.status_word(t.device)


def _same_device(what: str, t: torch.Tensor, **others) -> None:
    for name, o in others.items():
        if o is not None and o.device != t.device:
            raise ValueError(f"{what}: {name} is on {o.device}, the rows are on {t.device}")


def _has_tangent(*ts: torch.Tensor) -> bool:
    """A forward-mode derivative is asked for.  The formulas carry it; from the kernels an output would come without one, and read as
    a derivative of zero."""
    return fwAD._current_level >= 0 and any(t.is_floating_point() and fwAD.unpack_dual(t).tangent is not None for t in ts)


def _no_forward_mode(what: str) -> NotImplementedError:
    return NotImplementedError(f"{what}: the kernels have no forward-mode derivative")


def _fitting_buffer(what: str, name: str, w: torch.Tensor, main_grad: torch.Tensor) -> None:
    """The kernels add ``w``'s gradient into the buffer by its address."""
    if main_grad.device != w.device or main_grad.numel() != w.numel():
        raise ValueError(f"{what}: {name} of {w.numel()} numbers on {w.device} expected, got {main_grad.numel()} on {main_grad.device}")


def _heads(what: str, qkv: torch.Tensor, n_heads: int, n_kv: int, hd: int) -> None:
    if qkv.dim() != 3 or n_heads < 1 or n_kv < 1 or n_heads % n_kv or hd < 1 or qkv.shape[2] != (n_heads + 2 * n_kv) * hd:
        raise ValueError(f"{what}: a packed projection [B, S, (H + 2 KV) * hd] expected, got {tuple(qkv.shape)} for {n_heads} query heads on "
                         f"{n_kv} of {hd}")


def _packed_rows(qkv: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(qkv, elements from one row to the next) as the kernels read it: [B * S] rows evenly apart, in whole 16-byte pieces.  Anything
    else is copied."""
    B, S, C = qkv.shape
    ld = qkv.stride(1) if S > 1 else qkv.stride(0) if B > 1 else C
    if qkv.stride(2) != 1 or ld < C or ld % 8 or (B > 1 and qkv.stride(0) != S * ld) or qkv.data_ptr() % 16:
        return qkv.clone(memory_format=torch.contiguous_format), C
    return qkv, ld


# --------------------------------------------------------------------------- #
# starts of documents
# --------------------------------------------------------------------------- #
def document_starts(tokens: torch.Tensor, eos_id: int, window: int = 0) -> torch.Tensor:
    """int32 [B, S]: the row at which each token's document begins, for documents that end with ``eos_id``; ``window`` > 0: no
    earlier than the ``window - 1``-th row before it."""
    if tokens.dim() != 2:
        raise ValueError(f"document_starts: tokens [B, S] expected, got {tuple(tokens.shape)}")
    rows = torch.arange(tokens.shape[1], device=tokens.device, dtype=torch.int32)
    first = torch.zeros(tokens.shape, dtype=torch.int32, device=tokens.device)
    if tokens.shape[1] > 1:
        first[:, 1:] = torch.where(tokens[:, :-1] == eos_id, rows[1:], 0)
        first = first.cummax(1).values.to(torch.int32)
    return torch.maximum(first, rows - (min(int(window), tokens.shape[1]) - 1)) if window > 0 else first


# --------------------------------------------------------------------------- #
# attention within documents
# --------------------------------------------------------------------------- #
class _AttentionDocuments(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, starts, n_heads, n_kv, hd):
        qkv, ld = _packed_rows(qkv)
        out, lse, blocks = _attention_documents(qkv, ld, starts, n_heads, n_kv, hd, True)
        ctx.save_for_backward(qkv, starts, out, lse, blocks)
        ctx.dims = (n_heads, n_kv, hd, ld)
        return out

    @staticmethod
    def backward(ctx, dout):
        qkv, starts, out, lse, blocks = ctx.saved_tensors
        n_heads, n_kv, hd, ld = ctx.dims
        B, S, C = qkv.shape
        with _on(qkv):
            do = OF._dense(dout)
            dqkv = torch.empty(B, S, C, dtype=qkv.dtype, device=qkv.device)
            cols = native.lib().tplr_attention_docs_bwd_scratch_cols(B, S, n_heads, n_kv, hd)
            part = torch.empty(B * S * cols, dtype=torch.float32, device=qkv.device) if cols else None
            delta = torch.empty(B, n_heads, S, dtype=torch.float32, device=qkv.device)
            following = torch.empty(2, dtype=torch.int32, device=qkv.device)
            native.check(native.lib().tplr_attention_docs_bwd(
                qkv.data_ptr(), starts.data_ptr(), blocks.data_ptr(), out.data_ptr(), do.data_ptr(), lse.data_ptr(), delta.data_ptr(),
                following.data_ptr(), native.ptr(part), dqkv.data_ptr(), B, S, n_heads, n_kv, hd, ld, hd ** -0.5, OF.status_word(qkv.device).data_ptr(),
                native.stream_ptr()), "attention_docs_bwd")
        return dqkv, None, None, None, None


def _attention_documents(qkv, ld, starts, n_heads, n_kv, hd, keep):
    B, S, _ = qkv.shape
    with _on(qkv):
        out = torch.empty(B, S, n_heads * hd, dtype=qkv.dtype, device=qkv.device)
        lse = torch.empty(B, n_heads, S, dtype=torch.float32, device=qkv.device) if keep else None
        blocks = torch.empty(B * -(-S // 128), dtype=torch.int32, device=qkv.device) if keep else None
        native.check(native.lib().tplr_attention_docs_fwd(
            qkv.data_ptr(), starts.data_ptr(), out.data_ptr(), native.ptr(lse), native.ptr(blocks), B, S, n_heads, n_kv, hd, ld, n_heads * hd,
            hd ** -0.5, OF.status_word(qkv.device).data_ptr(), native.stream_ptr()), "attention_docs_fwd")
    return out, lse, blocks


_fallback_seen: set = set()


def _attention_documents_torch(qkv, starts, n_heads, n_kv, hd):
    B, S, _ = qkv.shape
    q, k, v = (t.float().transpose(1, 2) for t in OF._split_qkv(qkv, n_heads, n_kv, hd))
    if n_kv != n_heads:
        k, v = (t.repeat_interleave(n_heads // n_kv, dim=1) for t in (k, v))
    rows = torch.arange(S, device=qkv.device)
    seen = (rows[None, None, :] <= rows[None, :, None]) & (rows[None, None, :] >= starts[:, :, None])
    some = seen.any(-1, keepdim=True)
    # a row that sees nothing looks everywhere, and what it finds counts for nothing: no infinity meets its gradient
    p = torch.softmax((q @ k.transpose(2, 3) * hd ** -0.5).masked_fill(~(seen | ~some)[:, None], float("-inf")), dim=-1) * some[:, None]
    return (p @ v).to(qkv.dtype).transpose(1, 2).reshape(B, S, n_heads * hd)


def attention_documents(qkv: torch.Tensor, starts: torch.Tensor, n_heads: int, n_kv: int, hd: int) -> torch.Tensor:
    """Attention of ``qkv`` [B, S, (H + 2 KV) * hd] (query heads, key heads, value heads) in which row ``s`` sees the keys
    ``max(starts[b, s], 0) .. s``; returns [B, S, H * hd], zero in rows whose start lies behind them.  ``starts``: whole numbers [B, S].

    Every row has to hold finite numbers, one that nothing sees too, and so has the gradient: the rows of a block of 128 meet in the
    same products, where a weight of zero times an infinity is not zero.  The kernels (bf16, heads of 64 or 128) add nothing
    into memory: results and gradients have the same bits on every run.  Other heads and types take formulas in PyTorch, with the scores of
    every head in memory, which is said once."""
    tangent = _has_tangent(qkv)
    # operands that the kernels take as they are need no further look
    if qkv.is_cuda and not tangent and (host := native.host()) and (out := host.attention_documents(qkv, starts, n_heads, n_kv, hd, _word(qkv))) is not None:
        return out
    _heads("attention_documents", qkv, n_heads, n_kv, hd)
    B, S, C = qkv.shape
    if starts.shape != (B, S) or starts.is_floating_point() or starts.is_complex() or starts.dtype in (torch.bool, torch.uint64):
        raise ValueError(f"attention_documents: whole numbers [{B}, {S}] (not uint64) expected as starts, got {starts.dtype} {tuple(starts.shape)}")
    if starts.dtype in (torch.uint16, torch.uint32):
        starts = starts.to(torch.int64)
    _same_device("attention_documents", qkv, starts=starts)
    if not (qkv.is_cuda and qkv.dtype == torch.bfloat16 and hd in OF.OWN_HEAD_DIMS) or B * S == 0:
        if qkv.is_cuda and B * S > 0 and (hd, qkv.dtype) not in _fallback_seen:
            # said once per kind: the scores of every head are in memory there, and a run that is slow or out of memory for it should say why
            _fallback_seen.add((hd, qkv.dtype))
            warnings.warn(f"attention_documents: heads of {hd}, {qkv.dtype} are outside the own kernels (bf16, heads of 64 or 128); using formulas in "
                          f"PyTorch for them, with [B, H, S, S] scores in memory", stacklevel=2)
        return _attention_documents_torch(qkv, starts, n_heads, n_kv, hd)
    if tangent:
        raise _no_forward_mode("attention_documents")
    if starts.dtype != torch.int32:
        starts = starts.clamp(0, 2 ** 31 - 1).to(torch.int32) if starts.dtype == torch.int64 else starts.to(torch.int32)
    starts = starts.contiguous()
    if host := native.host():
        with _on(qkv):
            return host.attention_documents(qkv, starts, n_heads, n_kv, hd, _word(qkv))
    if torch.is_grad_enabled() and qkv.requires_grad:
        return _AttentionDocuments.apply(qkv, starts, n_heads, n_kv, hd)
    rows, ld = _packed_rows(qkv)
    return _attention_documents(rows, ld, starts, n_heads, n_kv, hd, False)[0]


# --------------------------------------------------------------------------- #
# norm of query and key heads, with the rotary embedding
# --------------------------------------------------------------------------- #
class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps, main_grad_q, main_grad_k):
        rows, ld = _packed_rows(qkv)
        wq, wk = OF._dense(wq), OF._dense(wk)
        ctx.save_for_backward(rows, wq, wk, cos, sin, positions)
        ctx.cfg = (n_heads, n_kv, hd, eps, ld, main_grad_q, main_grad_k)
        return _qk_norm_rope(rows, ld, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps)

    @staticmethod
    def backward(ctx, dy):
        rows, wq, wk, cos, sin, positions = ctx.saved_tensors
        n_heads, n_kv, hd, eps, ld, mg_q, mg_k = ctx.cfg
        B, S, C = rows.shape
        L = native.lib()
        with _on(rows):
            d, ldd = _packed_rows(dy)
            dx = torch.empty(B, S, C, dtype=rows.dtype, device=rows.device)
            part = torch.empty(L.tplr_qk_norm_rope_parts(B * S, n_heads, n_kv, hd), 2 * hd, dtype=torch.float32, device=rows.device)
            add, out, later = [], [], []
            for w, mg, needed in ((wq, mg_q, ctx.needs_input_grad[1]), (wk, mg_k, ctx.needs_input_grad[2])):
                direct = mg is not None and mg.dtype == torch.float32 and mg.is_contiguous() and mg.numel() == hd
                add.append(mg if direct else None)
                out.append(None if direct or not (needed or mg is not None) else torch.empty(w.shape, dtype=w.dtype, device=w.device))
                later.append(mg if mg is not None and not direct else None)
            native.check(L.tplr_qk_norm_rope_bwd(
                d.data_ptr(), ldd, rows.data_ptr(), ld, wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), native.ptr(positions),
                dx.data_ptr(), part.data_ptr(), native.ptr(out[0]), native.ptr(out[1]), native.ptr(add[0]), native.ptr(add[1]), B * S, S,
                cos.shape[0], n_heads, n_kv, hd, eps, OF.status_word(rows.device).data_ptr(), native.stream_ptr()), "qk_norm_rope_bwd")
            for i, mg in enumerate(later):
                if mg is not None:
                    mg.add_(out[i].view(mg.shape).to(mg.dtype))
                    out[i] = None
        return dx, out[0], out[1], None, None, None, None, None, None, None, None, None


def _qk_norm_rope(rows, ld, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps):
    B, S, C = rows.shape
    with _on(rows):
        y = torch.empty(B, S, C, dtype=rows.dtype, device=rows.device)
        native.check(native.lib().tplr_qk_norm_rope(
            rows.data_ptr(), ld, y.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), native.ptr(positions), B * S, S,
            cos.shape[0], n_heads, n_kv, hd, eps, OF.status_word(rows.device).data_ptr(), native.stream_ptr()), "qk_norm_rope")
    return y


class _AddMainGrad(torch.autograd.Function):
    """A weight as it is; its gradient goes onto ``main_grad``."""

    @staticmethod
    def forward(ctx, w, main_grad):
        ctx.main_grad = main_grad
        return w.view_as(w)

    @staticmethod
    def backward(ctx, dw):
        ctx.main_grad.add_(dw.view(ctx.main_grad.shape).to(ctx.main_grad.dtype))
        return None, None


def _qk_norm_rope_torch(qkv, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps):
    B, S, C = qkv.shape
    R = n_heads + n_kv
    x = qkv[..., :R * hd].float().reshape(B, S, R, hd)
    w = torch.cat((wq.float().reshape(1, hd).expand(n_heads, hd), wk.float().reshape(1, hd).expand(n_kv, hd)))
    z = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w
    at = torch.arange(S, device=qkv.device).expand(B, S) if positions is None else positions.long().clamp(0, cos.shape[0] - 1)
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    a, b = z[..., 0::2], z[..., 1::2]
    z = torch.stack((a * c - b * s, a * s + b * c), dim=-1).reshape(B, S, R * hd)
    return torch.cat((z.to(qkv.dtype), qkv[..., R * hd:]), dim=-1)


def qk_norm_rope(qkv: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, n_heads: int, n_kv: int, hd: int,
                 eps: float = 1e-5, positions: torch.Tensor | None = None, main_grad_q=None, main_grad_k=None) -> torch.Tensor:
    """``qkv`` [B, S, (H + 2 KV) * hd] with every query head normed and weighted by ``wq`` [hd], every key head by ``wk`` [hd], and both
    turned by the rotary embedding (interleaved pairs, tables of :func:`rope_tables`), in one pass; value heads as they are.
    ``positions``: int32 [B, S], the row of the tables that a token takes (its place in its document); without them its place
    in the sequence.  A position outside the tables takes their first or last row, and the kernels report it in the status word.
    One weight may serve both, and one buffer may take both gradients."""
    if main_grad_q is None:
        main_grad_q = getattr(wq, "main_grad", None)
    if main_grad_k is None:
        main_grad_k = getattr(wk, "main_grad", None)
    if any(b is not None and not torch.is_tensor(b) for b in (main_grad_q, main_grad_k)):
        if torch.is_grad_enabled() and (qkv.requires_grad or wq.requires_grad or wk.requires_grad):
            raise ValueError("qk_norm_rope: the weights' gradients are buffers here, not shards of other ranks")
        main_grad_q = main_grad_k = None
    tangent = _has_tangent(qkv, wq, wk, cos, sin)
    if qkv.is_cuda and not tangent and (host := native.host()) and (y := host.qk_norm_rope(qkv, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps, main_grad_q,
                                                                           main_grad_k, _word(qkv))) is not None:
        return y
    _heads("qk_norm_rope", qkv, n_heads, n_kv, hd)
    B, S, C = qkv.shape
    if wq.numel() != hd or wk.numel() != hd:
        raise ValueError(f"qk_norm_rope: weights of {hd} numbers expected, got {wq.numel()} and {wk.numel()}")
    if hd % 2 or cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != hd // 2 or cos.shape[0] < (S if positions is None else 1):
        raise ValueError(f"qk_norm_rope: tables of {hd // 2} columns{'' if positions is not None else f' and {S} rows'} expected, got "
                         f"{tuple(cos.shape)} and {tuple(sin.shape)}")
    if positions is not None and (positions.shape != (B, S) or positions.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"qk_norm_rope: int32 positions [{B}, {S}] expected, got {positions.dtype} {tuple(positions.shape)}")
    _same_device("qk_norm_rope", qkv, wq=wq, wk=wk, cos=cos, sin=sin, positions=positions)
    grad = torch.is_grad_enabled() and (qkv.requires_grad or wq.requires_grad or wk.requires_grad)
    for name, w, main_grad in (("main_grad_q", wq, main_grad_q), ("main_grad_k", wk, main_grad_k)):
        if grad and main_grad is not None:
            _fitting_buffer("qk_norm_rope", name, w, main_grad)
    # other buffers than dense ones in fp32 are added onto one behind the other
    if grad and all(t is not None and t.dtype == torch.float32 and t.is_contiguous() for t in (main_grad_q, main_grad_k)):
        q, k = ((t.data_ptr(), t.data_ptr() + t.nbytes) for t in (main_grad_q, main_grad_k))
        if q[0] != k[0] and q[0] < k[1] and k[0] < q[1]:
            raise ValueError("qk_norm_rope: main_grad_q and main_grad_k are one buffer or two, they do not overlap in part")
    if not (OF._native_ok(qkv, wq, wk) and hd % 8 == 0 and hd <= 256 and cos.dtype == sin.dtype == torch.float32) or B * S == 0:
        if main_grad_q is not None and wq.requires_grad:
            wq = _AddMainGrad.apply(wq, main_grad_q)
        if main_grad_k is not None and wk.requires_grad:
            wk = _AddMainGrad.apply(wk, main_grad_k)
        return _qk_norm_rope_torch(qkv, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps)
    if tangent:
        raise _no_forward_mode("qk_norm_rope")
    cos, sin = OF._dense(cos), OF._dense(sin)
    if positions is not None:
        positions = positions.clamp(-1, 2 ** 31 - 1).to(torch.int32).contiguous() if positions.dtype == torch.int64 else positions.contiguous()
    if host := native.host():
        with _on(qkv):
            y = host.qk_norm_rope(qkv, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps, main_grad_q, main_grad_k, _word(qkv))
        if y is not None:
            return y
    if grad:
        return _QKNormRope.apply(qkv, wq, wk, cos, sin, positions, n_heads, n_kv, hd, eps, main_grad_q, main_grad_k)
    rows, ld = _packed_rows(qkv)
    return _qk_norm_rope(rows, ld, OF._dense(wq), OF._dense(wk), cos, sin, positions, n_heads, n_kv, hd, eps)


# --------------------------------------------------------------------------- #
# cross entropy of an output projection whose logits are never stored
# --------------------------------------------------------------------------- #
def _chunks(T: int, V: int) -> list[tuple[int, int]]:
    """Runs of tokens whose weights fit ``CHUNK_BYTES``, of even size and whole tiles of 256."""
    most = max(256, CHUNK_BYTES // (2 * V) // 256 * 256)
    n = -(-T // most)
    size = -(-(-(-T // n)) // 256) * 256
    return [(a, min(T, a + size)) for a in range(0, T, size)]


class _Pieces:
    """Workspaces of the product with the softmax in pieces, for up to ``rows`` tokens."""

    def __init__(self, x2, w, rows: int, store: bool, scaled_rows: bool = False):
        self.V, self.D = w.shape
        dev = x2.device
        # rows on 128-byte boundaries, as the products' copies take them best: 1111 tokens, 1000 x 50257, dx 132 us with rows of 50264
        # elements, 105 with 50304, dw 107 and 92
        self.ld, self.ldxs = (-(-n // 64) * 64 for n in w.shape)
        self.e = torch.empty(rows, self.ld, dtype=torch.bfloat16, device=dev) if store else None
        # pieces of 64 columns or more, or fewer tokens with smaller ones, the last run's too
        least = min(64, native.lib().tplr_gemm2_softmax_columns(rows, self.V, self.D, int(store)))
        self.stats = torch.empty(rows * -(-self.V // least) * 2, dtype=torch.float32, device=dev)
        self.target = torch.empty(rows, dtype=torch.float32, device=dev)
        self.scale = torch.empty(rows, dtype=torch.float32, device=dev) if store else None
        self.xs = torch.empty(rows, self.ldxs, dtype=torch.bfloat16, device=dev) if scaled_rows else None

    def run(self, x, w, labels) -> tuple[int, int]:
        """(pieces of a row, columns of a piece)"""
        columns = native.lib().tplr_gemm2_softmax_columns(x.shape[0], self.V, self.D, int(self.e is not None))
        native.check(native.lib().tplr_gemm2_softmax(
            x.data_ptr(), w.data_ptr(), native.ptr(self.e), labels.data_ptr(), self.stats.data_ptr(), self.target.data_ptr(), x.shape[0], self.V,
            self.D, x.stride(0), w.stride(0), self.ld, OF.status_word(x.device).data_ptr(), native.stream_ptr()), "gemm2_softmax")
        return -(-self.V // columns), columns


def _token_losses(x2, w, labels, ignore_index):
    """Every token's loss, fp32."""
    T, V = x2.shape[0], w.shape[0]
    losses = torch.empty(T, dtype=torch.float32, device=x2.device)
    runs = _chunks(T, 16 * -(-V // 128))             # 8 bytes a piece
    ws = _Pieces(x2, w, runs[0][1], False)
    for a, b in runs:
        parts, columns = ws.run(x2[a:b], w, labels[a:b])
        native.check(native.lib().tplr_vocab_losses(ws.stats.data_ptr(), ws.target.data_ptr(), labels[a:].data_ptr(), losses[a:].data_ptr(),
                                                    b - a, parts, columns, V, ignore_index, native.stream_ptr()), "vocab_losses")
    return losses


def _gradients(x2, w, labels, ignore_index, row_grad, n_valid, grad_scale, losses, want_x, want_w, keep32):
    """(dx bf16, dw) of the sum of the rows' losses, each times its gradient; dw is bf16 where one run of tokens makes it, fp32
    where several add to it or ``keep32``."""
    T, D = x2.shape
    V = w.shape[0]
    runs = _chunks(T, V)
    ws = _Pieces(x2, w, runs[0][1], True, want_w)
    L, st = native.lib(), OF.status_word(x2.device).data_ptr()
    dx = torch.empty(T, D, dtype=x2.dtype, device=x2.device) if want_x else None
    dw = None
    for a, b in runs:
        x, e = x2[a:b], ws.e[:b - a, :V]
        parts, columns = ws.run(x, w, labels[a:b])
        native.check(L.tplr_vocab_rows(
            ws.e.data_ptr(), ws.ld, ws.stats.data_ptr(), ws.target.data_ptr(), labels[a:].data_ptr(),
            None if row_grad is None else row_grad[a:].data_ptr(), native.ptr(n_valid), grad_scale, x.data_ptr(), x.stride(0), native.ptr(ws.xs), ws.ldxs,
            ws.scale.data_ptr(), None if losses is None else losses[a:].data_ptr(), b - a, parts, columns, V, D, ignore_index,
            native.stream_ptr()), "vocab_rows")
        if want_x:
            cuts = L.tplr_gemm2_out_splits(b - a, D, V)
            planes = torch.empty(cuts * (-(-(b - a) // 32) * 32) * D, dtype=torch.float32, device=x2.device) if cuts > 1 else None
            native.check(L.tplr_gemm2_rows(ws.e.data_ptr(), w.data_ptr(), dx[a:].data_ptr(), native.ptr(planes), ws.scale.data_ptr(), b - a, D, V,
                                           ws.ld, w.stride(0), D, st, native.stream_ptr()), "gemm2_rows")
        if want_w:
            single = len(runs) == 1 and not keep32
            if dw is None:
                dw = torch.empty(V, D, dtype=torch.bfloat16 if single else torch.float32, device=x2.device)
                OF.gemm(e, ws.xs[:b - a, :D], a_mn=True, b_mn=True, out=dw)
            else:
                OF.gemm(e, ws.xs[:b - a, :D], a_mn=True, b_mn=True, out=dw, accumulate=True)
    return dx, dw


def _scaled(t, by, main_grad=None):
    """``t * by`` in bf16, or added onto ``main_grad``; ``by`` one fp32 number on the device."""
    direct = main_grad is not None and main_grad.dtype == torch.float32 and main_grad.is_contiguous() and main_grad.data_ptr() % 16 == 0
    out = main_grad if direct else torch.empty(t.shape, dtype=torch.bfloat16, device=t.device)
    native.check(native.lib().tplr_vocab_scale(t.data_ptr(), int(t.dtype == torch.float32), by.data_ptr(), out.data_ptr(), int(direct),
                                               t.numel(), native.stream_ptr()), "vocab_scale")
    if main_grad is None:
        return out
    if not direct:
        main_grad.add_(out.view(main_grad.shape).to(main_grad.dtype))
    return None


class _LinearCrossEntropy(torch.autograd.Function):
    """The mean: the gradients are made with the loss, run by run of tokens, while the run's weights are there."""

    @staticmethod
    def forward(ctx, x, w, labels, grad_scale, ignore_index, main_grad):
        x2, wd = _operand(x.reshape(-1, x.shape[-1])), _operand(w)
        T, V = x2.shape[0], wd.shape[0]
        with _on(x2):
            n_valid = torch.empty(1, dtype=torch.int32, device=x2.device)
            loss = torch.empty((), dtype=torch.float32, device=x2.device)
            L = native.lib()
            native.check(L.tplr_vocab_count(labels.data_ptr(), T, ignore_index, V, n_valid.data_ptr(), OF.status_word(x2.device).data_ptr(),
                                            native.stream_ptr()), "vocab_count")
            losses = torch.empty(T, dtype=torch.float32, device=x2.device)
            want_x, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
            dx, dw = _gradients(x2, wd, labels, ignore_index, None, n_valid, grad_scale, losses, want_x, want_w, main_grad is not None)
            native.check(L.tplr_vocab_mean(losses.data_ptr(), T, n_valid.data_ptr(), loss.data_ptr(), native.stream_ptr()), "vocab_mean")
        ctx.save_for_backward(dx, dw)
        ctx.shape, ctx.main_grad = x.shape, main_grad
        return loss

    @staticmethod
    def backward(ctx, dloss):
        dx, dw = ctx.saved_tensors
        d = dx if dx is not None else dw
        with _on(d):
            by = dloss.to(torch.float32)
            gx = None if dx is None else _scaled(dx, by).view(ctx.shape)
            gw = None if dw is None else _scaled(dw, by, ctx.main_grad)
        return gx, gw, None, None, None, None


class _LinearTokenLosses(torch.autograd.Function):
    """Every token's loss; its gradient is only known in the backward pass, which makes the product again."""

    @staticmethod
    def forward(ctx, x, w, labels, grad_scale, ignore_index, main_grad):
        x2, wd = _operand(x.reshape(-1, x.shape[-1])), _operand(w)
        with _on(x2):
            losses = _token_losses(x2, wd, labels, ignore_index)
        ctx.save_for_backward(x2, wd, labels)
        ctx.cfg = (x.shape, grad_scale, ignore_index, main_grad)
        return losses

    @staticmethod
    def backward(ctx, dlosses):
        x2, w, labels = ctx.saved_tensors
        shape, grad_scale, ignore_index, main_grad = ctx.cfg
        with _on(x2):
            g = (dlosses.float() * grad_scale).contiguous()
            dx, dw = _gradients(x2, w, labels, ignore_index, g, None, 1.0, None, ctx.needs_input_grad[0], ctx.needs_input_grad[1],
                                main_grad is not None)
            if dw is not None and (main_grad is not None or dw.dtype != torch.bfloat16):
                dw = _scaled(dw, torch.ones((), dtype=torch.float32, device=dw.device), main_grad)
        return None if dx is None else dx.view(shape), dw, None, None, None, None


def _operand(t: torch.Tensor) -> torch.Tensor:
    """A matrix as the products take it: rows in whole 16-byte pieces apart."""
    if t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < t.shape[1] or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _linear_cross_entropy_torch(x, w, labels, grad_scale, ignore_index, reduction):
    counts = (labels != ignore_index) & (labels >= 0) & (labels < w.shape[0])
    # a row that does not count may hold anything: no infinity meets its gradient of zero
    z = torch.where(counts[:, None], x.reshape(-1, x.shape[-1]).float(), 0.0) @ w.float().t()
    losses = torch.logsumexp(z, dim=1) - z.gather(1, labels.clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    losses = torch.where(counts, losses, 0.0)
    if reduction == "mean":
        losses = losses.sum() / counts.sum().clamp(min=1)
    return losses if grad_scale == 1.0 else losses.detach() + grad_scale * (losses - losses.detach())


def linear_cross_entropy(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, grad_scale: float = 1.0, ignore_index: int = -100,
                         main_grad=None, reduction: str = "mean") -> torch.Tensor:
    """Cross entropy (fp32) of the logits ``x @ w.T`` against ``labels``, without the logits in memory: ``x`` [.., D], ``w`` [V, D],
    ``labels`` [..] int64.  ``reduction``: the mean over ``labels != ignore_index`` (zero where there are none), or ``"none"``: every
    token's own, in the shape of ``labels``, zero where it is ignored.  A label that is neither ``ignore_index`` nor a column counts as ignored, and
    the kernels report it in the status word.  The gradient is ``grad_scale`` times the loss's, and the incoming one counts.

    The kernels hold ``exp(logit)`` (relative to a piece's largest where that is far from zero) for a run of tokens at a time
    (``CHUNK_BYTES``), from which the gradients of ``x`` and ``w`` are made at once; where nothing asks for a gradient, two numbers for
    every 64 or 128 columns.  A mean makes its gradients in the forward pass; the gradient of ``"none"`` costs the product a second time."""
    if main_grad is None:
        main_grad = getattr(w, "main_grad", None)
    if main_grad is not None and not torch.is_tensor(main_grad):
        if torch.is_grad_enabled() and w.requires_grad:
            raise ValueError("linear_cross_entropy: the weight's gradient is a buffer here, not shards of other ranks")
        main_grad = None
    mean, ignore_index, tangent = reduction == "mean", int(ignore_index), _has_tangent(x, w)
    host = native.host() if x.is_cuda and not tangent and (mean or reduction == "none") and OF.gemm_backend() == "tcgen05_2sm" else None
    if host and (out := host.linear_cross_entropy(x, w, labels, grad_scale, ignore_index, main_grad, mean, CHUNK_BYTES, _word(x))) is not None:
        return out
    if reduction not in ("mean", "none"):
        raise ValueError(f"linear_cross_entropy: reduction is 'mean' or 'none', got {reduction!r}")
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1] or w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError(f"linear_cross_entropy: rows [.., D] and a weight [V, D] expected, got {tuple(x.shape)} and {tuple(w.shape)}")
    if labels.shape != x.shape[:-1] or labels.is_floating_point() or labels.dtype == torch.bool:
        raise ValueError(f"linear_cross_entropy: labels {tuple(x.shape[:-1])} expected, got {labels.dtype} {tuple(labels.shape)}")
    _same_device("linear_cross_entropy", x, w=w, labels=labels)
    flat = labels.reshape(-1).contiguous().to(torch.int64)
    grad = torch.is_grad_enabled() and (x.requires_grad or w.requires_grad)
    if main_grad is not None and grad and w.requires_grad:
        _fitting_buffer("linear_cross_entropy", "main_grad", w, main_grad)
    T = flat.numel()
    if not OF._native_ok(x, w) or w.shape[1] % 8 or T == 0:
        if main_grad is not None and grad and w.requires_grad:
            w = _AddMainGrad.apply(w, main_grad)
        out = _linear_cross_entropy_torch(x, w, flat, float(grad_scale), ignore_index, reduction)
        return out if mean else out.view(labels.shape)
    if tangent:
        raise _no_forward_mode("linear_cross_entropy")
    if host:
        with _on(x):
            out = host.linear_cross_entropy(x, w, flat.view(labels.shape), grad_scale, ignore_index, main_grad, mean, CHUNK_BYTES, _word(x))
        if out is not None:
            return out
    if grad:
        node = _LinearCrossEntropy if mean else _LinearTokenLosses
        out = node.apply(x, w, flat, float(grad_scale), ignore_index, main_grad)
        return out if mean else out.view(labels.shape)
    x2, wd = _operand(x.detach().reshape(-1, x.shape[-1])), _operand(w.detach())
    with _on(x2):
        losses = _token_losses(x2, wd, flat, ignore_index)
        if reduction == "none":
            return losses.view(labels.shape)
        n_valid = torch.empty(1, dtype=torch.int32, device=x2.device)
        loss = torch.empty((), dtype=torch.float32, device=x2.device)
        native.check(native.lib().tplr_vocab_count(flat.data_ptr(), T, ignore_index, w.shape[0], n_valid.data_ptr(),
                                                   OF.status_word(x2.device).data_ptr(), native.stream_ptr()), "vocab_count")
        native.check(native.lib().tplr_vocab_mean(losses.data_ptr(), T, n_valid.data_ptr(), loss.data_ptr(), native.stream_ptr()), "vocab_mean")
    return loss
