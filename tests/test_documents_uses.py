"""Operators on packed documents in uses that are easily got wrong: forward mode, one buffer for two weights, graphs walked more than once,
labels that the model is sure of.  On the CPU the formulas, on the GPU the kernels."""

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
