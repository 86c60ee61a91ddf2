"""Forward passes of a LLaMA decoder with its projections in 8 bits: scoring text, logits for the next token.

:class:`Int8Llama` is made from a :class:`~templar_b200.models.llama.LlamaModel`; each block's four projections (packed
``[wq; wk; wv]``, ``wo``, packed ``[w1; w3]``, ``w2``) are laid out once as 8-bit codes with a scale for each output channel,
which is half their bytes, and multiply rows in 8 bits with a scale for each token.  Norms write those rows themselves, as
does the activation; embedding, attention and the output projection stay in the model's type.  The codes are a copy: after a
step of training a new one is made.
"""

from __future__ import annotations

import torch

from .. import ops
from ..ops import functional as OF
from .llama import LlamaModel


class Int8Llama:
    def __init__(self, model: LlamaModel):
        if getattr(model, "_param_gather", None) is not None:
            raise ValueError("Int8Llama: the model's weights are sharded and only present while a block runs; load them whole first")
        if getattr(model, "tp_world", 1) > 1 or model.output.weight.shape[0] != model.args.vocab_size:
            raise ValueError("Int8Llama: the model holds one rank's part of its heads, hidden units and (padded) vocabulary; "
                             "load the whole weights into a LlamaModel first")
        self.args = model.args
        self._model = model
        with torch.no_grad():
            self.blocks = [self._block(layer) for layer in model.layers.values()]

    @staticmethod
    def _block(layer) -> dict:
        att, ff = layer.attention, layer.feed_forward
        pack = lambda own, *ws: own[0] if own is not None else torch.cat([w.weight for w in ws])  # noqa: E731
        return {"wqkv": ops.quantize_weight(pack(att.packed, att.wq, att.wk, att.wv)), "wo": ops.quantize_weight(att.wo.weight),
                "w13": ops.quantize_weight(pack(ff.packed, ff.w1, ff.w3)), "w2": ops.quantize_weight(ff.w2.weight),
                "n1": layer.attention_norm, "n2": layer.ffn_norm, "attention": att}

    @torch.no_grad()
    def hidden_states(self, tokens: torch.Tensor) -> torch.Tensor:
        m = self._model
        cos, sin = m._rope(tokens.device)
        docs = m._documents(tokens)
        h, delta = OF.embedding(tokens, m.tok_embeddings.weight), None
        for b in self.blocks:
            h, rows = ops.add_rmsnorm_q8(h, delta, b["n1"].weight, b["n1"].eps)
            delta = ops.linear_q8(b["attention"].attend(ops.linear_q8(rows, b["wqkv"], h.dtype), cos, sin, docs), b["wo"])
            h, rows = ops.add_rmsnorm_q8(h, delta, b["n2"].weight, b["n2"].eps)
            delta = ops.linear_q8(ops.swiglu_q8(ops.linear_q8(rows, b["w13"], h.dtype)), b["w2"], h.dtype)
        if delta is None:
            return m.norm(h)
        return OF.add_rmsnorm(h, delta, m.norm.weight, m.norm.eps)[1]

    @torch.no_grad()
    def forward(self, tokens: torch.Tensor, labels: torch.Tensor | None = None) -> torch.Tensor:
        return self._model.output(self.hidden_states(tokens))

    __call__ = forward

    @torch.no_grad()
    def loss(self, tokens: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
        """Mean cross entropy over ``labels != ignore_index``."""
        if self.args.fused_loss:
            return ops.linear_cross_entropy(self.hidden_states(tokens), self._model.output.weight, labels, ignore_index=ignore_index)
        return OF.cross_entropy(self.forward(tokens), labels, 1.0, ignore_index)
