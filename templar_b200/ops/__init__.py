"""Kernels of the framework: ``functional`` (autograd ops with a CPU path), ``quantized`` (activations in
8 bits), ``documents`` (sequences of several documents), ``native`` (ctypes bindings of the sm_100a library) and ``build`` (in-tree nvcc build)."""

from .documents import attention_documents, document_starts, linear_cross_entropy, qk_norm_rope
from .functional import (add_rmsnorm, attention, cross_entropy, embedding, gemm, gemm_backend, linear, rmsnorm, rope,
                         rope_tables, set_gemm_backend, swiglu)
from .quantized import (QuantRows, QuantWeight, add_rmsnorm_q8, add_rmsnorm_saved8, attention_block_saved8, dequantize_rows,
                        feed_forward_saved8, linear_q8, linear_saved8, quantize_rows, quantize_weight, swiglu_q8)

__all__ = ["add_rmsnorm", "attention", "cross_entropy", "embedding", "gemm", "gemm_backend", "linear", "rmsnorm", "rope",
           "rope_tables", "set_gemm_backend", "swiglu",
           "attention_documents", "document_starts", "linear_cross_entropy", "qk_norm_rope",
           "QuantRows", "QuantWeight", "add_rmsnorm_q8", "add_rmsnorm_saved8", "attention_block_saved8", "dequantize_rows",
           "feed_forward_saved8", "linear_q8", "linear_saved8", "quantize_rows", "quantize_weight", "swiglu_q8"]
