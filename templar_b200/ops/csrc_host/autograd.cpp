// Autograd nodes of the decoder block's operators, host side.
//
// The same sequences of kernel launches as the Python nodes in functional.py (_RMSNorm, _AddRMSNorm, _Linear, _FeedForward,
// _AttentionBlock), for bf16 CUDA operands that those nodes would hand to the own kernels.  A Python node costs its
// interpreter time twice (the backward half on the autograd thread, behind the interpreter lock): for one residual add and
// norm of a small batch that was 115 us around 9 us of kernels.  Here it is 80 us, most of it the engine's own.
//
// functional.py decides which calls come here (operand types, strides and alignment) and keeps its nodes for all others.
// Tensors are saved as saved variables only; the gradient buffers of the flat store are held by reference as there.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <atomic>

#include "../csrc/entries.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef long long ll;

std::atomic<ll> g_launches{0};

// C entry points of the kernel library
struct Entries {
  decltype(&tplr_add_rmsnorm_fwd) add_rmsnorm_fwd;
  decltype(&tplr_add_rmsnorm_bwd_v2) add_rmsnorm_bwd;
  decltype(&tplr_gemm2_bf16) gemm;
  decltype(&tplr_gemm2_acc_splits) acc_splits;
  decltype(&tplr_gemm2_acc_split) acc_split;
  decltype(&tplr_gemm2_out_splits) out_splits;
  decltype(&tplr_gemm2_bf16_split) gemm_split;
  decltype(&tplr_gemm2_swiglu) swiglu;
  decltype(&tplr_gemm2_swiglu_bwd) swiglu_bwd;
  decltype(&tplr_gemm2_rope) gemm_rope;
  decltype(&tplr_attention_fwd) attention_fwd;
  decltype(&tplr_gemm2_attn_dout) attn_dout;
  decltype(&tplr_attention_bwd_scratch_cols) bwd_scratch_cols;
  decltype(&tplr_attention_bwd_unrope_delta) attention_bwd;
  decltype(&tplr_quantize_rows) quantize;
  decltype(&tplr_dequantize_rows) dequantize;
  decltype(&tplr_add_rmsnorm_q8) add_rmsnorm_q8;
  decltype(&tplr_add_rmsnorm_saved8) add_rmsnorm_saved8;
  decltype(&tplr_rmsnorm_saved8_parts) rmsnorm_saved8_parts;
  decltype(&tplr_rmsnorm_saved8_bwd) rmsnorm_saved8_bwd;
  decltype(&tplr_gemm_q8_workspace) gemm_q8_workspace;
  decltype(&tplr_gemm_q8) gemm_q8;
  decltype(&tplr_linear_q8_few) linear_q8_few;
  decltype(&tplr_gemm2_swiglu_saved8) swiglu_saved8;
  decltype(&tplr_gemm2_swiglu_bwd_saved8) swiglu_bwd_saved8;
  decltype(&tplr_attention_docs_fwd) docs_fwd;
  decltype(&tplr_attention_docs_bwd_scratch_cols) docs_bwd_scratch_cols;
  decltype(&tplr_attention_docs_bwd) docs_bwd;
  decltype(&tplr_qk_norm_rope) qk_norm;
  decltype(&tplr_qk_norm_rope_parts) qk_norm_parts;
  decltype(&tplr_qk_norm_rope_bwd) qk_norm_bwd;
  decltype(&tplr_gemm2_softmax_columns) softmax_columns;
  decltype(&tplr_gemm2_softmax) softmax;
  decltype(&tplr_gemm2_rows) gemm_rows;
  decltype(&tplr_vocab_count) vocab_count;
  decltype(&tplr_vocab_losses) vocab_losses;
  decltype(&tplr_vocab_rows) vocab_rows;
  decltype(&tplr_vocab_mean) vocab_mean;
  decltype(&tplr_vocab_scale) vocab_scale;
} E;

void bind(const std::string& path) {
  void* so = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(so, "cannot open ", path, ": ", dlerror());
  auto get = [&](auto& fn, const char* name) {
    void* p = dlsym(so, name);
    TORCH_CHECK(p, name, " is missing in ", path);
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(p);
  };
  decltype(&tplr_abi) abi;
  get(abi, "tplr_abi");
  TORCH_CHECK(abi() == TPLR_ABI, path, " was built from other entry declarations than the autograd nodes; build both again");
  get(E.add_rmsnorm_fwd, "tplr_add_rmsnorm_fwd");
  get(E.add_rmsnorm_bwd, "tplr_add_rmsnorm_bwd_v2");
  get(E.gemm, "tplr_gemm2_bf16");
  get(E.acc_splits, "tplr_gemm2_acc_splits");
  get(E.acc_split, "tplr_gemm2_acc_split");
  get(E.out_splits, "tplr_gemm2_out_splits");
  get(E.gemm_split, "tplr_gemm2_bf16_split");
  get(E.swiglu, "tplr_gemm2_swiglu");
  get(E.swiglu_bwd, "tplr_gemm2_swiglu_bwd");
  get(E.gemm_rope, "tplr_gemm2_rope");
  get(E.attention_fwd, "tplr_attention_fwd");
  get(E.attn_dout, "tplr_gemm2_attn_dout");
  get(E.bwd_scratch_cols, "tplr_attention_bwd_scratch_cols");
  get(E.attention_bwd, "tplr_attention_bwd_unrope_delta");
  get(E.quantize, "tplr_quantize_rows");
  get(E.dequantize, "tplr_dequantize_rows");
  get(E.add_rmsnorm_q8, "tplr_add_rmsnorm_q8");
  get(E.add_rmsnorm_saved8, "tplr_add_rmsnorm_saved8");
  get(E.rmsnorm_saved8_parts, "tplr_rmsnorm_saved8_parts");
  get(E.rmsnorm_saved8_bwd, "tplr_rmsnorm_saved8_bwd");
  get(E.gemm_q8_workspace, "tplr_gemm_q8_workspace");
  get(E.gemm_q8, "tplr_gemm_q8");
  get(E.linear_q8_few, "tplr_linear_q8_few");
  get(E.swiglu_saved8, "tplr_gemm2_swiglu_saved8");
  get(E.swiglu_bwd_saved8, "tplr_gemm2_swiglu_bwd_saved8");
  get(E.docs_fwd, "tplr_attention_docs_fwd");
  get(E.docs_bwd_scratch_cols, "tplr_attention_docs_bwd_scratch_cols");
  get(E.docs_bwd, "tplr_attention_docs_bwd");
  get(E.qk_norm, "tplr_qk_norm_rope");
  get(E.qk_norm_parts, "tplr_qk_norm_rope_parts");
  get(E.qk_norm_bwd, "tplr_qk_norm_rope_bwd");
  get(E.softmax_columns, "tplr_gemm2_softmax_columns");
  get(E.softmax, "tplr_gemm2_softmax");
  get(E.gemm_rows, "tplr_gemm2_rows");
  get(E.vocab_count, "tplr_vocab_count");
  get(E.vocab_losses, "tplr_vocab_losses");
  get(E.vocab_rows, "tplr_vocab_rows");
  get(E.vocab_mean, "tplr_vocab_mean");
  get(E.vocab_scale, "tplr_vocab_scale");
}

void check(int err, const char* what) {
  g_launches.fetch_add(1, std::memory_order_relaxed);
  TORCH_CHECK(err == 0, what, " failed with CUDA error ", err);
}
void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
// the device's status word, as the kernels take it; the nodes keep the tensor and no pointer into it
unsigned* word(const Tensor& status) { return reinterpret_cast<unsigned*>(status.data_ptr()); }

// A gradient as the kernels read it: dense, on a 16-byte boundary.
Tensor dense(const Tensor& t) {
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
Tensor f32(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor bf16(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options()); }

// a tensor that takes no part in differentiation (a gradient buffer, the rotary tables); may be undefined
struct Aside { Tensor t; };
Tensor aside(AutogradContext* ctx, const char* key) {
  auto it = ctx->saved_data.find(key);
  return it == ctx->saved_data.end() ? Tensor() : it->second.toTensor();
}
void keep(AutogradContext* ctx, const char* key, const Aside& a) {
  if (a.t.defined()) ctx->saved_data[key] = a.t;
}

// out = op(a) op(b)^T as functional.gemm; epi 0: store bf16, 1: add into fp32
void gemm(const Tensor& a, const Tensor& b, const Tensor& out, bool a_mn, bool b_mn, int epi, const Tensor& status) {
  const ll M = a_mn ? a.size(1) : a.size(0), K = a_mn ? a.size(0) : a.size(1), N = b_mn ? b.size(1) : b.size(0);
  const ll plane = (M + 31) / 32 * 32 * N;             // workspace of one part of K, where K is cut
  if (epi == 0) {
    if (const ll parts = E.out_splits((int)M, (int)N, (int)K); parts > 1) {
      Tensor ws = f32({parts * plane}, a);
      check(E.gemm_split(a.data_ptr(), b.data_ptr(), out.data_ptr(), ws.data_ptr<float>(), (int)M, (int)N, (int)K, a.stride(0),
                         b.stride(0), out.stride(0), a_mn, b_mn, word(status), stream()),
            "tplr_gemm2_bf16_split");
      return;
    }
  } else if (reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0) {
    if (const ll parts = E.acc_splits((int)M, (int)N, (int)K); parts > 1) {
      Tensor ws = f32({(parts - 1) * plane}, a);
      check(E.acc_split(a.data_ptr(), b.data_ptr(), out.data_ptr<float>(), ws.data_ptr<float>(), (int)M, (int)N, (int)K, a.stride(0),
                        b.stride(0), out.stride(0), a_mn, b_mn, word(status), stream()),
            "tplr_gemm2_acc_split");
      return;
    }
  }
  check(E.gemm(a.data_ptr(), b.data_ptr(), out.data_ptr(), (int)M, (int)N, (int)K, a.stride(0), b.stride(0), out.stride(0), a_mn,
               b_mn, epi, word(status), 0, stream()),
        "tplr_gemm_bf16");
}
// dW of y = x W^T: added into the gradient buffer when there is one, else returned when wanted
Tensor weight_grad(const Tensor& buffer, const Tensor& dy2, const Tensor& x2, const Tensor& w, bool wanted, const Tensor& status) {
  if (buffer.defined()) {
    gemm(dy2, x2, buffer, true, true, 1, status);
    return Tensor();
  }
  if (!wanted) return Tensor();
  Tensor dw = bf16(w.sizes(), w);
  gemm(dy2, x2, dw, true, true, 0, status);
  return dw;
}
// t as a matrix.  The stride of a single row may be anything (and the matrix counts as contiguous); reshape gives it the row's length.
Tensor rows(const Tensor& t) { return t.dim() == 2 && t.size(0) != 1 ? t : t.reshape({-1, t.size(-1)}); }
// rows of a tensor whose last dimension is D; an integer division by zero would end the process
ll count_rows(const Tensor& t, ll D) {
  TORCH_CHECK(D > 0, "rows of no elements");
  return t.numel() / D;
}

// ------------------------------------------------------------------------------------------ norms
// inputs: x (or res, delta), w, buffer, eps, status
variable_list norm_backward(AutogradContext* ctx, const Tensor& dh, const Tensor& dy_in, const Tensor& h, const Tensor& w,
                            const Tensor& rstd, int w_index) {
  const Tensor status = aside(ctx, "status");
  const Tensor buffer = aside(ctx, "buffer");
  const ll D = h.size(-1), T = count_rows(h, D);
  const Tensor dy = dy_in.defined() ? dense(dy_in) : at::zeros_like(h);
  const Tensor dres = dh.defined() ? dense(dh) : Tensor();
  Tensor dx = at::empty_like(h);
  Tensor dw = buffer.defined() ? buffer : at::zeros({D}, h.options().dtype(at::kFloat));
  check(E.add_rmsnorm_bwd(dy.data_ptr(), h.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dres.defined() ? dres.data_ptr() : nullptr,
                          dx.data_ptr(), dw.data_ptr<float>(), T, (int)D, word(status), stream()),
        "add_rmsnorm_bwd");
  return {dx, buffer.defined() || !ctx->needs_input_grad(w_index) ? Tensor() : dw.to(w.scalar_type())};
}

struct RMSNorm : Function<RMSNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, Aside buffer, double eps, Aside status) {
    const ll D = x.size(-1), T = count_rows(x, D);
    Tensor y = at::empty_like(x), rstd = f32({T}, x);
    check(E.add_rmsnorm_fwd(x.data_ptr(), nullptr, w.data_ptr(), nullptr, y.data_ptr(), rstd.data_ptr<float>(), T, (int)D, (float)eps,
                            stream()),
          "rmsnorm_fwd");
    ctx->save_for_backward({x, w, rstd});
    keep(ctx, "buffer", buffer);
    keep(ctx, "status", status);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    auto r = norm_backward(ctx, Tensor(), g[0], s[0], s[1], s[2], 1);
    return {r[0], r[1], Tensor(), Tensor(), Tensor()};
  }
};

struct AddRMSNorm : Function<AddRMSNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& res, const Tensor& delta, const Tensor& w, Aside buffer, double eps,
                               Aside status) {
    const ll D = res.size(-1), T = count_rows(res, D);
    Tensor h = at::empty_like(res), y = at::empty_like(res), rstd = f32({T}, res);
    check(E.add_rmsnorm_fwd(res.data_ptr(), delta.data_ptr(), w.data_ptr(), h.data_ptr(), y.data_ptr(), rstd.data_ptr<float>(), T,
                            (int)D, (float)eps, stream()),
          "add_rmsnorm_fwd");
    ctx->save_for_backward({h, w, rstd});
    keep(ctx, "buffer", buffer);
    keep(ctx, "status", status);
    return {h, y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    auto r = norm_backward(ctx, g[0], g[1], s[0], s[1], s[2], 2);
    return {r[0], r[0], r[1], Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------------------ projections
struct Linear : Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, Aside buffer, Aside status) {
    auto shape = x.sizes().vec();
    shape.back() = w.size(0);
    Tensor y = bf16(shape, x);
    gemm(rows(x), w, y.view({-1, w.size(0)}), false, false, 0, status.t);
    ctx->save_for_backward({x, w});
    keep(ctx, "buffer", buffer);
    keep(ctx, "status", status);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor status = aside(ctx, "status");
    const Tensor dy2 = dense(rows(g[0])), x2 = rows(s[0]);
    Tensor dx;
    if (ctx->needs_input_grad(0)) {
      dx = bf16(s[0].sizes(), s[0]);
      gemm(dy2, s[1], dx.view({-1, s[1].size(1)}), false, true, 0, status);
    }
    return {dx, weight_grad(aside(ctx, "buffer"), dy2, x2, s[1], ctx->needs_input_grad(1), status), Tensor(), Tensor()};
  }
};

struct FeedForward : Function<FeedForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w13, const Tensor& w2, Aside buffer13, Aside buffer2,
                        Aside status) {
    const Tensor x2 = rows(x);
    const ll T = x2.size(0), F2 = w13.size(0), F = F2 / 2;
    Tensor gu = bf16({T, F2}, x), h = bf16({T, F}, x);
    check(E.swiglu(x2.data_ptr(), w13.data_ptr(), gu.data_ptr(), h.data_ptr(), (int)T, (int)F, (int)x2.size(1), x2.stride(0),
                   w13.stride(0), F2, F, word(status.t), stream()),
          "gemm2_swiglu");
    auto shape = x.sizes().vec();
    shape.back() = w2.size(0);
    Tensor y = bf16(shape, x);
    gemm(h, w2, y.view({-1, w2.size(0)}), false, false, 0, status.t);
    ctx->save_for_backward({x, w13, w2, gu, h});
    keep(ctx, "buffer13", buffer13);
    keep(ctx, "buffer2", buffer2);
    keep(ctx, "status", status);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w13 = s[1], &w2 = s[2], &gu = s[3], &h = s[4];
    const Tensor status = aside(ctx, "status");
    const Tensor dy2 = dense(rows(g[0])), x2 = rows(x);
    const ll T = gu.size(0), F = gu.size(1) / 2;
    Tensor dgu = at::empty_like(gu);
    check(E.swiglu_bwd(dy2.data_ptr(), w2.data_ptr(), gu.data_ptr(), dgu.data_ptr(), (int)T, (int)F, (int)dy2.size(1), dy2.stride(0),
                       w2.stride(0), gu.stride(0), dgu.stride(0), word(status), stream()),
          "gemm2_swiglu_bwd");
    Tensor dw2 = weight_grad(aside(ctx, "buffer2"), dy2, h, w2, ctx->needs_input_grad(2), status);
    Tensor dx;
    if (ctx->needs_input_grad(0)) {
      dx = bf16(x.sizes(), x);
      gemm(dgu, w13, dx.view({-1, w13.size(1)}), false, true, 0, status);
    }
    Tensor dw13 = weight_grad(aside(ctx, "buffer13"), dgu, x2, w13, ctx->needs_input_grad(1), status);
    return {dx, dw13, dw2, Tensor(), Tensor(), Tensor()};
  }
};

struct AttentionBlock : Function<AttentionBlock> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wqkv, const Tensor& wo, Aside buffer_qkv, Aside buffer_o,
                        Aside cos, Aside sin, int64_t heads, int64_t kv, int64_t hd, Aside status) {
    const ll B = x.size(0), S = x.size(1), C = wqkv.size(0), N = heads * hd;
    const Tensor x2 = rows(x);
    Tensor qkv = bf16({B, S, C}, x);
    check(E.gemm_rope(x2.data_ptr(), wqkv.data_ptr(), qkv.data_ptr(), (int)x2.size(0), (int)C, (int)x2.size(1), x2.stride(0),
                      wqkv.stride(0), C, cos.t.data_ptr<float>(), sin.t.data_ptr<float>(), (int)S, (int)((heads + kv) * hd), (int)hd,
                      word(status.t), stream()),
          "gemm2_rope");
    Tensor out = bf16({B, S, N}, x), lse = f32({B, heads, S}, x);
    check(E.attention_fwd(qkv.data_ptr(), out.data_ptr(), lse.data_ptr<float>(), (int)B, (int)S, (int)heads, (int)kv, (int)hd, C, N,
                          (float)std::pow((double)hd, -0.5), word(status.t), stream()),
          "attention_fwd");
    Tensor y = bf16({B, S, wo.size(0)}, x);
    gemm(out.view({-1, N}), wo, y.view({-1, wo.size(0)}), false, false, 0, status.t);
    ctx->save_for_backward({x, wqkv, wo, qkv, out, lse, cos.t, sin.t});
    keep(ctx, "buffer_qkv", buffer_qkv);
    keep(ctx, "buffer_o", buffer_o);
    keep(ctx, "status", status);
    ctx->saved_data["dims"] = std::vector<int64_t>{heads, kv, hd};
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &wqkv = s[1], &wo = s[2], &qkv = s[3], &out = s[4], &lse = s[5], &cos = s[6], &sin = s[7];
    const auto dims = ctx->saved_data["dims"].toIntVector();
    const int64_t heads = dims[0], kv = dims[1], hd = dims[2];
    const Tensor status = aside(ctx, "status");
    const ll B = qkv.size(0), S = qkv.size(1), C = qkv.size(2), T = B * S, N = heads * hd;
    const Tensor dy2 = dense(rows(g[0])), out2 = out.view({T, N});
    Tensor dO = bf16({T, N}, qkv), delta = f32({B, heads, S}, qkv);
    check(E.attn_dout(dy2.data_ptr(), wo.data_ptr(), out2.data_ptr(), dO.data_ptr(), delta.data_ptr<float>(), (int)T, (int)N,
                      (int)dy2.size(1), (int)S, (int)hd, dy2.stride(0), wo.stride(0), out2.stride(0), dO.stride(0), word(status),
                      stream()),
          "gemm2_attn_dout");
    Tensor dwo = weight_grad(aside(ctx, "buffer_o"), dy2, out2, wo, ctx->needs_input_grad(2), status);
    Tensor dqkv = at::empty_like(qkv);
    {
      Tensor scratch = f32({T * E.bwd_scratch_cols((int)B, (int)S, (int)heads, (int)kv, (int)hd)}, qkv);
      scratch.narrow(0, 0, T * N).zero_();                   // dQ accumulates; the parts behind it are written whole
      check(E.attention_bwd(qkv.data_ptr(), out.data_ptr(), dO.data_ptr(), lse.data_ptr<float>(), delta.data_ptr<float>(),
                            scratch.data_ptr<float>(), dqkv.data_ptr(), (int)B, (int)S, (int)heads, (int)kv, (int)hd, C, N,
                            (float)std::pow((double)hd, -0.5), cos.data_ptr<float>(), sin.data_ptr<float>(), word(status), stream()),
            "attention_bwd_unrope_delta");
    }
    const Tensor d2 = dqkv.view({T, C}), x2 = rows(x);
    Tensor dx;
    if (ctx->needs_input_grad(0)) {
      dx = bf16(x.sizes(), x);
      gemm(d2, wqkv, dx.view({-1, wqkv.size(1)}), false, true, 0, status);
    }
    Tensor dwqkv = weight_grad(aside(ctx, "buffer_qkv"), d2, x2, wqkv, ctx->needs_input_grad(1), status);
    return {dx, dwqkv, dwo, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------------------ rows in 8 bits
// The same calls as ops/quantized.py makes, for the operands that it hands here: bf16 CUDA tensors with contiguous columns.
constexpr ll GROUP = 64;
ll padded(ll n) { return (n + 15) / 16 * 16; }
Tensor int8(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kChar)); }
// x as rows of D with contiguous columns
Tensor dense_rows(const Tensor& x) {
  Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  return x2.stride(1) == 1 ? x2 : x2.contiguous();
}
// codes [T, D rounded up to 16] and scales [T, 1] or [T, groups]
std::pair<Tensor, Tensor> quantize(const Tensor& x, int group) {
  const Tensor x2 = dense_rows(x);
  const ll T = x2.size(0), D = x2.size(1);
  Tensor q = int8({T, padded(D)}, x), scale = f32({T, group ? (D + group - 1) / group : 1}, x);
  check(E.quantize(x2.data_ptr(), x2.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr<float>(), scale.stride(0), scale.stride(1), T,
                   (int)D, group, stream()),
        "quantize_rows");
  return {q, scale};
}
// the values of codes, in bf16: `shape` is that of the result, w may be undefined
Tensor dequantize(const Tensor& q, const Tensor& scale, ll group, at::IntArrayRef shape, const Tensor& w) {
  const at::AutoDispatchBelowADInplaceOrView guard;
  const ll D = shape.back();
  Tensor y = at::empty(shape, q.options().dtype(at::kBFloat16));
  const Tensor wc = w.defined() ? w.contiguous() : w;
  check(E.dequantize(q.data_ptr(), q.stride(0), scale.data_ptr<float>(), scale.stride(0), group ? scale.stride(1) : 0,
                     (int)(group ? group : D), wc.defined() ? wc.data_ptr() : nullptr, y.data_ptr(), q.size(0), (int)D, stream()),
        "dequantize_rows");
  return y;
}
void multiply_q8(const void* q, ll ldq, const float* sx, const Tensor& wq, const Tensor& ws, const Tensor& y, ll T, ll K, const Tensor& status) {
  const ll N = wq.size(0), n = E.gemm_q8_workspace((int)T, (int)N, (int)K);
  const Tensor parts = n ? at::empty({n}, y.options().dtype(at::kInt)) : Tensor();            // of a long inner dimension
  check(E.gemm_q8(q, wq.data_ptr(), sx, ws.data_ptr<float>(), y.data_ptr(), n ? parts.data_ptr() : nullptr, (int)T, (int)N, (int)K, ldq,
                  wq.stride(0), N, 0, word(status), stream()),
        "gemm_q8");
}
// x in 8 bits by rows, times an 8-bit weight; the codes live for this call alone, with their scales behind them
Tensor linear_q8(const Tensor& x, const Tensor& wq, const Tensor& ws, const Tensor& status) {
  const at::AutoDispatchBelowADInplaceOrView guard;
  const Tensor x2 = dense_rows(x);
  const ll T = x2.size(0), K = x2.size(1), N = wq.size(0), ldq = padded(K);
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = bf16(shape, x);
  if (T <= 8) {
    const int err = E.linear_q8_few(x2.data_ptr(), wq.data_ptr(), ws.data_ptr<float>(), y.data_ptr(), (int)T, (int)N, (int)K, x2.stride(0),
                                    wq.stride(0), N, stream());
    if (err != -111) {
      check(err, "linear_q8_few");
      return y;
    }
  }
  Tensor codes = int8({T * (ldq + 4)}, x);
  char* q = static_cast<char*>(codes.data_ptr());
  float* scale = reinterpret_cast<float*>(q + T * ldq);
  check(E.quantize(x2.data_ptr(), x2.stride(0), q, ldq, scale, 1, 1, T, (int)K, 0, stream()), "quantize_rows");
  multiply_q8(q, ldq, scale, wq, ws, y, T, K, status);
  return y;
}
// rows of codes that are there already: sx one scale a row, dense
Tensor linear_q8_rows(const Tensor& q, const Tensor& sx, at::IntArrayRef shape, const Tensor& wq, const Tensor& ws, const Tensor& status) {
  auto out = shape.vec();
  out.back() = wq.size(0);
  Tensor y = at::empty(out, q.options().dtype(at::kBFloat16));
  multiply_q8(q.data_ptr(), q.stride(0), sx.data_ptr<float>(), wq, ws, y, q.size(0), shape.back(), status);
  return y;
}
// codes [N, K] and scales [N] that the product takes as they are: rows, and every 16-byte piece of a row, inside the storage
bool weight_as_it_is(const Tensor& q, const Tensor& scale) {
  if (q.scalar_type() != at::kChar || q.dim() != 2 || scale.scalar_type() != at::kFloat || scale.dim() != 1 || q.device() != scale.device())
    return false;
  const ll N = q.size(0), K = q.size(1), ld = q.stride(0), wide = padded(K);
  return K > 0 && K <= 131072 && scale.size(0) == N && q.stride(1) == 1 && ld % 16 == 0 && ld >= wide && scale.is_contiguous() &&
         reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(scale.data_ptr()) % 16 == 0 &&
         q.storage_offset() + (N - 1) * ld + wide <= (ll)q.storage().nbytes();
}
bool bf16_cuda(const Tensor& t) { return t.is_cuda() && t.scalar_type() == at::kBFloat16; }
// nothing: operands that are not for the kernels, or not for this call, of which ops/quantized.py says more
std::optional<std::tuple<Tensor, Tensor, Tensor>> add_rmsnorm_q8(const Tensor& res, const std::optional<Tensor>& delta, const Tensor& w,
                                                                 double eps) {
  if (!bf16_cuda(res) || !bf16_cuda(w) || (delta && !(bf16_cuda(*delta) && delta->sizes() == res.sizes()))) return std::nullopt;
  if (res.dim() == 0 || res.size(-1) == 0 || w.dim() != 1 || w.size(0) != res.size(-1)) return std::nullopt;
  if (at::GradMode::is_enabled() && (res.requires_grad() || w.requires_grad() || (delta && delta->requires_grad()))) return std::nullopt;
  const at::AutoDispatchBelowADInplaceOrView guard;
  const Tensor x2 = rows(res).contiguous(), wc = w.contiguous(), d = delta ? delta->contiguous() : Tensor();
  const ll T = x2.size(0), D = x2.size(1);
  Tensor h = delta ? bf16(res.sizes(), res) : res, q = int8({T, padded(D)}, res), scale = f32({T, 1}, res);
  check(E.add_rmsnorm_q8(x2.data_ptr(), delta ? d.data_ptr() : nullptr, wc.data_ptr(), delta ? h.data_ptr() : nullptr, q.data_ptr(),
                         q.stride(0), scale.data_ptr<float>(), T, (int)D, (float)eps, stream()),
        "add_rmsnorm_q8");
  return std::make_tuple(h, q, scale);
}

// (h, y, codes, scales) of the training norm; delta undefined: h is the input's and not a result
struct Saved8 { Tensor h, y, q, scale, rstd; };
Saved8 add_rmsnorm_saved8(const Tensor& res, const Tensor& delta, const Tensor& w, double eps) {
  const Tensor x2 = rows(res).contiguous(), d = delta.defined() ? delta.contiguous() : delta;
  const ll T = x2.size(0), D = x2.size(1);
  Saved8 s;
  if (d.defined()) s.h = bf16(res.sizes(), res);
  s.y = bf16(res.sizes(), res);
  s.q = int8({T, padded(D)}, res);
  s.scale = f32({T, (D + GROUP - 1) / GROUP}, res);
  s.rstd = f32({T}, res);
  check(E.add_rmsnorm_saved8(x2.data_ptr(), d.defined() ? d.data_ptr() : nullptr, w.data_ptr(), d.defined() ? s.h.data_ptr() : nullptr,
                             s.y.data_ptr(), s.q.data_ptr(), s.q.stride(0), s.scale.data_ptr<float>(), s.scale.stride(0), s.scale.stride(1),
                             s.rstd.data_ptr<float>(), T, (int)D, (float)eps, stream()),
        "add_rmsnorm_saved8");
  return s;
}
// dx, dw (undefined where it went into the buffer or nothing asks for it) from the saved (q, scale, rstd, w)
std::pair<Tensor, Tensor> norm_saved8_backward(AutogradContext* ctx, const Tensor& dh, const Tensor& dy, int w_index) {
  auto s = ctx->get_saved_variables();
  const Tensor &q = s[0], &scale = s[1], &rstd = s[2], &w = s[3];
  if (!dy.defined()) return {dh, Tensor()};                  // only the sum was used
  const Tensor buffer = aside(ctx, "buffer"), g = dy.contiguous(), dres = dh.defined() ? dh.contiguous() : dh;
  const ll T = q.size(0), D = w.size(0);
  Tensor dx = bf16(dy.sizes(), dy), part = f32({E.rmsnorm_saved8_parts(T, (int)D) * D}, dy);
  Tensor dw;
  if (!buffer.defined() && ctx->needs_input_grad(w_index)) dw = T ? at::empty_like(w) : at::zeros_like(w);
  check(E.rmsnorm_saved8_bwd(g.data_ptr(), q.data_ptr(), q.stride(0), scale.data_ptr<float>(), scale.stride(0), scale.stride(1),
                             rstd.data_ptr<float>(), w.data_ptr(), dres.defined() ? dres.data_ptr() : nullptr, dx.data_ptr(),
                             part.data_ptr<float>(), buffer.defined() ? buffer.data_ptr<float>() : nullptr,
                             dw.defined() ? dw.data_ptr() : nullptr, T, (int)D, stream()),
        "rmsnorm_saved8_bwd");
  return {dx, dw};
}
struct RMSNormSaved8 : Function<RMSNormSaved8> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, Aside buffer, double eps) {
    ctx->set_materialize_grads(false);
    const Tensor wc = w.contiguous();
    Saved8 s = add_rmsnorm_saved8(x, Tensor(), wc, eps);
    ctx->save_for_backward({s.q, s.scale, s.rstd, wc});
    ctx->mark_non_differentiable({s.q, s.scale});
    keep(ctx, "buffer", buffer);
    return {s.y, s.q, s.scale};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto r = norm_saved8_backward(ctx, Tensor(), g[0], 1);
    return {r.first, r.second, Tensor(), Tensor()};
  }
};
struct AddRMSNormSaved8 : Function<AddRMSNormSaved8> {
  static variable_list forward(AutogradContext* ctx, const Tensor& res, const Tensor& delta, const Tensor& w, Aside buffer, double eps) {
    ctx->set_materialize_grads(false);
    const Tensor wc = w.contiguous();
    Saved8 s = add_rmsnorm_saved8(res, delta, wc, eps);
    ctx->save_for_backward({s.q, s.scale, s.rstd, wc});
    ctx->mark_non_differentiable({s.q, s.scale});
    keep(ctx, "buffer", buffer);
    return {s.h, s.y, s.q, s.scale};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto r = norm_saved8_backward(ctx, g[0], g[1], 2);
    return {r.first, r.first, r.second, Tensor(), Tensor()};
  }
};

// xq, xscale and, where the codes are those of a norm's rows, its weight stand for x until the backward pass
struct FeedForwardSaved8 : Function<FeedForwardSaved8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w13, const Tensor& w2, Aside buffer13, Aside buffer2,
                        Aside status, Aside xq, Aside xscale, Aside xweight) {
    const Tensor x2 = rows(x);
    const ll T = x2.size(0), F2 = w13.size(0), F = F2 / 2;
    if (!xq.t.defined()) std::tie(xq.t, xscale.t) = quantize(x2, GROUP);
    // scales of a group side by side for consecutive rows
    Tensor q = int8({T, F2}, x), scale = f32({2 * ((F + GROUP - 1) / GROUP), T}, x), h = bf16({T, F}, x);
    check(E.swiglu_saved8(x2.data_ptr(), w13.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), h.data_ptr(), (int)T, (int)F,
                          (int)x2.size(1), x2.stride(0), w13.stride(0), F2, T, F, word(status.t), stream()),
          "gemm2_swiglu_saved8");
    auto shape = x.sizes().vec();
    shape.back() = w2.size(0);
    Tensor y = bf16(shape, x);
    gemm(h, w2, y.view({-1, w2.size(0)}), false, false, 0, status.t);
    ctx->save_for_backward({xq.t, xscale.t, xweight.t, w13, w2, q, scale});
    keep(ctx, "buffer13", buffer13);
    keep(ctx, "buffer2", buffer2);
    keep(ctx, "status", status);
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &xq = s[0], &xscale = s[1], &xweight = s[2], &w13 = s[3], &w2 = s[4], &q = s[5], &scale = s[6];
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Tensor status = aside(ctx, "status"), buffer13 = aside(ctx, "buffer13");
    const Tensor dy2 = dense(rows(g[0]));
    const ll T = q.size(0), F2 = q.size(1), F = F2 / 2;
    Tensor dgu = bf16({T, F2}, dy2), dw2;
    {
      Tensor h = bf16({T, F}, dy2);
      check(E.swiglu_bwd_saved8(dy2.data_ptr(), w2.data_ptr(), q.data_ptr(), scale.data_ptr<float>(), dgu.data_ptr(), h.data_ptr(), (int)T,
                                (int)F, (int)dy2.size(1), dy2.stride(0), w2.stride(0), F2, T, F2, F, word(status), stream()),
            "gemm2_swiglu_bwd_saved8");
      dw2 = weight_grad(aside(ctx, "buffer2"), dy2, h, w2, ctx->needs_input_grad(2), status);
    }
    Tensor dx, dw13;
    if (ctx->needs_input_grad(0)) {
      dx = bf16(shape, dy2);
      gemm(dgu, w13, dx.view({-1, w13.size(1)}), false, true, 0, status);
    }
    if (buffer13.defined() || ctx->needs_input_grad(1))        // the product takes bf16: the values are rounded to it, as _input_again does
      dw13 = weight_grad(buffer13, dgu, dequantize(xq, xscale, GROUP, {T, w13.size(1)}, xweight), w13, true, status);
    return {dx, dw13, dw2, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ------------------------------------------------------------------------------------------ sequences of several documents
// A call whose operands the kernels take as they are comes straight here: None sends it to the checks of documents.py, which say what is
// wrong or bring it into shape.
typedef std::optional<Tensor> Maybe;
bool here(const Tensor& t, c10::DeviceIndex d) { return t.is_cuda() && t.get_device() == d; }
bool heads_fit(const Tensor& qkv, int64_t heads, int64_t kv, int64_t hd) {
  return qkv.dim() == 3 && qkv.scalar_type() == at::kBFloat16 && qkv.numel() > 0 && heads > 0 && kv > 0 && hd > 0 && heads % kv == 0 &&
         qkv.size(2) == (heads + 2 * kv) * hd;
}
bool buffer_fits(const Maybe& b, const Tensor& w) {
  return !b || (b->scalar_type() == at::kFloat && b->sizes() == w.sizes() && b->is_contiguous() && b->device() == w.device() &&
                reinterpret_cast<uintptr_t>(b->data_ptr()) % 16 == 0);
}
bool on_boundary(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor copy(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
float* ptr32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// [B, S, C] as rows evenly apart in whole 16-byte pieces, ld elements from one to the next (documents.py, _packed_rows)
Tensor packed(const Tensor& t, ll& ld) {
  const ll B = t.size(0), S = t.size(1), C = t.size(2);
  ld = S > 1 ? t.stride(1) : B > 1 ? t.stride(0) : C;
  if (t.stride(2) == 1 && ld >= C && ld % 8 == 0 && (B == 1 || t.stride(0) == S * ld) && on_boundary(t)) return t;
  ld = C;
  return copy(t);
}
// a matrix as the products take it (documents.py, _operand)
Tensor operand(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && on_boundary(t) ? t : copy(t);
}

// (out, lse, blocks); the last two for a backward pass alone
std::tuple<Tensor, Tensor, Tensor> docs_forward(const Tensor& qkv, ll ld, const Tensor& starts, int64_t heads, int64_t kv, int64_t hd,
                                                const Tensor& status, bool keep) {
  const ll B = qkv.size(0), S = qkv.size(1);
  Tensor out = bf16({B, S, heads * hd}, qkv), lse, blocks;
  if (keep) {
    lse = f32({B, heads, S}, qkv);
    blocks = at::empty({B * ((S + 127) / 128)}, starts.options());
  }
  check(E.docs_fwd(qkv.data_ptr(), starts.data_ptr<int>(), out.data_ptr(), ptr32(lse), keep ? blocks.data_ptr<int>() : nullptr, (int)B, (int)S,
                   (int)heads, (int)kv, (int)hd, ld, heads * hd, (float)std::pow((double)hd, -0.5), word(status), stream()),
        "attention_docs_fwd");
  return {out, lse, blocks};
}

struct AttentionDocuments : Function<AttentionDocuments> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv_in, Aside starts, int64_t heads, int64_t kv, int64_t hd, Aside status) {
    ll ld;
    const Tensor qkv = packed(qkv_in, ld);
    auto [out, lse, blocks] = docs_forward(qkv, ld, starts.t, heads, kv, hd, status.t, true);
    ctx->save_for_backward({qkv, starts.t, out, lse, blocks});
    keep(ctx, "status", status);
    ctx->saved_data["dims"] = std::vector<int64_t>{heads, kv, hd, ld};
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &qkv = s[0], &starts = s[1], &out = s[2], &lse = s[3], &blocks = s[4];
    const auto d = ctx->saved_data["dims"].toIntVector();
    const ll B = qkv.size(0), S = qkv.size(1), heads = d[0], kv = d[1], hd = d[2];
    const Tensor dout = dense(g[0]);
    Tensor dqkv = bf16({B, S, qkv.size(2)}, qkv), delta = f32({B, heads, S}, qkv), next = at::empty({2}, starts.options()), part;
    if (const ll cols = E.docs_bwd_scratch_cols((int)B, (int)S, (int)heads, (int)kv, (int)hd)) part = f32({B * S * cols}, qkv);
    check(E.docs_bwd(qkv.data_ptr(), starts.data_ptr<int>(), blocks.data_ptr<int>(), out.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(),
                     delta.data_ptr<float>(), next.data_ptr<int>(), ptr32(part), dqkv.data_ptr(), (int)B, (int)S, (int)heads, (int)kv, (int)hd, d[3],
                     (float)std::pow((double)hd, -0.5), word(aside(ctx, "status")), stream()),
          "attention_docs_bwd");
    return {dqkv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Maybe attention_documents(const Tensor& qkv, const Tensor& starts, int64_t heads, int64_t kv, int64_t hd, const Tensor& status) {
  const auto dev = c10::cuda::current_device();
  if (!here(qkv, dev) || !heads_fit(qkv, heads, kv, hd) || (hd != 64 && hd != 128) || !here(starts, dev) || starts.scalar_type() != at::kInt ||
      starts.dim() != 2 || starts.size(0) != qkv.size(0) || starts.size(1) != qkv.size(1) || !starts.is_contiguous())
    return std::nullopt;
  if (at::GradMode::is_enabled() && qkv.requires_grad()) return AttentionDocuments::apply(qkv, Aside{starts}, heads, kv, hd, Aside{status});
  ll ld;
  const Tensor rows = packed(qkv, ld);
  return std::get<0>(docs_forward(rows, ld, starts, heads, kv, hd, status, false));
}

Tensor qk_norm_forward(const Tensor& x, ll ld, const Tensor& wq, const Tensor& wk, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                       int64_t heads, int64_t kv, int64_t hd, double eps, const Tensor& status) {
  Tensor y = bf16(x.sizes(), x);
  check(E.qk_norm(x.data_ptr(), ld, y.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr<float>(), sin.data_ptr<float>(),
                  pos.defined() ? pos.data_ptr<int>() : nullptr, x.size(0) * x.size(1), (int)x.size(1), (int)cos.size(0), (int)heads, (int)kv,
                  (int)hd, (float)eps, word(status), stream()),
        "qk_norm_rope");
  return y;
}
struct QKNormRope : Function<QKNormRope> {
  static Tensor forward(AutogradContext* ctx, const Tensor& qkv, const Tensor& wq_in, const Tensor& wk_in, Aside cos, Aside sin, Aside pos,
                        int64_t heads, int64_t kv, int64_t hd, double eps, Aside buffer_q, Aside buffer_k, Aside status) {
    ll ld;
    const Tensor x = packed(qkv, ld), wq = dense(wq_in), wk = dense(wk_in);
    Tensor y = qk_norm_forward(x, ld, wq, wk, cos.t, sin.t, pos.t, heads, kv, hd, eps, status.t);
    ctx->save_for_backward({x, wq, wk, cos.t, sin.t, pos.t});
    keep(ctx, "buffer_q", buffer_q);
    keep(ctx, "buffer_k", buffer_k);
    keep(ctx, "status", status);
    ctx->saved_data["dims"] = std::vector<int64_t>{heads, kv, hd, ld};
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &wq = s[1], &wk = s[2], &cos = s[3], &sin = s[4], &pos = s[5];
    const auto d = ctx->saved_data["dims"].toIntVector();
    const ll B = x.size(0), S = x.size(1), hd = d[2];
    const Tensor bq = aside(ctx, "buffer_q"), bk = aside(ctx, "buffer_k");
    ll ldd;
    const Tensor dy = packed(g[0], ldd);
    Tensor dx = bf16(x.sizes(), x), part = f32({E.qk_norm_parts(B * S, (int)d[0], (int)d[1], (int)hd), 2 * hd}, x), dwq, dwk;
    if (!bq.defined() && ctx->needs_input_grad(1)) dwq = bf16({hd}, wq);
    if (!bk.defined() && ctx->needs_input_grad(2)) dwk = bf16({hd}, wk);
    check(E.qk_norm_bwd(dy.data_ptr(), ldd, x.data_ptr(), d[3], wq.data_ptr(), wk.data_ptr(), cos.data_ptr<float>(), sin.data_ptr<float>(),
                        pos.defined() ? pos.data_ptr<int>() : nullptr, dx.data_ptr(), part.data_ptr<float>(), ptr(dwq), ptr(dwk), ptr32(bq),
                        ptr32(bk), B * S, (int)S, (int)cos.size(0), (int)d[0], (int)d[1], (int)hd, (float)ctx->saved_data["eps"].toDouble(),
                        word(aside(ctx, "status")), stream()),
          "qk_norm_rope_bwd");
    return {dx, dwq.defined() ? dwq.view(wq.sizes()) : dwq, dwk.defined() ? dwk.view(wk.sizes()) : dwk, Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Maybe qk_norm_rope(const Tensor& qkv, const Tensor& wq, const Tensor& wk, const Tensor& cos, const Tensor& sin, const Maybe& at, int64_t heads,
                   int64_t kv, int64_t hd, double eps, const Maybe& bq, const Maybe& bk, const Tensor& status) {
  const auto dev = c10::cuda::current_device();
  if (!here(qkv, dev) || !heads_fit(qkv, heads, kv, hd) || hd % 8 || hd > 256 || !buffer_fits(bq, wq) || !buffer_fits(bk, wk)) return std::nullopt;
  for (const Tensor* w : {&wq, &wk})
    if (!here(*w, dev) || w->scalar_type() != at::kBFloat16 || w->numel() != hd) return std::nullopt;
  for (const Tensor* t : {&cos, &sin})
    if (!here(*t, dev) || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(1) != hd / 2 || t->size(0) != cos.size(0) ||
        !t->is_contiguous() || !on_boundary(*t))
      return std::nullopt;
  if (cos.size(0) < (at ? 1 : qkv.size(1))) return std::nullopt;
  // two weights may add into one buffer, but not into parts of each other's
  if (bq && bk && bq->data_ptr() != bk->data_ptr() && bq->data_ptr<float>() < bk->data_ptr<float>() + hd &&
      bk->data_ptr<float>() < bq->data_ptr<float>() + hd)
    return std::nullopt;
  if (at && (!here(*at, dev) || at->scalar_type() != at::kInt || at->dim() != 2 || at->size(0) != qkv.size(0) || at->size(1) != qkv.size(1) ||
             !at->is_contiguous()))
    return std::nullopt;
  const Aside pos{at ? *at : Tensor()}, buffer_q{bq ? *bq : Tensor()}, buffer_k{bk ? *bk : Tensor()};
  if (at::GradMode::is_enabled() && (qkv.requires_grad() || wq.requires_grad() || wk.requires_grad()))
    return QKNormRope::apply(qkv, wq, wk, Aside{cos}, Aside{sin}, pos, heads, kv, hd, eps, buffer_q, buffer_k, Aside{status});
  ll ld;
  const Tensor x = packed(qkv, ld);
  return qk_norm_forward(x, ld, dense(wq), dense(wk), cos, sin, pos.t, heads, kv, hd, eps, status);
}

// tokens of a run whose weights fit `bytes`: of even size, whole tiles of 256 (documents.py, _chunks)
ll run_length(ll T, ll V, ll bytes) {
  const ll most = std::max<ll>(256, bytes / (2 * V) / 256 * 256), n = (T + most - 1) / most;
  return ((T + n - 1) / n + 255) / 256 * 256;
}
// Workspaces of the product with the softmax in pieces (documents.py, _Pieces): one buffer of fp32, the weights, the scaled rows.
struct Pieces {
  Tensor numbers, e, xs;
  float *stats, *target, *scale;
  ll V, D, ld, ldxs;                                   // rows on 128-byte boundaries, as the products' copies take them best
  Pieces(const Tensor& x, const Tensor& w, ll rows, bool store, bool scaled)
      : V(w.size(0)), D(w.size(1)), ld((w.size(0) + 63) / 64 * 64), ldxs((w.size(1) + 63) / 64 * 64) {
    // pieces of 64 columns or more, or fewer tokens with smaller ones, the last run's too
    const ll least = std::min(64, E.softmax_columns((int)rows, (int)V, (int)D, store)), per = (V + least - 1) / least * 2;
    numbers = f32({rows * (per + 2)}, x);
    stats = numbers.data_ptr<float>();
    target = stats + rows * per;
    scale = target + rows;
    if (store) e = bf16({rows, ld}, x);
    if (scaled) xs = bf16({rows, ldxs}, x);
  }
  // columns of a piece
  ll run(const Tensor& x, ll T, const Tensor& w, const void* from, const ll* labels, const Tensor& status) {
    check(E.softmax(from, w.data_ptr(), ptr(e), labels, stats, target, (int)T, (int)V, (int)D, x.stride(0), w.stride(0), ld, word(status), stream()),
          "gemm2_softmax");
    return E.softmax_columns((int)T, (int)V, (int)D, e.defined());
  }
};
const char* row_of(const Tensor& x, ll at) { return static_cast<const char*>(x.data_ptr()) + 2 * at * x.stride(0); }

Tensor token_losses(const Tensor& x, const Tensor& w, const Tensor& labels, int64_t ignore, int64_t bytes, const Tensor& status) {
  const ll T = x.size(0), V = w.size(0), run = std::min(T, run_length(T, 16 * ((V + 127) / 128), bytes));
  Tensor losses = f32({T}, x);
  Pieces ws(x, w, run, false, false);
  const ll* lab = reinterpret_cast<const ll*>(labels.data_ptr<int64_t>());
  for (ll a = 0; a < T; a += run) {
    const ll n = std::min(run, T - a), columns = ws.run(x, n, w, row_of(x, a), lab + a, status);
    check(E.vocab_losses(ws.stats, ws.target, lab + a, losses.data_ptr<float>() + a, n, (int)((V + columns - 1) / columns), (int)columns,
                         (int)V, ignore, stream()),
          "vocab_losses");
  }
  return losses;
}
Tensor count_labels(const Tensor& labels, const Tensor& like, int64_t ignore, ll V, const Tensor& status) {
  Tensor n = at::empty({1}, like.options().dtype(at::kInt));
  check(E.vocab_count(reinterpret_cast<const ll*>(labels.data_ptr<int64_t>()), labels.numel(), ignore, (int)V, n.data_ptr<int>(), word(status), stream()),
        "vocab_count");
  return n;
}
Tensor mean_loss(const Tensor& losses, const Tensor& n_valid) {
  Tensor loss = f32({}, losses);
  check(E.vocab_mean(losses.data_ptr<float>(), losses.numel(), n_valid.data_ptr<int>(), loss.data_ptr<float>(), stream()), "vocab_mean");
  return loss;
}
// t * by in bf16, or added onto the buffer; `ours`: in t's own place, where nobody sees t again
Tensor scaled_by(const Tensor& t, const Tensor& by, const Tensor& buffer, at::IntArrayRef shape, bool ours) {
  ours = ours && t.scalar_type() == at::kBFloat16;
  Tensor out = buffer.defined() ? buffer : ours ? t.view(shape) : at::empty(shape, t.options().dtype(at::kBFloat16));
  check(E.vocab_scale(t.data_ptr(), t.scalar_type() == at::kFloat, by.data_ptr<float>(), out.data_ptr(), buffer.defined(), t.numel(), stream()),
        "vocab_scale");
  return buffer.defined() ? Tensor() : out;
}

struct LinearCrossEntropy : Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in, Aside labels, double grad_scale, int64_t ignore,
                        Aside buffer, int64_t bytes, Aside status) {
    const Tensor x = operand(rows(x_in)), w = operand(w_in);
    const ll T = x.size(0), V = w.size(0), D = w.size(1), run = std::min(T, run_length(T, V, bytes));
    const bool want_x = x_in.requires_grad(), want_w = w_in.requires_grad();
    Tensor n_valid = count_labels(labels.t, x, ignore, V, status.t), losses = f32({T}, x), dx, dw;
    Pieces ws(x, w, run, true, want_w);
    if (want_x) dx = bf16({T, D}, x);
    const bool single = run >= T && !buffer.t.defined();
    if (want_w) dw = single ? bf16({V, D}, x) : f32({V, D}, x);
    const ll* lab = reinterpret_cast<const ll*>(labels.t.data_ptr<int64_t>());
    for (ll a = 0; a < T; a += run) {
      const ll n = std::min(run, T - a), columns = ws.run(x, n, w, row_of(x, a), lab + a, status.t);
      check(E.vocab_rows(ws.e.data_ptr(), ws.ld, ws.stats, ws.target, lab + a, nullptr, n_valid.data_ptr<int>(), (float)grad_scale, row_of(x, a),
                         x.stride(0), ptr(ws.xs), ws.ldxs, ws.scale, losses.data_ptr<float>() + a, n, (int)((V + columns - 1) / columns), (int)columns,
                         (int)V, (int)D, ignore, stream()),
            "vocab_rows");
      if (want_x) {
        Tensor planes;
        if (const ll parts = E.out_splits((int)n, (int)D, (int)V); parts > 1) planes = f32({parts * ((n + 31) / 32 * 32) * D}, x);
        check(E.gemm_rows(ws.e.data_ptr(), w.data_ptr(), const_cast<char*>(row_of(dx, a)), ptr32(planes), ws.scale, (int)n, (int)D, (int)V, ws.ld,
                          w.stride(0), D, word(status.t), stream()),
              "gemm2_rows");
      }
      if (want_w) {
        const Tensor e = ws.e.narrow(0, 0, n).narrow(1, 0, V), xs = ws.xs.narrow(0, 0, n).narrow(1, 0, D);
        if (a > 0 || single) {
          gemm(e, xs, dw, true, true, a > 0 ? 1 : 0, status.t);
        } else {                                         // the first of several stores fp32
          check(E.gemm(e.data_ptr(), xs.data_ptr(), dw.data_ptr(), (int)V, (int)D, (int)n, ws.ld, ws.ldxs, D, 1, 1, 2, word(status.t), 0, stream()),
                "tplr_gemm_bf16");
        }
      }
    }
    ctx->save_for_backward({dx, dw});
    keep(ctx, "buffer", buffer);
    ctx->saved_data["shape"] = x_in.sizes().vec();
    return mean_loss(losses, n_valid);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    auto s = ctx->get_saved_variables();
    const Tensor by = g[0].to(at::kFloat);
    // A graph that is not kept lets go of what it saved behind this call, and cannot be walked again; a captured call can, by every replay.
    const bool ours = !torch::autograd::get_current_graph_task_keep_graph() &&
                      c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None;
    Tensor dx, dw;
    if (s[0].defined()) dx = scaled_by(s[0], by, Tensor(), ctx->saved_data["shape"].toIntVector(), ours);
    if (s[1].defined()) dw = scaled_by(s[1], by, aside(ctx, "buffer"), s[1].sizes(), ours);
    return {dx, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
// The mean, or every token's loss where nothing asks for a gradient; None also for a gradient of single tokens.
Maybe linear_cross_entropy(const Tensor& x, const Tensor& w, const Tensor& labels, double grad_scale, int64_t ignore, const Maybe& buffer, bool mean,
                           int64_t bytes, const Tensor& status) {
  const auto dev = c10::cuda::current_device();
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad());
  if (!here(x, dev) || !here(w, dev) || !here(labels, dev) || x.scalar_type() != at::kBFloat16 || w.scalar_type() != at::kBFloat16 ||
      labels.scalar_type() != at::kLong || !labels.is_contiguous() || x.dim() < 1 || w.dim() != 2 || w.numel() == 0 || x.numel() == 0 ||
      w.size(1) % 8 || x.size(-1) != w.size(1) || labels.sizes() != x.sizes().slice(0, x.dim() - 1) || (grad && !mean) || !buffer_fits(buffer, w))
    return std::nullopt;
  if (grad) return LinearCrossEntropy::apply(x, w, Aside{labels}, grad_scale, ignore, Aside{buffer ? *buffer : Tensor()}, bytes, Aside{status});
  const Tensor losses = token_losses(operand(rows(x)), operand(w), labels, ignore, bytes, status);
  return mean ? mean_loss(losses, count_labels(labels, losses, ignore, w.size(0), status)) : losses.view(labels.sizes());
}

Aside opt(const std::optional<Tensor>& t) { return Aside{t ? *t : Tensor()}; }

}  // namespace

PYBIND11_MODULE(tplr_host, m) {
  typedef py::call_guard<py::gil_scoped_release> nogil;
  m.def("bind", &bind);
  // what every call of an entry goes through
  m.def("check", [](int err, const std::string& what) { check(err, what.c_str()); }, nogil());
  m.def("launches", [] { return g_launches.load(std::memory_order_relaxed); });
  m.def("rmsnorm", [](const Tensor& x, const Tensor& w, const std::optional<Tensor>& buffer, double eps, const Tensor& status) {
    return RMSNorm::apply(x, w, opt(buffer), eps, Aside{status});
  }, nogil());
  m.def("add_rmsnorm", [](const Tensor& res, const Tensor& delta, const Tensor& w, const std::optional<Tensor>& buffer, double eps,
                          const Tensor& status) {
    auto r = AddRMSNorm::apply(res, delta, w, opt(buffer), eps, Aside{status});
    return std::make_tuple(r[0], r[1]);
  }, nogil());
  m.def("linear", [](const Tensor& x, const Tensor& w, const std::optional<Tensor>& buffer, const Tensor& status) {
    return Linear::apply(x, w, opt(buffer), Aside{status});
  }, nogil());
  m.def("feed_forward", [](const Tensor& x, const Tensor& w13, const Tensor& w2, const std::optional<Tensor>& b13,
                           const std::optional<Tensor>& b2, const Tensor& status) {
    return FeedForward::apply(x, w13, w2, opt(b13), opt(b2), Aside{status});
  }, nogil());
  m.def("attention_block", [](const Tensor& x, const Tensor& wqkv, const Tensor& wo, const std::optional<Tensor>& bq,
                              const std::optional<Tensor>& bo, const Tensor& cos, const Tensor& sin, int64_t heads, int64_t kv,
                              int64_t hd, const Tensor& status) {
    return AttentionBlock::apply(x, wqkv, wo, opt(bq), opt(bo), Aside{cos}, Aside{sin}, heads, kv, hd, Aside{status});
  }, nogil());
  m.def("quantize_rows", &quantize, nogil());
  m.def("dequantize_rows", [](const Tensor& q, const Tensor& scale, int64_t group, const std::vector<int64_t>& shape,
                              const std::optional<Tensor>& w) { return dequantize(q, scale, group, shape, w ? *w : Tensor()); }, nogil());
  m.def("linear_q8", &linear_q8, nogil());
  m.def("linear_q8_rows", [](const Tensor& q, const Tensor& sx, const std::vector<int64_t>& shape, const Tensor& wq, const Tensor& ws,
                             const Tensor& status) { return linear_q8_rows(q, sx, shape, wq, ws, status); }, nogil());
  m.def("weight_as_it_is", &weight_as_it_is);
  m.def("add_rmsnorm_q8", &add_rmsnorm_q8, nogil());
  m.def("rmsnorm_saved8", [](const Tensor& x, const Tensor& w, const std::optional<Tensor>& buffer, double eps) {
    auto r = RMSNormSaved8::apply(x, w, opt(buffer), eps);
    return std::make_tuple(r[0], r[1], r[2]);
  }, nogil());
  m.def("add_rmsnorm_saved8", [](const Tensor& res, const Tensor& delta, const Tensor& w, const std::optional<Tensor>& buffer, double eps) {
    auto r = AddRMSNormSaved8::apply(res, delta, w, opt(buffer), eps);
    return std::make_tuple(r[0], r[1], r[2], r[3]);
  }, nogil());
  m.def("feed_forward_saved8", [](const Tensor& x, const Tensor& w13, const Tensor& w2, const std::optional<Tensor>& b13,
                                  const std::optional<Tensor>& b2, const Tensor& status, const std::optional<Tensor>& xq,
                                  const std::optional<Tensor>& xscale, const std::optional<Tensor>& xweight) {
    return FeedForwardSaved8::apply(x, w13, w2, opt(b13), opt(b2), Aside{status}, opt(xq), opt(xscale), opt(xweight));
  }, nogil());
  m.def("attention_documents", &attention_documents, nogil());
  m.def("qk_norm_rope", &qk_norm_rope, nogil());
  m.def("linear_cross_entropy", &linear_cross_entropy, nogil());
}
