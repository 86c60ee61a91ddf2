// Entry points of the kernel library that the autograd nodes in C++ call (csrc_host/autograd.cpp), declared once: the CUDA
// sources define them against these declarations and the nodes take the types of their function pointers from them, so that a
// changed argument list does not compile on either side alone.  The builder hands both a number made from this file
// (TPLR_ABI), and the nodes refuse a library with another one.
#pragma once

extern "C" {
int tplr_abi();
int tplr_add_rmsnorm_fwd(const void* res, const void* delta, const void* w, void* h_out, void* y, float* rstd, long long T, int D,
                         float eps, void* stream);
int tplr_add_rmsnorm_bwd_v2(const void* dy, const void* x, const void* w, const float* rstd, const void* dres, void* dx, float* dw,
                            long long T, int D, unsigned int* status, void* stream);
int tplr_gemm2_bf16(const void* A, const void* B, void* C, int M, int N, int K, long long lda, long long ldb, long long ldc, int a_mn,
                    int b_mn, int epi, unsigned int* status, int max_pairs, void* stream);
int tplr_gemm2_acc_splits(int M, int N, int K);
int tplr_gemm2_acc_split(const void* A, const void* B, float* C, float* ws, int M, int N, int K, long long lda, long long ldb,
                         long long ldc, int a_mn, int b_mn, unsigned int* status, void* stream);
int tplr_gemm2_out_splits(int M, int N, int K);
int tplr_gemm2_bf16_split(const void* A, const void* B, void* C, float* ws, int M, int N, int K, long long lda, long long ldb,
                          long long ldc, int a_mn, int b_mn, unsigned int* status, void* stream);
int tplr_gemm2_swiglu(const void* X, const void* W, void* GU, void* H, int M, int F, int K, long long ldx, long long ldw, long long ldgu,
                      long long ldh, unsigned int* status, void* stream);
int tplr_gemm2_swiglu_bwd(const void* dY, const void* W2, const void* GU, void* dGU, int M, int F, int K, long long lddy,
                          long long ldw2, long long ldgu, long long lddgu, unsigned int* status, void* stream);
int tplr_gemm2_rope(const void* X, const void* W, void* QKV, int M, int N, int K, long long ldx, long long ldw, long long ldc,
                    const float* cosb, const float* sinb, int S, int rope_cols, int head_dim, unsigned int* status, void* stream);
int tplr_attention_fwd(const void* qkv, void* out, float* lse, int B, int S, int H, int KV, int head_dim, long long ld_qkv,
                       long long ld_o, float scale, unsigned int* status, void* stream);
int tplr_gemm2_attn_dout(const void* dY, const void* Wo, const void* O, void* dO, float* delta, int M, int N, int K, int S, int head_dim,
                         long long lddy, long long ldwo, long long ldo, long long lddo, unsigned int* status, void* stream);
int tplr_attention_bwd_scratch_cols(int B, int S, int H, int KV, int head_dim);
int tplr_attention_bwd_unrope_delta(const void* qkv, const void* out, const void* dout, const float* lse, float* delta, float* dq32,
                                    void* dqkv, int B, int S, int H, int KV, int head_dim, long long ld_qkv, long long ld_o,
                                    float scale, const float* cosb, const float* sinb, unsigned int* status, void* stream);
// rows in 8 bits
int tplr_quantize_rows(const void* x, long long ldx, void* q, long long ldq, float* scale, long long scale_row, long long scale_group,
                       long long T, int D, int group, void* stream);
int tplr_dequantize_rows(const void* q, long long ldq, const float* scale, long long scale_row, long long scale_group, int group,
                         const void* w, void* y, long long T, int D, void* stream);
int tplr_add_rmsnorm_q8(const void* res, const void* delta, const void* w, void* h_out, void* q, long long ldq, float* scale, long long T,
                        int D, float eps, void* stream);
int tplr_add_rmsnorm_saved8(const void* res, const void* delta, const void* w, void* h_out, void* y, void* q, long long ldq, float* scale,
                            long long scale_row, long long scale_group, float* rstd, long long T, int D, float eps, void* stream);
int tplr_rmsnorm_saved8_parts(long long T, int D);
int tplr_rmsnorm_saved8_bwd(const void* dy, const void* q, long long ldq, const float* scale, long long scale_row, long long scale_group,
                            const float* rstd, const void* w, const void* dres, void* dx, float* part, float* dw_add, void* dw_out,
                            long long T, int D, void* stream);
long long tplr_gemm_q8_workspace(int T, int N, int K);
int tplr_gemm_q8(const void* x, const void* w, const float* sx, const float* sw, void* y, void* ws, int T, int N, int K, long long ldx,
                 long long ldw, long long ldy, int out_fp32, unsigned int* status, void* stream);
int tplr_linear_q8_few(const void* x, const void* w, const float* sw, void* y, int T, int N, int K, long long ldx, long long ldw,
                       long long ldy, void* stream);
int tplr_gemm2_swiglu_saved8(const void* X, const void* W, void* Q, float* scale, void* H, int M, int F, int K, long long ldx, long long ldw,
                             long long ldq, long long ld_scale, long long ldh, unsigned int* status, void* stream);
int tplr_gemm2_swiglu_bwd_saved8(const void* dY, const void* W2, const void* Q, const float* scale, void* dGU, void* H, int M, int F, int K,
                                 long long lddy, long long ldw2, long long ldq, long long ld_scale, long long lddgu, long long ldh,
                                 unsigned int* status, void* stream);
// sequences of several documents
int tplr_attention_docs_fwd(const void* qkv, const int* starts, void* out, float* lse, int* blocks, int B, int S, int H, int KV, int head_dim,
                            long long ld_qkv, long long ld_o, float scale, unsigned int* status, void* stream);
int tplr_attention_docs_bwd_scratch_cols(int B, int S, int H, int KV, int head_dim);
int tplr_attention_docs_bwd(const void* qkv, const int* starts, const int* blocks, const void* out, const void* dout, const float* lse, float* delta,
                            int* next, float* part, void* dqkv, int B, int S, int H, int KV, int head_dim, long long ld_qkv, float scale,
                            unsigned int* status, void* stream);
int tplr_qk_norm_rope(const void* x, long long ldx, void* y, const void* wq, const void* wk, const float* cosb, const float* sinb,
                      const int* pos, long long tokens, int S, int table_rows, int n_q, int n_k, int hd, float eps, unsigned int* status,
                      void* stream);
int tplr_qk_norm_rope_parts(long long tokens, int n_q, int n_k, int hd);
int tplr_qk_norm_rope_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* wq, const void* wk, const float* cosb,
                          const float* sinb, const int* pos, void* dx, float* part, void* dwq, void* dwk, float* add_q, float* add_k,
                          long long tokens, int S, int table_rows, int n_q, int n_k, int hd, float eps, unsigned int* status, void* stream);
int tplr_gemm2_softmax_columns(int M, int N, int K, int store);
int tplr_gemm2_softmax(const void* X, const void* W, void* P, const long long* labels, float* stats, float* target, int M, int N, int K,
                       long long ldx, long long ldw, long long ldp, unsigned int* status, void* stream);
int tplr_gemm2_rows(const void* A, const void* B, void* C, float* ws, const float* row_scale, int M, int N, int K, long long lda,
                    long long ldb, long long ldc, unsigned int* status, void* stream);
int tplr_vocab_count(const long long* labels, long long T, long long ignore, int V, int* n_valid, unsigned int* status, void* stream);
int tplr_vocab_losses(const float* stats, const float* target, const long long* labels, float* losses, long long T, int parts, int columns, int V,
                      long long ignore, void* stream);
int tplr_vocab_rows(void* E, long long ld, const float* stats, const float* target, const long long* labels, const float* row_grad,
                    const int* n_valid, float grad_scale, const void* x, long long ldx, void* xs, long long ldxs, float* row_scale, float* losses, long long T,
                    int parts, int columns, int V, int D, long long ignore, void* stream);
int tplr_vocab_mean(const float* losses, long long T, const int* n_valid, float* loss, void* stream);
int tplr_vocab_scale(const void* x, int x_fp32, const float* by, void* y, int add_fp32, long long n, void* stream);
}
