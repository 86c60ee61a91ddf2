// Cross entropy from the pieces that tplr_gemm2_softmax leaves of a row of logits z: (r_i, s_i) of every piece i, its whole reference and the
// sum of its e_ij = 2^(z_ij log2 e - r_i) but for the label's; the label's exponent a, relative to its own piece's reference r; and the e_ij in
// bf16.  With c the largest reference of the row, all weights but the label's t = sum_i s_i 2^(r_i - c), and the label's e = 2^(a + r - c):
//   s = t + e,   loss = log(s / e) = log1p(t / e),   d_ij = g * (e_ij 2^(r_i - c) / s - [ij is the label])
// with g the gradient of the row's loss.  d is the row's factor f = g / s times E, which is e_ij where the piece's reference is c, as
// it nearly always is, e_ij 2^(r_i - c) where it is not, and e - s = -t in the label's column.  Where the model is sure of the label, t has all its
// digits, and the difference of p and 1 would be little more than p's rounding.  So
//   dx = f * (E w),   dw = E^T (f x)
// and E is not read or written here but for the label's column and pieces of another reference.  f x is rounded to bf16, as d would be.
//
// A row whose label is ignored, or is no column, has loss and gradient zero.  Sums over rows and pieces are taken in one order.
//
// One B200, 1111 rows of 1000, 50257 columns: the product with the softmax 126 us, this file's pass over rows 11, dx 94 + 6, dw 79, count and mean 5
// each; logits stored, read and turned into their gradient would be 670 MB more, 100 us.
#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;

// out[0] = labels that count
__global__ void __launch_bounds__(1024) vocab_count_kernel(const long long* labels, long long T, long long ignore, int V, int* out,
                                                           unsigned int* status) {
  __shared__ int total;
  grid_wait();
  grid_release();
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  int n = 0;
  bool bad = false;
  for (long long i = threadIdx.x; i < T; i += blockDim.x) {
    const long long l = labels[i];
    if (l == ignore) continue;
    if (l < 0 || l >= V) bad = true; else ++n;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) atomicAdd(&total, n);               // whole numbers: the same in any order
  if (bad && status) atomicOr(status, TPLR_ST_BAD_INDEX);
  __syncthreads();
  if (threadIdx.x == 0) out[0] = total;
}

// log(s / e) of a row with t beside the label's e = 2^a: by t / e where the label is the more likely, else by the logarithm of s, as e may be zero.
__device__ __forceinline__ float row_loss(float t, float e, float a) {
  return t < e ? log1pf(t / e) : (log2f(t + e) - a) * 0.6931471805599453f;
}

// Loss of each row: a warp a row, or (WIDE) its block of eight, where there are no more rows than SMs: 30 rows of 1000 pieces, product
// and this, 20.6 us with a warp a row, 16.1 with a block.
template <bool WIDE>
__global__ void __launch_bounds__(256) vocab_losses_kernel(const float2* stats, const float* target, const long long* labels, float* losses,
                                                           long long T, int parts, int columns, int V, long long ignore) {
  __shared__ float red[2][8];
  grid_wait();
  grid_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = WIDE ? (long long)blockIdx.x : blockIdx.x * 8LL + warp;
  if (row >= T) return;
  const int first = WIDE ? (int)threadIdx.x : lane, step = WIDE ? 256 : 32;
  const long long label = labels[row];
  const bool counts = label != ignore && label >= 0 && label < V;
  float loss = 0.f;
  if (counts) {                                      // the same in all lanes, and all of a block's threads where it has one row
    const float2* st = stats + row * parts;
    const float own = target[row], ref = st[(int)label / columns].x;
    float m = -INFINITY;
#pragma unroll 4
    for (int i = first; i < parts; i += step) m = fmaxf(m, st[i].x);
    m = warp_max(m);
    if (WIDE) {
      if (lane == 0) red[0][warp] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, red[0][i]);
    }
    float s = 0.f;
#pragma unroll 4
    for (int i = first; i < parts; i += step) { const float2 v = st[i]; s += v.y * exp2f(v.x - m); }
    s = warp_sum(s);
    if (WIDE) {
      if (lane == 0) red[1][warp] = s;
      __syncthreads();
      s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += red[1][i];
    }
    const float a = own + (ref - m);
    loss = row_loss(s, exp2f(a), a);
  }
  if (WIDE ? threadIdx.x == 0 : lane == 0) losses[row] = loss;
}

// What both products need of a row (see above), a warp a row: f in row_scale, E in place of e, f x in xs; and the
// row's loss.  g = row_grad[row], or grad_scale / *n_valid.
__global__ void __launch_bounds__(256) vocab_rows_kernel(bf16* e, long long ld, const float2* stats, const float* target, const long long* labels,
                                                         const float* row_grad, const int* n_valid, float grad_scale, const bf16* x, long long ldx,
                                                         bf16* xs, long long ldxs, float* row_scale, float* losses, long long T, int parts, int columns, int V,
                                                         int D, long long ignore) {
  grid_wait();
  grid_release();
  const long long row = blockIdx.x * 8LL + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= T) return;
  const float2* st = stats + row * parts;
  bf16* er = e + row * ld;
  const long long label = labels[row];
  const bool counts = label != ignore && label >= 0 && label < V;
  float c = -INFINITY, low = INFINITY, t = 0.f, a = 0.f;
  for (int i = lane; i < parts; i += 32) { c = fmaxf(c, st[i].x); low = fminf(low, st[i].x); }
  c = warp_max(c);
  low = -warp_max(-low);
  for (int i = lane; i < parts; i += 32) { const float2 v = st[i]; t += v.y * exp2f(v.x - c); }
  t = warp_sum(t);
  if (counts) a = target[row] + (st[(int)label / columns].x - c);
  const float e1 = counts ? exp2f(a) : 0.f, s = t + e1;
  const float g = !counts ? 0.f : row_grad ? row_grad[row] : grad_scale / (float)max(n_valid[0], 1);
  const float f = counts ? g / s : 0.f;
  if (counts) {
    if (low < c) {                                   // the same in all lanes
      for (int i = 0; i < parts; ++i) {
        if (st[i].x == c) continue;
        const float by = exp2f(st[i].x - c);
        for (int k = i * columns + lane * 8; k < min(i * columns + columns, V); k += 256) {      // the columns behind V are nobody's
          uint4 q = *reinterpret_cast<uint4*>(er + k);
          uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(w[j] << 16) * by, __uint_as_float(w[j] & 0xffff0000u) * by);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *reinterpret_cast<uint4*>(er + k) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
    }
    if (lane == 0) {
      er[label] = __float2bfloat16(-t);
      if (losses) losses[row] = row_loss(t, e1, a);
    }
  } else {
    // what the row holds is multiplied by zero, which takes numbers
    if (!(s < INFINITY)) for (int k = lane * 8; k < V; k += 256) *reinterpret_cast<uint4*>(er + k) = make_uint4(0u, 0u, 0u, 0u);
    if (lane == 0 && losses) losses[row] = 0.f;
  }
  if (lane == 0) row_scale[row] = f;
  if (!xs) return;
  const uint4* xr = reinterpret_cast<const uint4*>(x + row * ldx);
  uint4* out = reinterpret_cast<uint4*>(xs + row * ldxs);
#pragma unroll 4
  for (int i = lane; i < D / 8; i += 32) {
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (counts) {
      q = xr[i];
      uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
      q = make_uint4(w[0], w[1], w[2], w[3]);
    }
    out[i] = q;
  }
}

// out = sum of x / max(*n_valid, 1)
__global__ void __launch_bounds__(1024) vocab_mean_kernel(const float* x, long long T, const int* n_valid, float* out) {
  __shared__ double red[32];
  grid_wait();
  grid_release();
  double s = 0.0;                                    // many rows' losses
  for (long long i = threadIdx.x; i < T; i += blockDim.x) s += (double)x[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  s = red[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (threadIdx.x == 0) out[0] = (float)(s / (double)max(n_valid[0], 1));
}

// y = x * (*by), from bf16 or fp32 to bf16, or onto fp32; eight values a thread.  In its own place x is left alone where the factor is 1, as
// that of a loss that is walked back from itself is: 50257 x 1000, 29 us otherwise.
template <class In, bool ADD>
__global__ void __launch_bounds__(256) vocab_scale_kernel(const In* x, const float* by, void* y, long long n8) {
  grid_wait();
  grid_release();
  const float f = *by;
  if (sizeof(In) == 2 && static_cast<const void*>(x) == y && f == 1.f) return;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n8; i += gridDim.x * 256LL) {
    float v[8];
    if (sizeof(In) == 2) {
      const uint4 q = reinterpret_cast<const uint4*>(x)[i];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) { v[2 * k] = __uint_as_float(w[k] << 16); v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
    } else {
      const float4 a = reinterpret_cast<const float4*>(x)[2 * i], b = reinterpret_cast<const float4*>(x)[2 * i + 1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    if (ADD) {
      float4* o = reinterpret_cast<float4*>(y) + 2 * i;
      float4 a = o[0], b = o[1];
      a.x += v[0] * f; a.y += v[1] * f; a.z += v[2] * f; a.w += v[3] * f;
      b.x += v[4] * f; b.y += v[5] * f; b.z += v[6] * f; b.w += v[7] * f;
      o[0] = a; o[1] = b;
    } else {
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k] * f, v[2 * k + 1] * f);
        r[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
      reinterpret_cast<uint4*>(y)[i] = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}
}  // namespace

// n_valid[0] = labels that are columns and not `ignore`
TPLR_API int tplr_vocab_count(const long long* labels, long long T, long long ignore, int V, int* n_valid, unsigned int* status, void* stream) {
  TPLR_ENTER();
  return (int)launch_pdl(vocab_count_kernel, 1, 1024, 0, (cudaStream_t)stream, labels, T, ignore, V, n_valid, status);
}

// losses [T] from tplr_gemm2_softmax's stats [T, parts], of columns each, and target [T]
TPLR_API int tplr_vocab_losses(const float* stats, const float* target, const long long* labels, float* losses, long long T, int parts, int columns,
                               int V, long long ignore, void* stream) {
  TPLR_ENTER();
  if (T <= 0) return 0;
  if (columns <= 0 || (long long)parts * columns < V) return -401;
  const bool wide = T <= tplr_sm_count();
  return (int)launch_pdl(wide ? vocab_losses_kernel<true> : vocab_losses_kernel<false>, (unsigned)(wide ? T : (T + 7) / 8), 256, 0, (cudaStream_t)stream,
                         reinterpret_cast<const float2*>(stats), target, labels, losses, T, parts, columns, V, ignore);
}

// What tplr_gemm2_softmax left of T rows, E [T, V] (rows of ld elements), made ready for the products of the gradients: dx = row_scale * (E w),
// dw = E^T xs.  x and xs [T, D] (rows of ldx and ldxs elements), xs or null; losses [T] may be null.  row_grad [T] the gradients of the rows'
// losses, or null: grad_scale / n_valid[0] for every row.  columns: of a piece.
TPLR_API int tplr_vocab_rows(void* E, long long ld, const float* stats, const float* target, const long long* labels, const float* row_grad,
                             const int* n_valid, float grad_scale, const void* x, long long ldx, void* xs, long long ldxs, float* row_scale, float* losses,
                             long long T, int parts, int columns, int V, int D, long long ignore, void* stream) {
  TPLR_ENTER();
  if (T <= 0) return 0;
  if ((ld % 8) || ld < V || (columns % 8) || columns <= 0 || (long long)parts * columns < V || (ldx % 8) || (ldxs % 8) || (xs && ldxs < D) || (D % 8) || (((uintptr_t)E | (uintptr_t)x | (uintptr_t)xs) & 15)) return -401;
  return (int)launch_pdl(vocab_rows_kernel, (unsigned)((T + 7) / 8), 256, 0, (cudaStream_t)stream, (bf16*)E, ld,
                         reinterpret_cast<const float2*>(stats), target, labels, row_grad, n_valid, grad_scale, (const bf16*)x, ldx, (bf16*)xs,
                         ldxs, row_scale, losses, T, parts, columns, V, D, ignore);
}

// loss[0] = sum of losses [T] / max(n_valid[0], 1)
TPLR_API int tplr_vocab_mean(const float* losses, long long T, const int* n_valid, float* loss, void* stream) {
  TPLR_ENTER();
  return (int)launch_pdl(vocab_mean_kernel, 1, 1024, 0, (cudaStream_t)stream, losses, T, n_valid, loss);
}

// y = x * by[0] for n (a multiple of 8) values, dense, on 16-byte boundaries: x bf16 or fp32, y bf16; or, of fp32 alone, y fp32 that is added onto
TPLR_API int tplr_vocab_scale(const void* x, int x_fp32, const float* by, void* y, int add_fp32, long long n, void* stream) {
  TPLR_ENTER();
  if (n <= 0) return 0;
  if ((n % 8) || (((uintptr_t)x | (uintptr_t)y) & 15) || (add_fp32 && !x_fp32)) return -401;
  const long long blocks = (n / 8 + 255) / 256, most = 8LL * tplr_sm_count();
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  cudaStream_t st = (cudaStream_t)stream;
  if (add_fp32) return (int)launch_pdl(vocab_scale_kernel<float, true>, grid, 256, 0, st, (const float*)x, by, y, n / 8);
  if (x_fp32) return (int)launch_pdl(vocab_scale_kernel<float, false>, grid, 256, 0, st, (const float*)x, by, y, n / 8);
  return (int)launch_pdl(vocab_scale_kernel<bf16, false>, grid, 256, 0, st, (const bf16*)x, by, y, n / 8);
}
