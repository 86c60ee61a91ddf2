// Norm of every query and key head together with the rotary embedding, on a packed projection [tokens, (H + 2 KV) * hd]: for each
// head x of q and k
//   z = x * rsqrt(mean(x^2) + eps) * w,   the pairs (2i, 2i + 1) of z turned by the angle of the token's position,
// value heads as they are.  Backward, with u the gradient turned back by the same angle, xh = x * rsqrt(..), g = u * w:
//   dx = rsqrt(..) * (g - xh * mean(g * xh)),   dw = sum over tokens and heads of u * xh.
// All of it in fp32, rounded once where it is stored.  Nothing is kept for the backward pass but the projection itself.
//
// Bound by memory, so a thread moves 16-byte pieces: LANES (8, 16 or 32) of them are a head, and a warp takes 32 / LANES
// neighbouring heads at a time, a few such steps in flight, of one token: its angles are read once for all of them.
//
// One B200, 16384 tokens, 16 + 2 x 16 heads of 128: forward 67 us for 403 MB (6.0 TB/s; a pair of kernels, norm and rotation, would move it twice),
// backward 102 for 540 MB (5.3 TB/s, 122 registers, instruction issue at 54 %) and 8 for the sums of its blocks.  30 tokens: 2.4 us, a launch.
#include "common.cuh"

namespace {
typedef __nv_bfloat16 bf16;

constexpr int WARPS = 4;             // of a block

struct QkNorm {
  const bf16* x; long long ldx;      // packed projection
  const bf16* dy; long long lddy;    // backward: the gradient of y
  bf16* y;                           // y, or dx; dense rows
  const bf16 *wq, *wk;
  const float *cosb, *sinb;          // [table_rows, hd / 2]
  const int* pos;                    // [tokens], or null: the row of its sequence of S
  long long tokens;
  int S, table_rows, n_q, n_k, hd;
  float eps, inv_hd;
  int chunks;                        // pieces of work of a token: its heads in runs of STEPS * 32 / LANES
  float* part;                       // backward: [blocks, 2 * hd] sums of dwq | dwk
  unsigned int* status;
};

__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) { f[2 * e] = __uint_as_float(w[e] << 16); f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    w[e] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int LANES> __device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cosines and sines of this lane's four pairs at the token's position; a position outside the tables is reported and takes their edge
__device__ __forceinline__ void angles(const QkNorm& p, long long tok, int l, bool on, float4& c, float4& s) {
  int at = p.pos ? p.pos[tok] : (int)(tok % p.S);
  if (at < 0 || at >= p.table_rows) {
    if (l == 0 && p.status) atomicOr(p.status, TPLR_ST_BAD_INDEX);
    at = at < 0 ? 0 : p.table_rows - 1;
  }
  c = s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (on) {
    const long long o = (long long)at * (p.hd / 2) + l * 4;
    c = *reinterpret_cast<const float4*>(p.cosb + o);
    s = *reinterpret_cast<const float4*>(p.sinb + o);
  }
}

template <int LANES, int STEPS>
__global__ void __launch_bounds__(WARPS * 32) qk_norm_fwd_kernel(const QkNorm p) {
  grid_wait();
  grid_release();
  constexpr int HEADS = 32 / LANES;                  // of a step
  const int lane = threadIdx.x & 31, l = lane % LANES;
  const long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const long long tok = item / p.chunks;
  if (tok >= p.tokens) return;                       // the whole warp
  const int first = (int)(item - tok * p.chunks) * STEPS * HEADS, mine = first + lane / LANES;
  const int rot = p.n_q + p.n_k, total = rot + p.n_k;
  const bool on = l * 8 < p.hd;
  const bf16* x = p.x + tok * p.ldx + l * 8;
  bf16* y = p.y + tok * (long long)total * p.hd + l * 8;
  uint4 v[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int head = mine + i * HEADS;
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (on && head < total) v[i] = *reinterpret_cast<const uint4*>(x + head * p.hd);
  }
  if (first < rot) {                                 // warp-uniform
    float4 c, s;
    angles(p, tok, l, on, c, s);
    uint4 wq = make_uint4(0u, 0u, 0u, 0u), wk = wq;
    if (on) { wq = *reinterpret_cast<const uint4*>(p.wq + l * 8); wk = *reinterpret_cast<const uint4*>(p.wk + l * 8); }
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (first + i * HEADS >= rot) break;           // warp-uniform: value heads only from here on
      const int head = mine + i * HEADS;
      float f[8], w[8], sq = 0.f;
      unpack(v[i], f);
      unpack(head < p.n_q ? wq : wk, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(f[e], f[e], sq);
      const float r = rsqrtf(head_sum<LANES>(sq) * p.inv_hd + p.eps);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = f[2 * e] * r * w[2 * e], b = f[2 * e + 1] * r * w[2 * e + 1];
        f[2 * e] = a * cc[e] - b * ss[e];
        f[2 * e + 1] = a * ss[e] + b * cc[e];
      }
      if (head < rot) v[i] = pack(f);
    }
  }
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int head = mine + i * HEADS;
    if (on && head < total) *reinterpret_cast<uint4*>(y + head * p.hd) = v[i];
  }
}

template <int LANES, int STEPS>
__global__ void __launch_bounds__(WARPS * 32, 4) qk_norm_bwd_kernel(const QkNorm p) {
  __shared__ float sums[WARPS * (32 / LANES)][2][LANES * 8];
  grid_wait();
  grid_release();
  constexpr int HEADS = 32 / LANES;
  const int lane = threadIdx.x & 31, l = lane % LANES, warp = threadIdx.x >> 5;
  const int rot = p.n_q + p.n_k, total = rot + p.n_k;
  const bool on = l * 8 < p.hd;
  float aq[8] = {}, ak[8] = {};                      // this lane's sums for the two weights
  const long long items = p.tokens * p.chunks;
  for (long long item = (long long)blockIdx.x * WARPS + warp; item < items; item += (long long)gridDim.x * WARPS) {
    const long long tok = item / p.chunks;
    const int first = (int)(item - tok * p.chunks) * STEPS * HEADS, mine = first + lane / LANES;
    const bf16* x = p.x + tok * p.ldx + l * 8;
    const bf16* dy = p.dy + tok * p.lddy + l * 8;
    bf16* dx = p.y + tok * (long long)total * p.hd + l * 8;
    uint4 v[STEPS], d[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int head = mine + i * HEADS;
      v[i] = d[i] = make_uint4(0u, 0u, 0u, 0u);
      if (on && head < rot) v[i] = *reinterpret_cast<const uint4*>(x + head * p.hd);
      if (on && head < total) d[i] = *reinterpret_cast<const uint4*>(dy + head * p.hd);
    }
    if (first < rot) {                               // warp-uniform
      float4 c, s;
      angles(p, tok, l, on, c, s);
      uint4 wq = make_uint4(0u, 0u, 0u, 0u), wk = wq;
      if (on) { wq = *reinterpret_cast<const uint4*>(p.wq + l * 8); wk = *reinterpret_cast<const uint4*>(p.wk + l * 8); }
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (first + i * HEADS >= rot) break;         // warp-uniform
        const int head = mine + i * HEADS;
        const bool is_q = head < p.n_q;
        float f[8], u[8], w[8], sq = 0.f, gx = 0.f;
        unpack(v[i], f);
        unpack(d[i], u);
        unpack(is_q ? wq : wk, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {                // turned back
          const float a = u[2 * e], b = u[2 * e + 1];
          u[2 * e] = a * cc[e] + b * ss[e];
          u[2 * e + 1] = b * cc[e] - a * ss[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sq = fmaf(f[e], f[e], sq);
          w[e] *= u[e];                              // g
          gx = fmaf(w[e], f[e], gx);
        }
        sq = head_sum<LANES>(sq);
        gx = head_sum<LANES>(gx);
        const float r = rsqrtf(sq * p.inv_hd + p.eps), m = gx * r * r * p.inv_hd;      // xh * mean(g * xh) = x * m * r
        if (head < rot) {                            // a value head in the same step has no part in the sums
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float t = u[e] * (f[e] * r);
            if (is_q) aq[e] += t; else ak[e] += t;
            f[e] = r * fmaf(-f[e], m, w[e]);
          }
          d[i] = pack(f);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int head = mine + i * HEADS;
      if (on && head < total) *reinterpret_cast<uint4*>(dx + head * p.hd) = d[i];
    }
  }
  const int row = warp * HEADS + lane / LANES;
#pragma unroll
  for (int e = 0; e < 8; ++e) { sums[row][0][l * 8 + e] = aq[e]; sums[row][1][l * 8 + e] = ak[e]; }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.hd; i += WARPS * 32) {
    const int which = i >= p.hd, col = i - which * p.hd;
    float t = 0.f;
#pragma unroll 4
    for (int k = 0; k < WARPS * HEADS; ++k) t += sums[k][which][col];
    p.part[(long long)blockIdx.x * 2 * p.hd + i] = t;
  }
}

// The blocks' sums added in one order, 32 columns a block: into out (bf16) or onto add (fp32), for wq and for wk.  Where both have the same
// buffer (one weight for queries and keys) a thread has both sums of an element: two threads that add onto it could lose one.
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* part, int blocks, int hd, bf16* dwq, bf16* dwk, float* add_q,
                                                          float* add_k) {
  __shared__ float red[32][33];
  grid_wait();
  grid_release();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), row = threadIdx.x >> 5;
  const bool both = add_q && add_q == add_k;
  const int cols = both ? hd : 2 * hd;
  float t = 0.f;
  if (col < cols) {
    for (int k = row; k < blocks; k += 32) t += part[(long long)k * 2 * hd + col];
    if (both)
      for (int k = row; k < blocks; k += 32) t += part[(long long)k * 2 * hd + hd + col];
  }
  red[row][threadIdx.x & 31] = t;
  __syncthreads();
  if (row != 0 || col >= cols) return;
  t = 0.f;
#pragma unroll
  for (int k = 0; k < 32; ++k) t += red[k][threadIdx.x & 31];
  const bool is_q = col < hd;
  const int at = is_q ? col : col - hd;
  if (float* add = is_q ? add_q : add_k) add[at] += t;
  else if (bf16* out = is_q ? dwq : dwk) out[at] = __float2bfloat16(t);
}

bool fits(const QkNorm& p) {
  return p.hd > 0 && p.hd % 8 == 0 && p.hd <= 256 && p.n_q >= 0 && p.n_k >= 0 && p.S > 0 && p.table_rows > 0 && p.ldx % 8 == 0 &&
         p.lddy % 8 == 0 && !(((uintptr_t)p.x | (uintptr_t)p.dy | (uintptr_t)p.y | (uintptr_t)p.wq | (uintptr_t)p.wk | (uintptr_t)p.cosb |
                               (uintptr_t)p.sinb) & 15);
}
constexpr int FWD_STEPS = 4, BWD_STEPS = 4;
int lanes_of(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }
int chunks_of(int n_q, int n_k, int hd, int steps) {
  const int heads = steps * 32 / lanes_of(hd);
  return (n_q + 2 * n_k + heads - 1) / heads;
}
// Blocks of the backward pass: as many as are resident at a time, each of which leaves one row of sums.
int bwd_blocks(long long tokens, int n_q, int n_k, int hd) {
  const long long all = (tokens * chunks_of(n_q, n_k, hd, BWD_STEPS) + WARPS - 1) / WARPS, most = 4LL * tplr_sm_count();
  return (int)(all < most ? all : most);
}
}  // namespace

// y [tokens, (n_q + 2 n_k) * hd] dense from x (rows of ldx elements).  hd a multiple of 8 up to 256; all pointers on 16-byte boundaries,
// ldx a multiple of 8; cosb / sinb [table_rows, hd / 2] fp32; pos [tokens] int32, or null: token t is at t % S.
TPLR_API int tplr_qk_norm_rope(const void* x, long long ldx, void* y, const void* wq, const void* wk, const float* cosb, const float* sinb,
                               const int* pos, long long tokens, int S, int table_rows, int n_q, int n_k, int hd, float eps,
                               unsigned int* status, void* stream) {
  TPLR_ENTER();
  if (tokens <= 0) return 0;
  QkNorm p = {};
  p.x = (const bf16*)x; p.ldx = ldx; p.y = (bf16*)y; p.wq = (const bf16*)wq; p.wk = (const bf16*)wk; p.cosb = cosb; p.sinb = sinb;
  p.pos = pos; p.tokens = tokens; p.S = S; p.table_rows = table_rows; p.n_q = n_q; p.n_k = n_k; p.hd = hd; p.eps = eps;
  p.inv_hd = 1.f / (float)hd; p.status = status;
  if (!fits(p)) return -301;
  p.chunks = chunks_of(n_q, n_k, hd, FWD_STEPS);
  auto kern = lanes_of(hd) == 8 ? qk_norm_fwd_kernel<8, FWD_STEPS> : lanes_of(hd) == 16 ? qk_norm_fwd_kernel<16, FWD_STEPS>
                                                                                        : qk_norm_fwd_kernel<32, FWD_STEPS>;
  const long long blocks = (tokens * p.chunks + WARPS - 1) / WARPS;
  if (blocks > 0x7fffffffLL) return -301;
  return (int)launch_pdl(kern, (unsigned)blocks, WARPS * 32, 0, (cudaStream_t)stream, p);
}

// Rows of 2 * hd fp32 sums that the backward pass leaves in its workspace.
TPLR_API int tplr_qk_norm_rope_parts(long long tokens, int n_q, int n_k, int hd) {
  if (tokens <= 0 || hd <= 0 || hd > 256) return 0;
  return bwd_blocks(tokens, n_q, n_k, hd);
}

// dx (dense) from dy (rows of lddy elements) and the forward's x; part: tplr_qk_norm_rope_parts rows of 2 * hd fp32, contents
// irrelevant.  Each weight's gradient is added onto add_* (fp32) where that is given, else stored to dw* (bf16) where that is.  add_q and
// add_k may be the same buffer, but not overlap in part.
TPLR_API int tplr_qk_norm_rope_bwd(const void* dy, long long lddy, const void* x, long long ldx, const void* wq, const void* wk,
                                   const float* cosb, const float* sinb, const int* pos, void* dx, float* part, void* dwq, void* dwk,
                                   float* add_q, float* add_k, long long tokens, int S, int table_rows, int n_q, int n_k, int hd, float eps,
                                   unsigned int* status, void* stream) {
  TPLR_ENTER();
  if (tokens <= 0) return 0;
  QkNorm p = {};
  p.x = (const bf16*)x; p.ldx = ldx; p.dy = (const bf16*)dy; p.lddy = lddy; p.y = (bf16*)dx; p.wq = (const bf16*)wq; p.wk = (const bf16*)wk;
  p.cosb = cosb; p.sinb = sinb; p.pos = pos; p.tokens = tokens; p.S = S; p.table_rows = table_rows; p.n_q = n_q; p.n_k = n_k; p.hd = hd;
  p.eps = eps; p.inv_hd = 1.f / (float)hd; p.part = part; p.status = status;
  if (!fits(p) || (add_q && add_k && add_q != add_k && add_q < add_k + hd && add_k < add_q + hd)) return -301;
  p.chunks = chunks_of(n_q, n_k, hd, BWD_STEPS);
  auto kern = lanes_of(hd) == 8 ? qk_norm_bwd_kernel<8, BWD_STEPS> : lanes_of(hd) == 16 ? qk_norm_bwd_kernel<16, BWD_STEPS>
                                                                                        : qk_norm_bwd_kernel<32, BWD_STEPS>;
  const int blocks = bwd_blocks(tokens, n_q, n_k, hd);
  if (const cudaError_t e = launch_pdl(kern, (unsigned)blocks, WARPS * 32, 0, (cudaStream_t)stream, p)) return (int)e;
  return (int)launch_pdl(qk_norm_dw_kernel, (unsigned)((2 * hd + 31) / 32), 1024, 0, (cudaStream_t)stream, part, blocks, hd, (bf16*)dwq,
                         (bf16*)dwk, add_q, add_k);
}
