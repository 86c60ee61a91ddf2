// Rows in 8 bits (sm_100a): what an 8-bit product takes as its operand and what a backward pass reads again.
//
// A group of a row (the whole row for products, 64 columns for saved activations) with the largest magnitude a is held as
//   q = rint(x * (127 / a)) in [-127, 127],   scale = a / 127,   value = q * scale
// with IEEE division, in fp32.  A group below 2^-100 (127 / a would overflow not far below) is zero with scale zero; a group with a
// member that is not finite has scale NaN and q zero, so that all that is made of it is NaN and nothing is hidden.  Magnitudes are
// compared by their bits, where NaN is above infinity and both above every number.
#include "quant.cuh"

namespace {
typedef __nv_bfloat16 bf16;
typedef long long ll;

// what is not finite converts to 0
__device__ __forceinline__ int code(float x, float inv) { return __float2int_rn(x * inv); }

// ------------------------------------------------------------------------------------------ rows -> 8 bits
enum Mode {
  ROWS = 0,          // a: bf16 rows of D, one scale a row
  GROUPS = 1,        // a: bf16 rows of D, a scale for every 64 columns
  NORM_ROWS = 2,     // h = a + b, rows h * rstd * w, one scale a row
  NORM_SAVED = 3,    // h = a + b, y = h * rstd * w in bf16, rows h * rstd with a scale for every 64 columns, rstd
  SWIGLU_ROWS = 4,   // a: bf16 [gate | up] rows of 2 D, rows silu(gate) * up, one scale a row
};
constexpr int GROUP = QUANT_GROUP;

struct RowsArgs {
  const bf16 *a, *b, *w;
  ll lda, ldb;
  bf16 *h, *y;
  int8_t* q;
  ll ldq;            // bytes; columns from D on are written as zeros
  float* scale;
  ll scale_row, scale_group;
  float* rstd;
  ll T;
  int D;
  float eps;
};

__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// One CTA a row, element by element: every width and alignment.  A row of up to 256 * EPT elements stays in registers, EPT a
// thread, 32 * EPT consecutive ones a warp, so that a group of 64 columns is two values of every lane; EPT 0: it is read again for each
// pass.  1111 x 1001, norm in 8 bits: 7.0 us read three times, 4.8 from registers.
template <int MODE, int EPT>
__global__ void __launch_bounds__(256) rows_q8_any_kernel(const RowsArgs p) {
  constexpr bool NORM = MODE == NORM_ROWS || MODE == NORM_SAVED, BY_GROUP = MODE == GROUPS || MODE == NORM_SAVED;
  constexpr int HELD = EPT ? EPT : 1;
  __shared__ float red[32];
  __shared__ uint32_t s_top[8];
  grid_wait();
  grid_release();
  const ll row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, D = p.D;
  const bf16 *a = p.a + row * p.lda, *b = p.b ? p.b + row * p.ldb : nullptr;
  int8_t* q = p.q + row * p.ldq;
  auto in = [&](int i) -> float {
    if (MODE == SWIGLU_ROWS) return silu_mul(__bfloat162float(a[i]), __bfloat162float(a[D + i]));
    if (!NORM || !b) return __bfloat162float(a[i]);
    return __bfloat162float(__float2bfloat16(__bfloat162float(a[i]) + __bfloat162float(b[i])));   // as the residual stream stores it
  };
  auto column = [&](int c) { return (warp * HELD + c) * 32 + lane; };
  float v[HELD];
  float r = 1.f;
  if (EPT) {
#pragma unroll
    for (int c = 0; c < HELD; ++c) v[c] = column(c) < D ? in(column(c)) : 0.f;
  }
  if (NORM) {
    float ss = 0.f;
    if (EPT) {
#pragma unroll
      for (int c = 0; c < HELD; ++c) {
        if (p.h && column(c) < D) p.h[row * D + column(c)] = __float2bfloat16(v[c]);
        ss = fmaf(v[c], v[c], ss);
      }
    } else {
      for (int i = threadIdx.x; i < D; i += 256) {
        const float x = in(i);
        if (p.h) p.h[row * D + i] = __float2bfloat16(x);
        ss = fmaf(x, x, ss);
      }
    }
    r = rsqrtf(block_sum(ss, red) / (float)D + p.eps);
    if (MODE == NORM_SAVED && threadIdx.x == 0) p.rstd[row] = r;
    if (EPT) {
#pragma unroll
      for (int c = 0; c < HELD; ++c) {
        v[c] *= r;
        if (MODE == NORM_ROWS && column(c) < D) v[c] *= __bfloat162float(p.w[column(c)]);
      }
    }
  }
  auto value = [&](int i) -> float {                                     // of a column that is not held
    const float x = NORM ? in(i) * r : in(i);
    return MODE == NORM_ROWS ? x * __bfloat162float(p.w[i]) : x;
  };
  if (BY_GROUP) {
    auto group = [&](int i0, float x0, float x1) {                       // columns i0 and i0 + 32 of a group
      const Codes k = codes_of(__reduce_max_sync(0xffffffffu, max(magnitude(x0), magnitude(x1))));
      const int i1 = i0 + 32;
      if (lane == 0 && i0 < D) p.scale[row * p.scale_row + (i0 >> 6) * p.scale_group] = k.scale;
      if (i0 < p.ldq) q[i0] = (int8_t)code(x0, k.inv);
      if (i1 < p.ldq) q[i1] = (int8_t)code(x1, k.inv);
      if (MODE == NORM_SAVED) {
        if (i0 < D) p.y[row * D + i0] = __float2bfloat16(x0 * __bfloat162float(p.w[i0]));
        if (i1 < D) p.y[row * D + i1] = __float2bfloat16(x1 * __bfloat162float(p.w[i1]));
      }
    };
    if (EPT) {
#pragma unroll
      for (int c = 0; c + 1 < HELD; c += 2) group(column(c), v[c], v[c + 1]);
    } else {
      for (int g = warp; g * GROUP < D; g += 8) {
        const int i0 = g * GROUP + lane;
        group(i0, i0 < D ? value(i0) : 0.f, i0 + 32 < D ? value(i0 + 32) : 0.f);
      }
    }
    return;
  }
  uint32_t top = 0;
  if (EPT) {
#pragma unroll
    for (int c = 0; c < HELD; ++c) top = max(top, magnitude(v[c]));
  } else {
    for (int i = threadIdx.x; i < D; i += 256) top = max(top, magnitude(value(i)));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  for (int k = 0; k < 8; ++k) top = max(top, s_top[k]);
  const Codes k = codes_of(top);
  if (threadIdx.x == 0) p.scale[row * p.scale_row] = k.scale;
  if (EPT) {
#pragma unroll
    for (int c = 0; c < HELD; ++c)
      if (column(c) < p.ldq) q[column(c)] = (int8_t)code(v[c], k.inv);   // zeros behind column D
  } else {
    for (int i = threadIdx.x; i < p.ldq; i += 256) q[i] = i < D ? (int8_t)code(value(i), k.inv) : 0;
  }
}

struct alignas(16) bf16x8 { __nv_bfloat162 v[4]; };
__device__ __forceinline__ void unpack8(const bf16x8& p, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = __bfloat1622float2(p.v[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
}
__device__ __forceinline__ bf16x8 pack8(const float* f) {
  bf16x8 p;
#pragma unroll
  for (int i = 0; i < 4; ++i) p.v[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return p;
}
__device__ __forceinline__ uint2 codes8(const float* x, float inv) { return make_uint2(codes4(x, inv), codes4(x + 4, inv)); }
__device__ __forceinline__ void values8(const uint2& q, float scale, float* f) {
  numbers4(q.x, f); numbers4(q.y, f + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] *= scale;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }

// The same from registers, for rows of whole 16-byte pieces: `tpr` threads (a power of two) share a row, VPL pieces each, so a row is
// read once and its two reductions (the squares, the largest magnitude) run on values that are already there.  Several rows a CTA
// share its barriers.  A thread asks for all its pieces before it waits for the first.
//
// RING: CTAs that stay, RING of them on an SM, and ask for the next row while they work on one, each thread's own pieces into its own
// shared memory, so that no barrier stands between a copy and its use and a CTA's loads, barriers and stores do not come in turn.  Without
// and with it: norm in 8 bits 4096 x 4096 26.4 and 21.6 us, 16384 x 2048 45.4 and 39.0 (6.0 TB/s, 92 % of what a plain copy of 2 GB moves), its training
// form 31.1 and 28.1, 56.2 and 50.6; codes by row 12.2 and 10.8, 21.8 and 19.3.  Three rows in flight, CTAs of 128 threads, two pieces a thread and
// neighbouring rows to a CTA were even or slower.  Not faster: a norm without a residual to add (17.7 and 18.7, 31.5 and 35.3) and the activation of
// [gate | up] rows (16384 x 1024 17.5 and 17.4, 4096 x 2048 10.9 and 12.2).
template <int MODE, int VPL, int BLOCK, int RING>
__global__ void __launch_bounds__(BLOCK, RING ? RING : 1024 / BLOCK) rows_q8_kernel(const RowsArgs p, const int tpr) {
  constexpr bool NORM = MODE == NORM_ROWS || MODE == NORM_SAVED, BY_GROUP = MODE == GROUPS || MODE == NORM_SAVED;
  constexpr int OPERANDS = NORM ? 2 : 1, PIECE = BLOCK * 16, STAGE = OPERANDS * VPL * PIECE;
  extern __shared__ __align__(16) uint8_t ring[];                                   // [this row, the next][operand][piece][thread]
  __shared__ float s_sum[RING ? 2 : 1][32];                              // by row in turn: the next row's are written while this one's are read
  __shared__ uint32_t s_top[RING ? 2 : 1][32];
  grid_wait();
  grid_release();
  const int t = threadIdx.x & (tpr - 1), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.D, nv = D / 8, warps = tpr >> 5;
  const int row_warp = threadIdx.x / tpr * warps;                        // first warp of this thread's row
  const bool two = MODE == SWIGLU_ROWS || (NORM && p.b);
  const ll rows = blockDim.x / tpr, step = (ll)gridDim.x * rows;
  uint8_t* mine = ring + threadIdx.x * 16;
  auto ask = [&](ll row, int stage) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(mine) + stage * STAGE;
    if (row < p.T) {
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (t + tpr * j < nv) {
          copy16(to + j * PIECE, p.a + row * p.lda + (t + tpr * j) * 8);
          if (OPERANDS == 2) copy16(to + (VPL + j) * PIECE, p.b + row * p.ldb + (t + tpr * j) * 8);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  bf16x8 wp[VPL];
  if (RING) {
    if (NORM) {
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (t + tpr * j < nv) wp[j] = reinterpret_cast<const bf16x8*>(p.w)[t + tpr * j];
    }
    ask((ll)blockIdx.x * rows + threadIdx.x / tpr, 0);
  }
  int stage = 0;
  for (ll first = (ll)blockIdx.x * rows; first < p.T; first += step, stage ^= 1) {   // once without a ring
    const ll row = first + threadIdx.x / tpr;
    const bool live = row < p.T;
    if (RING) {
      ask(row + step, stage ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    }
    const int at = RING ? stage : 0;
    float v[VPL][8];
    {
      bf16x8 ra[VPL], rb[VPL];
      if (RING) {
        const bf16x8* from = reinterpret_cast<const bf16x8*>(mine + stage * STAGE);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (live && t + tpr * j < nv) {
            ra[j] = from[j * BLOCK];
            if (OPERANDS == 2) rb[j] = from[(VPL + j) * BLOCK];
          }
      } else {
        const bf16x8* a = reinterpret_cast<const bf16x8*>(p.a + (live ? row : 0) * p.lda);
        const bf16x8* b = MODE == SWIGLU_ROWS ? a + nv : p.b ? reinterpret_cast<const bf16x8*>(p.b + (live ? row : 0) * p.ldb) : nullptr;
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (live && t + tpr * j < nv) {
            ra[j] = a[t + tpr * j];
            if (two) rb[j] = b[t + tpr * j];
          }
      }
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int i = t + tpr * j;
        if (!live || i >= nv) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = 0.f;
          continue;
        }
        if (NORM && two) {                                               // the norm sees the sum as the residual stream stores it
#pragma unroll
          for (int e = 0; e < 4; ++e) ra[j].v[e] = __hadd2(ra[j].v[e], rb[j].v[e]);
          reinterpret_cast<bf16x8*>(p.h + row * D)[i] = ra[j];
        }
        unpack8(ra[j], v[j]);
        if (MODE == SWIGLU_ROWS) {
          float o[8];
          unpack8(rb[j], o);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = silu_mul(v[j][e], o[e]);
        }
      }
    }
    if (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < VPL; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(v[j][e], v[j][e], ss);
      if (MODE == NORM_SAVED && !RING) {                                 // all asked for here: no load passes the stores below
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (t + tpr * j < nv) wp[j] = reinterpret_cast<const bf16x8*>(p.w)[t + tpr * j];
      }
      ss = warp_sum(ss);
      if (warps > 1) {
        if (lane == 0) s_sum[at][warp] = ss;
        __syncthreads();
        ss = 0.f;
        for (int k = 0; k < warps; ++k) ss += s_sum[at][row_warp + k];
      }
      const float r = rsqrtf(ss / (float)D + p.eps);
      if (MODE == NORM_SAVED && live && t == 0) p.rstd[row] = r;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int i = t + tpr * j;
        if (!live || i >= nv) continue;
        float w[8];
        unpack8(RING || MODE == NORM_SAVED ? wp[j] : reinterpret_cast<const bf16x8*>(p.w)[i], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[j][e] *= r;
          w[e] *= v[j][e];
        }
        if (MODE == NORM_ROWS) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] = w[e];
        } else {
          reinterpret_cast<bf16x8*>(p.y + row * D)[i] = pack8(w);
        }
      }
    }
    uint32_t tops[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e += 2) top = top3(top, v[j][e], v[j][e + 1]);
      tops[j] = magnitude(top);
    }
    Codes all = {};
    if (!BY_GROUP) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < VPL; ++j) top = max(top, tops[j]);
      top = __reduce_max_sync(0xffffffffu, top);
      if (warps > 1) {
        if (lane == 0) s_top[at][warp] = top;
        __syncthreads();
        for (int k = 0; k < warps; ++k) top = max(top, s_top[at][row_warp + k]);
      }
      all = codes_of(top);
      if (live && t == 0) p.scale[row * p.scale_row] = all.scale;
    }
    if (BY_GROUP) {                                                      // eight lanes hold a group's 64 columns
#pragma unroll
      for (int j = 0; j < VPL; ++j)
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) tops[j] = max(tops[j], __shfl_xor_sync(0xffffffffu, tops[j], o));
      // lane j of the eight divides for their j-th group
      const int k = lane & 7;
      uint32_t top = tops[0];
#pragma unroll
      for (int j = 1; j < VPL; ++j) top = k == j ? tops[j] : top;
      all = codes_of(top);
      const int i = t - k + tpr * k;
      if (live && k < VPL && i < nv) p.scale[row * p.scale_row + (i >> 3) * p.scale_group] = all.scale;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int i = t + tpr * j;
      const float inv = BY_GROUP ? __shfl_sync(0xffffffffu, all.inv, (lane & ~7) + j) : all.inv;
      if (live && (ll)i * 8 < p.ldq)                                     // zeros behind the row: v is 0 there
        reinterpret_cast<uint2*>(p.q + row * p.ldq)[i] = codes8(v[j], i < nv ? inv : 0.f);
    }
    if (!RING) break;
  }
}

// ------------------------------------------------------------------------------------------ 8 bits -> rows
// y = q * scale (* w of the column), rows of D; a scale for the row or for every 64 columns.
__global__ void __launch_bounds__(256) dequantize_any_kernel(const int8_t* q, ll ldq, const float* scale, ll scale_row, ll scale_group,
                                                             bool by_group, const bf16* w, bf16* y, ll T, int D) {
  grid_wait();
  grid_release();
  for (ll row = blockIdx.x; row < T; row += gridDim.x) {
    const float* s = scale + row * scale_row;
    for (int c0 = threadIdx.x; c0 < D; c0 += 4 * 256) {
      float v[4], m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + 256 * j;
        v[j] = c < D ? (float)q[row * ldq + c] * s[by_group ? c / GROUP * scale_group : 0] : 0.f;
        m[j] = w && c < D ? __bfloat162float(w[c]) : 1.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + 256 * j < D) y[row * D + c0 + 256 * j] = __float2bfloat16(w ? v[j] * m[j] : v[j]);
    }
  }
}

// The same for whole 16-byte pieces of y, a scale for a row or for 64 columns: `tpr` threads (a power of two) on a row, four pieces each,
// all asked for before the first is written.  16384 x 2048 by 64 columns: 21 us (4.7 TB/s), 32 in a loop whose loads stood behind its stores.
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* q, ll ldq, const float* scale, ll scale_row, ll scale_group,
                                                         const bf16* w, bf16* y, ll T, int D, int tpr) {
  grid_wait();
  grid_release();
  const int nv = D / 8, t = threadIdx.x & (tpr - 1);
  const ll row = (ll)blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
  if (row >= T) return;
  const uint2* src = reinterpret_cast<const uint2*>(q + row * ldq);
  bf16x8* dst = reinterpret_cast<bf16x8*>(y + row * D);
  for (int i0 = t; i0 < nv; i0 += 4 * tpr) {
    uint2 c[4];
    float s[4];
    bf16x8 m[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + tpr * j;
      if (i < nv) {
        c[j] = src[i];
        s[j] = scale[row * scale_row + (i >> 3) * scale_group];
        if (w) m[j] = reinterpret_cast<const bf16x8*>(w)[i];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + tpr * j;
      if (i >= nv) continue;
      float f[8];
      values8(c[j], s[j], f);
      if (w) {
        float g[8];
        unpack8(m[j], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= g[e];
      }
      dst[i] = pack8(f);
    }
  }
}

// ------------------------------------------------------------------------------------------ norm, backward from 8 bits
// xn = q * scale; g = dy * w; dx = dres + rstd * (g - xn * mean(g * xn)); the CTA's sum of dy * xn goes to part[blockIdx.x].  Every width and
// alignment; a row of up to BLOCK * EPT elements stays in registers, and so do the sums (EPT 0: read again, sums in memory).
template <int EPT, int BLOCK>
__global__ void __launch_bounds__(BLOCK) rmsnorm_saved8_bwd_any_kernel(const bf16* dy, const int8_t* q, ll ldq, const float* scale, ll scale_row,
                                                                       ll scale_group, const float* rstd, const bf16* w, const bf16* dres,
                                                                       bf16* dx, float* part, ll T, int D) {
  constexpr int HELD = EPT ? EPT : 1;
  __shared__ float red[32];
  grid_wait();
  grid_release();
  float* mine = part + (ll)blockIdx.x * D;
  auto xn = [&](ll row, int i) { return (float)q[row * ldq + i] * scale[row * scale_row + i / GROUP * scale_group]; };
  if (EPT) {
    float dw[HELD] = {}, m[HELD];
#pragma unroll
    for (int c = 0; c < HELD; ++c) m[c] = threadIdx.x + BLOCK * c < D ? __bfloat162float(w[threadIdx.x + BLOCK * c]) : 0.f;
    for (ll row = blockIdx.x; row < T; row += gridDim.x) {
      float dot = 0.f, x[HELD], g[HELD], a[HELD];
      const float r = rstd[row];
#pragma unroll
      for (int c = 0; c < HELD; ++c) {
        const int i = threadIdx.x + BLOCK * c;
        g[c] = i < D ? __bfloat162float(dy[row * D + i]) : 0.f;
        x[c] = i < D ? xn(row, i) : 0.f;
        a[c] = dres && i < D ? __bfloat162float(dres[row * D + i]) : 0.f;
      }
#pragma unroll
      for (int c = 0; c < HELD; ++c) {
        dw[c] = fmaf(g[c], x[c], dw[c]);
        g[c] *= m[c];
        dot = fmaf(g[c], x[c], dot);
      }
      dot = block_sum(dot, red) / (float)D;
#pragma unroll
      for (int c = 0; c < HELD; ++c)
        if (threadIdx.x + BLOCK * c < D) dx[row * D + threadIdx.x + BLOCK * c] = __float2bfloat16(fmaf(r, g[c] - x[c] * dot, a[c]));
      __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < HELD; ++c)
      if (threadIdx.x + BLOCK * c < D) mine[threadIdx.x + BLOCK * c] = dw[c];
    return;
  }
  for (int i = threadIdx.x; i < D; i += BLOCK) mine[i] = 0.f;            // this thread's own columns
  for (ll row = blockIdx.x; row < T; row += gridDim.x) {
    float dot = 0.f;
    for (int i = threadIdx.x; i < D; i += BLOCK) {
      const float d = __bfloat162float(dy[row * D + i]), xi = xn(row, i);
      mine[i] += d * xi;
      dot = fmaf(d * __bfloat162float(w[i]), xi, dot);
    }
    dot = block_sum(dot, red) / (float)D;
    const float r = rstd[row];
    for (int i = threadIdx.x; i < D; i += BLOCK) {
      const float o = r * (__bfloat162float(dy[row * D + i]) * __bfloat162float(w[i]) - xn(row, i) * dot);
      dx[row * D + i] = __float2bfloat16(dres ? o + __bfloat162float(dres[row * D + i]) : o);
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void copy8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }

// The same for whole 16-byte pieces: `tpr` threads on a row, VPL pieces each, the weight gradient's sums of a thread's columns in registers
// over all rows of the CTA.  What keeps the memory busy are the copies of the two rows after the present one, each thread's own
// pieces into its own shared memory, so that no barrier stands between them and their use.
// Counters of a first form (16384 x 2048): the memory 45 % busy, an instruction issued in 72 % of the cycles; so the weight stays unpacked, the
// products and the codes' numbers of a piece stay for its output, and a scale multiplies once a piece where it can, and the next row's scales are asked for
// a row ahead: 57 -> 47 us, 5.0 TB/s.
// Two pieces a thread, or three where two leave more threads idle (widths of three times a power of two): 16384 x 768 21.5 us against
// 24.5, x 1536 38.2 against 45.9; at 2048 two take 48.8, three 53.3, one (24 warps an SM) 54.1, four 52.9.
constexpr int BWD_STAGES = 3;
constexpr int bwd_ctas(int vpl, int block) { return vpl == 3 ? 3 : 512 / block; }                      // resident on an SM
template <int VPL, int BLOCK>
__global__ void __launch_bounds__(BLOCK, bwd_ctas(VPL, BLOCK))
rmsnorm_saved8_bwd_kernel(const bf16* dy, const int8_t* q, ll ldq, const float* scale, ll scale_row, ll scale_group, const float* rstd, const bf16* w,
                          const bf16* dres, bf16* dx, float* part, ll T, int D, int tpr) {
  constexpr int PIECE = 40 * BLOCK, STAGE = VPL * PIECE;
  extern __shared__ __align__(16) uint8_t pieces[];        // [stage][piece][dy 16 | dres 16 | codes 8][thread]
  __shared__ float s_dot[2][BLOCK / 32];
  __shared__ float s_dw[BLOCK * 8];
  grid_wait();
  grid_release();
  const int t = threadIdx.x & (tpr - 1), slot = threadIdx.x / tpr, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nv = D / 8;
  const int warps = tpr >> 5, rows = BLOCK / tpr;
  const uint32_t mine16 = (uint32_t)__cvta_generic_to_shared(pieces) + threadIdx.x * 16u;
  const uint32_t mine8 = (uint32_t)__cvta_generic_to_shared(pieces) + 32u * BLOCK + threadIdx.x * 8u;
  float m[VPL][8], dw[VPL][8];
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    if (t + tpr * j < nv) unpack8(reinterpret_cast<const bf16x8*>(w)[t + tpr * j], m[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = 0.f;
  }
  auto ask = [&](ll row, int stage) {
    if (row < T) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const int i = t + tpr * j;
        if (i < nv) {
          const uint32_t at = stage * STAGE + j * PIECE;
          copy16(mine16 + at, dy + row * D + i * 8);
          if (dres) copy16(mine16 + at + 16 * BLOCK, dres + row * D + i * 8);
          copy8(mine8 + at, q + row * ldq + i * 8);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float sc2[VPL] = {}, r2 = 0.f;                                           // the next row's scales: their latency would be in every turn
  auto ask_scales = [&](ll row) {
    if (row >= T) return;
    r2 = rstd[row];
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (t + tpr * j < nv) sc2[j] = scale[row * scale_row + ((t + tpr * j) >> 3) * scale_group];
  };
  const ll step = (ll)gridDim.x * rows;
  ask((ll)blockIdx.x * rows + slot, 0);
  ask((ll)blockIdx.x * rows + slot + step, 1);
  ask_scales((ll)blockIdx.x * rows + slot);
  int turn = 0, stage = 0;
  for (ll first = (ll)blockIdx.x * rows; first < T; first += step, turn ^= 1, stage = stage == BWD_STAGES - 1 ? 0 : stage + 1) {
    const ll row = first + slot;
    const bool live = row < T;
    float sc[VPL];
    const float r = r2;
#pragma unroll
    for (int j = 0; j < VPL; ++j) sc[j] = sc2[j];
    ask_scales(row + step);
    ask(row + 2 * step, stage == 0 ? 2 : stage - 1);
    asm volatile("cp.async.wait_group 2;" ::: "memory");
    float gm[VPL][8], x[VPL][8], dot = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (live && t + tpr * j < nv) {
        const uint8_t* at = pieces + stage * STAGE + j * PIECE;
        const uint2 c = reinterpret_cast<const uint2*>(at + 32 * BLOCK)[threadIdx.x];
        float d[8], sum = 0.f;
        unpack8(reinterpret_cast<const bf16x8*>(at)[threadIdx.x], d);
        numbers4(c.x, x[j]); numbers4(c.y, x[j] + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gm[j][e] = d[e] * m[j][e];
          dw[j][e] = fmaf(d[e] * sc[j], x[j][e], dw[j][e]);
          sum = fmaf(gm[j][e], x[j][e], sum);
        }
        dot = fmaf(sum, sc[j], dot);
      }
    dot = warp_sum(dot);
    if (warps > 1) {                                                     // two buffers: one barrier a row
      if (lane == 0) s_dot[turn][warp] = dot;
      __syncthreads();
      dot = 0.f;
      for (int k = 0; k < warps; ++k) dot += s_dot[turn][slot * warps + k];
    }
    dot *= r / (float)D;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      const int i = t + tpr * j;
      if (live && i < nv) {
        const float k = dot * sc[j];
        float o[8];
        if (dres) {
          unpack8(reinterpret_cast<const bf16x8*>(pieces + stage * STAGE + j * PIECE + 16 * BLOCK)[threadIdx.x], o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = fmaf(r, gm[j][e], o[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = r * gm[j][e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(-k, x[j][e], o[e]);
        reinterpret_cast<bf16x8*>(dx + row * D)[i] = pack8(o);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  float* mine = part + (ll)blockIdx.x * D;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int i = t + tpr * j;
    if (rows > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) s_dw[e * BLOCK + threadIdx.x] = dw[j][e];
      __syncthreads();
      if (slot == 0)
        for (int k = 1; k < rows; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) dw[j][e] += s_dw[e * BLOCK + k * tpr + t];
    }
    if (slot == 0 && i < nv) {
      reinterpret_cast<float4*>(mine + i * 8)[0] = make_float4(dw[j][0], dw[j][1], dw[j][2], dw[j][3]);
      reinterpret_cast<float4*>(mine + i * 8)[1] = make_float4(dw[j][4], dw[j][5], dw[j][6], dw[j][7]);
    }
  }
}

// Sum of the CTAs' parts in their order, the same on every run: added into an fp32 buffer or stored in bf16.
__global__ void __launch_bounds__(1024) sum_parts_kernel(const float* part, int n, int D, float* add, bf16* out) {
  __shared__ float s[32][33];
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int k = slice; k < n; k += 32) v += part[(ll)k * D + c];
  }
  s[slice][lane] = v;
  __syncthreads();
  if (slice == 0 && c < D) {
#pragma unroll
    for (int k = 1; k < 32; ++k) v += s[k][lane];
    if (add) add[c] += v;
    else out[c] = __float2bfloat16(v);
  }
}

// ------------------------------------------------------------------------------------------ SwiGLU around a saved projection
// gu: fp32 [gate | up] rows of 2 F; act = silu(gate) * up in bf16; gate and up in 8 bits, a scale for every 64 columns of each
// half.  One warp a group of both halves.
__global__ void __launch_bounds__(256) swiglu_saved8_kernel(const float* gu, bf16* act, int8_t* q, ll ldq, float* scale, ll scale_row,
                                                            ll scale_group, ll T, int F) {
  grid_wait();
  grid_release();
  const int lane = threadIdx.x & 31, groups = (F + GROUP - 1) / GROUP;
  for (ll at = blockIdx.x * 8LL + (threadIdx.x >> 5); at < T * groups; at += gridDim.x * 8LL) {
    const ll row = at / groups;
    const int g = (int)(at - row * groups);
    float v[2][2];
    for (int h = 0; h < 2; ++h) {
      const int i0 = g * GROUP + lane, i1 = i0 + 32;
      const float* src = gu + row * 2 * F + (ll)h * F;
      v[h][0] = i0 < F ? src[i0] : 0.f;
      v[h][1] = i1 < F ? src[i1] : 0.f;
      const Codes c = codes_of(__reduce_max_sync(0xffffffffu, max(magnitude(v[h][0]), magnitude(v[h][1]))));
      if (lane == 0) scale[row * scale_row + (h * groups + g) * scale_group] = c.scale;
      if (i0 < F) q[row * ldq + (ll)h * F + i0] = (int8_t)code(v[h][0], c.inv);
      if (i1 < F) q[row * ldq + (ll)h * F + i1] = (int8_t)code(v[h][1], c.inv);
    }
    for (int k = 0; k < 2; ++k) {
      const int i = g * GROUP + lane + 32 * k;
      if (i < F) act[row * F + i] = __float2bfloat16(silu_mul(v[0][k], v[1][k]));
    }
  }
}

// dact: fp32 [T, F]; the kept gate and up -> dgu = [dgate | dup] and the activation again, bf16.
__global__ void __launch_bounds__(256) swiglu_saved8_bwd_kernel(const float* dact, const int8_t* q, ll ldq, const float* scale, ll scale_row,
                                                                ll scale_group, bf16* dgu, bf16* act, ll T, int F) {
  grid_wait();
  grid_release();
  const int groups = (F + GROUP - 1) / GROUP;
  const ll total = T * F;
  for (ll i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const ll row = i / F;
    const int c = (int)(i - row * F);
    const float* s = scale + row * scale_row;
    const float g = (float)q[row * ldq + c] * s[c / GROUP * scale_group];
    const float u = (float)q[row * ldq + F + c] * s[(groups + c / GROUP) * scale_group];
    const float sg = 1.f / (1.f + __expf(-g)), sl = g * sg, d = dact[i];
    dgu[row * 2 * F + c] = __float2bfloat16(d * u * (sg + sl * (1.f - sg)));
    dgu[row * 2 * F + F + c] = __float2bfloat16(d * sl);
    act[i] = __float2bfloat16(sl * u);
  }
}

// ------------------------------------------------------------------------------------------ product, few tokens
// y[t, n] = sx[t] * sw[n] * sum_k x[t, k] w[n, k] where the weight's bytes are all that counts: they are read once, 16 bytes a lane,
// straight into the operands of mma.m16n8k32: nothing is set up before the first load, which for 2048 x 2048 is a third of
// the time.  The sum over k may be taken in any order, so a lane's 16 bytes of a row are its words of two instructions as they lie:
// word j of a weight row and word j of a token are multiplied wherever the instruction thinks they are.  A CTA's eight warps take
// 64-byte pieces of 16 rows in turn, 512 bytes of a row together, and add their sums in shared memory, while the next rows' are on
// their way.
__device__ __forceinline__ uint4 ld_once(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t first_bytes(int n) { return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }
//
// HELD: x is bf16 and its rows are put in 8 bits here, by every CTA for itself, while its first pieces of the weight are on their way: as
// many values as the threads hold, HELD_MOST; one launch instead of two.  One token, one launch and two: 2048 x 2048 3.1 and 4.1 us, 4096 x 6144
// 6.9 and 8.5, 2048 x 16384 8.5 and 9.8; with 16384 values held a call of the last took 13.7, two CTAs an SM.  Those are times of one weight,
// which stays in L2; with weights in turn one launch takes 3.2, 6.9 and 8.6 us (1.3, 3.6 and 3.9 TB/s).
// TAIL: K is not whole 16-byte pieces, and codes behind it, which are the caller's, are masked; in one form for both 1 x 4096 x 6144 took 4.8 us, not 4.4.
constexpr int FEW = 8, FEW_UNROLL = 4, HELD_MOST = 4096, HELD_PIECES = HELD_MOST / 2048;
__host__ __device__ constexpr int held_stride(int kp) { return (kp + 511) / 512 * 512 + 64; }          // rows 64 bytes apart in the banks
template <class Out, bool HELD, bool TAIL>
__global__ void __launch_bounds__(256, 3) gemm_q8_few_kernel(const void* x, const int8_t* w, const float* sx, const float* sw, Out* y, int T, int N,
                                                          int K, ll ldx, ll ldw, ll ldy) {
  __shared__ int s_sum[2][8][8][17];
  __shared__ __align__(16) int8_t s_x[HELD ? HELD_MOST + FEW * (512 + 64) : 16];
  __shared__ float s_sx[FEW];
  __shared__ uint32_t s_top[8];
  grid_wait();
  grid_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kp = (K + 15) / 16 * 16, tok = lane >> 2;
  const int stride = held_stride(kp), blocks = (N + 15) / 16;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 a[FEW_UNROLL][2];
  auto ask = [&](int block, int k0) {
    const int n = block * 16 + (lane >> 2);
    const int8_t *r0 = w + (ll)min(n, N - 1) * ldw, *r1 = w + (ll)min(n + 8, N - 1) * ldw;
#pragma unroll
    for (int u = 0; u < FEW_UNROLL; ++u) {
      const int k = k0 + u * 512 + (lane & 3) * 16;
      a[u][0] = k < kp && n < N ? ld_once(r0 + k) : zero;
      a[u][1] = k < kp && n + 8 < N ? ld_once(r1 + k) : zero;
    }
  };
  ask(blockIdx.x, warp * 64);
  if (HELD) {
    int share = 256;                                                     // threads of a token
    while (share * T > 256) share /= 2;
    const int t = threadIdx.x / share, i0 = threadIdx.x & (share - 1), nv = K / 8;
    const bf16x8* row = reinterpret_cast<const bf16x8*>(static_cast<const bf16*>(x) + (t < T ? t : 0) * ldx);
    bf16x8 p[HELD_PIECES];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < HELD_PIECES; ++j)
      if (t < T && i0 + share * j < nv) p[j] = row[i0 + share * j];
#pragma unroll
    for (int j = 0; j < HELD_PIECES; ++j)
      if (t < T && i0 + share * j < nv) {
        float f[8];
        unpack8(p[j], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(f[e]));
      }
    top = __reduce_max_sync(0xffffffffu, top);
    if (share > 32) {
      if (lane == 0) s_top[warp] = top;
      __syncthreads();
      const int first = t * (share >> 5);
      for (int k = 0; k < (share >> 5); ++k) top = max(top, s_top[first + k]);
    }
    const Codes c = codes_of(top);
    if (t < T) {
      if (i0 == 0) s_sx[t] = c.scale;
#pragma unroll
      for (int j = 0; j < HELD_PIECES; ++j) {
        const int i = i0 + share * j;
        if (i * 8 >= kp) continue;
        float f[8] = {};
        if (i < nv) unpack8(p[j], f);
        *reinterpret_cast<uint2*>(s_x + t * stride + i * 8) = codes8(f, i < nv ? c.inv : 0.f);
      }
    }
    __syncthreads();
  }
  int turn = 0;
  for (int block = blockIdx.x; block < blocks; block += gridDim.x, turn ^= 1) {
    int acc[4] = {};
    for (int k0 = warp * 64; k0 < kp; k0 += 512 * FEW_UNROLL) {
      if (k0 != warp * 64) ask(block, k0);
      uint4 b[FEW_UNROLL];
#pragma unroll
      for (int u = 0; u < FEW_UNROLL; ++u) {
        const int k = k0 + u * 512 + (lane & 3) * 16;
        b[u] = zero;
        if (k < kp && tok < T)
          b[u] = HELD ? *reinterpret_cast<const uint4*>(s_x + tok * stride + k) : *reinterpret_cast<const uint4*>(static_cast<const int8_t*>(x) + tok * ldx + k);
        if (TAIL && k < K && k + 16 > K) {                              // what lies behind a row's last column counts for nothing
          b[u].x &= first_bytes(K - k); b[u].y &= first_bytes(K - k - 4);
          b[u].z &= first_bytes(K - k - 8); b[u].w &= first_bytes(K - k - 12);
        }
      }
#pragma unroll
      for (int u = 0; u < FEW_UNROLL; ++u) {
        mma_s8(acc, a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u].x, b[u].y);
        mma_s8(acc, a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u].z, b[u].w);
      }
    }
    if (block + (int)gridDim.x < blocks) ask(block + gridDim.x, warp * 64);          // on their way while the sums meet
#pragma unroll
    for (int e = 0; e < 4; ++e) s_sum[turn][warp][(lane & 3) * 2 + (e & 1)][(lane >> 2) + (e >> 1) * 8] = acc[e];
    __syncthreads();                                                     // two buffers: one barrier a block
    const int t = threadIdx.x >> 4, c = threadIdx.x & 15, n = block * 16 + c;
    if (t < T && n < N) {                                                // 16 threads a token: those from 8 on have none
      int sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += s_sum[turn][k][t][c];
      y[t * ldy + n] = (Out)scaled(sum, HELD ? s_sx[t] : sx[t], sw[n]);
    }
  }
}

template <class Out, bool HELD, bool TAIL>
int gemm_q8_few(const void* x, const void* w, const float* sx, const float* sw, void* y, int T, int N, int K, ll ldx, ll ldw, ll ldy, void* st) {
  const int blocks = (N + 15) / 16, resident = 3 * tplr_sm_count(), turns = (blocks + resident - 1) / resident;
  return (int)launch_pdl(gemm_q8_few_kernel<Out, HELD, TAIL>, (blocks + turns - 1) / turns, 256, 0, (cudaStream_t)st, x, (const int8_t*)w, sx, sw, (Out*)y, T, N, K, ldx,
                         ldw, ldy);
}

template <class... P>
bool whole_pieces(P... ptrs) { return ((reinterpret_cast<uintptr_t>(ptrs) | ...) & 15) == 0; }
// Threads of a row of `pieces` 16-byte pieces at `vpl` each.
int row_threads(int pieces, int vpl) {
  int n = 32;
  while (n * vpl < pieces) n *= 2;
  return n;
}

unsigned waves(ll ctas, int resident) {
  const ll most = (ll)tplr_sm_count() * resident;
  return (unsigned)(ctas < most ? ctas : most);
}

template <int MODE, int BLOCK, int RING>
int rows_q8_ring(const RowsArgs& p, int tpr, cudaStream_t st) {
  constexpr int OPERANDS = MODE == NORM_ROWS || MODE == NORM_SAVED ? 2 : 1, SMEM = 2 * OPERANDS * 4 * BLOCK * 16;
  auto kern = rows_q8_kernel<MODE, 4, BLOCK, RING>;
  if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)) return (int)e;
  const ll groups = (p.T + BLOCK / tpr - 1) / (BLOCK / tpr);
  return (int)launch_pdl(kern, waves(groups, RING), BLOCK, SMEM, st, p, tpr);
}

template <int MODE>
int rows_q8(const RowsArgs& p, void* stream) {
  if (p.T <= 0) return 0;
  if (p.T > 0x7fffffffLL || p.D <= 0 || p.ldq < p.D) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  const int pieces = (int)((p.ldq + 7) / 8);
  if (p.D % 8 || p.ldq % 8 || p.lda % 8 || (p.b && p.ldb % 8) || p.D > 32760 || !whole_pieces(p.a, p.b, p.w, p.h, p.y, p.q))
    return (int)launch_pdl(p.D <= 1024 ? rows_q8_any_kernel<MODE, 4> : p.D <= 2048 ? rows_q8_any_kernel<MODE, 8> : p.D <= 4096 ? rows_q8_any_kernel<MODE, 16>
                           : p.D <= 8192 ? rows_q8_any_kernel<MODE, 32> : rows_q8_any_kernel<MODE, 0>, (unsigned)p.T, 256, 0, st, p);
  // One piece a thread while rows are few, four where they are many.  Microseconds with one and with four: norm in 8 bits 1 x 2048 2.3 and 3.3,
  // 128 x 2048 2.4 and 4.0, 512 x 2048 3.6 and 4.1, 1024 x 2048 6.1 and 5.9, 4096 x 768 8.2 and 7.3; codes alone 64 x 768 1.6 and 2.0, 128 x 2048
  // 1.8 and 2.1, 512 x 2048 2.7 and 2.2.
  const bool codes_alone = MODE == ROWS || MODE == GROUPS;
  const int vpl = p.T * pieces <= (codes_alone ? 512LL : 1024LL) * tplr_sm_count() && pieces <= 1024 ? 1 : 4;
  const int tpr = row_threads(pieces, vpl), block = tpr > 256 ? tpr : 256;
  const unsigned grid = (unsigned)((p.T + block / tpr - 1) / (block / tpr));
  if constexpr (MODE == NORM_SAVED)
    // Four arrays are written: beyond twice the L2, fewer CTAs keep longer runs of each together.  Microseconds with two of 256 threads an SM and with
    // one of 512: 12000 x 2048 38.2 and 39.9, 16384 x 1536 39.9 and 41.1, 16000 x 2048 53.5 and 50.4, 32768 x 2048 106.6 and 95.8.
    if (vpl == 4 && block == 256 && p.b && p.T * p.D > 28LL << 20) return rows_q8_ring<MODE, 512, 1>(p, tpr, st);
  if constexpr (MODE != SWIGLU_ROWS)
    if (vpl == 4 && block == 256 && (codes_alone || p.b)) return rows_q8_ring<MODE, 256, 2>(p, tpr, st);
  if (block > 256) return (int)(vpl == 1 ? launch_pdl(rows_q8_kernel<MODE, 1, 1024, 0>, grid, block, 0, st, p, tpr)
                                         : launch_pdl(rows_q8_kernel<MODE, 4, 1024, 0>, grid, block, 0, st, p, tpr));
  if constexpr (MODE != ROWS && MODE != GROUPS)
    if (vpl == 4) return (int)launch_pdl(rows_q8_kernel<MODE, 4, 256, 0>, grid, block, 0, st, p, tpr);
  return (int)launch_pdl(rows_q8_kernel<MODE, 1, 256, 0>, grid, block, 0, st, p, tpr);
}
}  // namespace

// bf16 rows (T of D, row stride ldx) in 8 bits: one scale a row (group 0) or for every 64 columns (group 64).  q: rows of ldq >= D bytes,
// zeros behind column D; scale[row * scale_row + group * scale_group].
TPLR_API int tplr_quantize_rows(const void* x, ll ldx, void* q, ll ldq, float* scale, ll scale_row, ll scale_group, ll T, int D, int group,
                                void* stream) {
  TPLR_ENTER();
  RowsArgs p = {};
  p.a = (const bf16*)x; p.lda = ldx; p.q = (int8_t*)q; p.ldq = ldq; p.scale = scale; p.scale_row = scale_row; p.scale_group = scale_group;
  p.T = T; p.D = D;
  if (group != 0 && group != GROUP) return (int)cudaErrorInvalidValue;
  return group ? rows_q8<GROUPS>(p, stream) : rows_q8<ROWS>(p, stream);
}

// h = res + delta (delta null: h = res, h_out unused) and the rows h * rstd * w in 8 bits, one scale a row.  Dense rows of D.
TPLR_API int tplr_add_rmsnorm_q8(const void* res, const void* delta, const void* w, void* h_out, void* q, ll ldq, float* scale, ll T, int D,
                                 float eps, void* stream) {
  TPLR_ENTER();
  RowsArgs p = {};
  p.a = (const bf16*)res; p.b = (const bf16*)delta; p.w = (const bf16*)w; p.lda = p.ldb = D; p.h = delta ? (bf16*)h_out : nullptr;
  p.q = (int8_t*)q; p.ldq = ldq; p.scale = scale; p.scale_row = 1; p.T = T; p.D = D; p.eps = eps;
  return rows_q8<NORM_ROWS>(p, stream);
}

// The training step's form: y = h * rstd * w in bf16, and for the backward pass rstd [T] and the rows h * rstd in 8 bits by 64 columns.
TPLR_API int tplr_add_rmsnorm_saved8(const void* res, const void* delta, const void* w, void* h_out, void* y, void* q, ll ldq, float* scale,
                                     ll scale_row, ll scale_group, float* rstd, ll T, int D, float eps, void* stream) {
  TPLR_ENTER();
  RowsArgs p = {};
  p.a = (const bf16*)res; p.b = (const bf16*)delta; p.w = (const bf16*)w; p.lda = p.ldb = D; p.h = delta ? (bf16*)h_out : nullptr;
  p.y = (bf16*)y; p.q = (int8_t*)q; p.ldq = ldq; p.scale = scale; p.scale_row = scale_row; p.scale_group = scale_group; p.rstd = rstd;
  p.T = T; p.D = D; p.eps = eps;
  return rows_q8<NORM_SAVED>(p, stream);
}

// silu(gate) * up of bf16 [gate | up] rows of 2 F (row stride ldgu) in 8 bits, one scale a row.
TPLR_API int tplr_swiglu_q8(const void* gu, ll ldgu, void* q, ll ldq, float* scale, ll T, int F, void* stream) {
  TPLR_ENTER();
  RowsArgs p = {};
  p.a = (const bf16*)gu; p.lda = ldgu; p.q = (int8_t*)q; p.ldq = ldq; p.scale = scale; p.scale_row = 1; p.T = T; p.D = F;
  return rows_q8<SWIGLU_ROWS>(p, stream);
}

// y[T, D] (dense bf16) = q * scale, times w[column] where w is given; a scale for the row (group D or more) or for every 64 columns.
TPLR_API int tplr_dequantize_rows(const void* q, ll ldq, const float* scale, ll scale_row, ll scale_group, int group, const void* w, void* y,
                                  ll T, int D, void* stream) {
  TPLR_ENTER();
  if (T <= 0) return 0;
  if (D <= 0 || (group != GROUP && group < D)) return (int)cudaErrorInvalidValue;
  if (D % 8 == 0 && ldq % 8 == 0 && T <= 0x7fffffffLL && whole_pieces(q, w, y)) {
    int tpr = row_threads(D / 8, 4);
    if (tpr > 256) tpr = 256;
    const int rows = 256 / tpr;
    return (int)launch_pdl(dequantize_kernel, (unsigned)((T + rows - 1) / rows), 256, 0, (cudaStream_t)stream, (const int8_t*)q, ldq, scale,
                           scale_row, group == GROUP ? scale_group : 0, (const bf16*)w, (bf16*)y, T, D, tpr);
  }
  return (int)launch_pdl(dequantize_any_kernel, waves(T, 64), 256, 0, (cudaStream_t)stream, (const int8_t*)q, ldq, scale,
                         scale_row, scale_group, group == GROUP, (const bf16*)w, (bf16*)y, T, D);
}

// Rows (each of D elements) of the fp32 workspace that tplr_rmsnorm_saved8_bwd takes: its CTAs at most.
TPLR_API int tplr_rmsnorm_saved8_parts(ll T, int D) { return (int)waves(T, 4); }

// dx of the norm from its rows in 8 bits (dres null: 0), and its weight's gradient: added into dw_add (fp32) or stored in dw_out (bf16); both
// null: not formed.
TPLR_API int tplr_rmsnorm_saved8_bwd(const void* dy, const void* q, ll ldq, const float* scale, ll scale_row, ll scale_group,
                                     const float* rstd, const void* w, const void* dres, void* dx, float* part, float* dw_add, void* dw_out,
                                     ll T, int D, void* stream) {
  TPLR_ENTER();
  if (T <= 0) return 0;
  if (D <= 0) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  const bf16 *g = (const bf16*)dy, *wp = (const bf16*)w, *a = (const bf16*)dres;
  const int8_t* c = (const int8_t*)q;
  int n;
  cudaError_t e;
  if (D % 8 || D > 8192 || ldq % 8 || !whole_pieces(dy, q, w, dres, dx, part)) {
    const int block = D <= 1024 ? 256 : D <= 2048 ? 512 : 1024;
    n = (int)waves(T, block == 256 ? 4 : 2048 / block);
    auto kern = block == 256 ? rmsnorm_saved8_bwd_any_kernel<4, 256> : block == 512 ? rmsnorm_saved8_bwd_any_kernel<4, 512>
                : D <= 4096 ? rmsnorm_saved8_bwd_any_kernel<4, 1024> : D <= 8192 ? rmsnorm_saved8_bwd_any_kernel<8, 1024> : rmsnorm_saved8_bwd_any_kernel<0, 1024>;
    e = launch_pdl(kern, n, block, 0, st, g, c, ldq, scale, scale_row, scale_group, rstd, wp, a, (bf16*)dx, part, T, D);
  } else {
    const int two = row_threads(D / 8, 2), three = row_threads(D / 8, 3);
    const int vpl = three <= 128 && 3 * three < 2 * two ? 3 : 2, tpr = vpl == 3 ? three : two, block = vpl == 3 ? 128 : tpr > 256 ? 512 : 256;
    const int rows = block / tpr;
    n = (int)waves((T + rows - 1) / rows, bwd_ctas(vpl, block));
    auto kern = vpl == 3 ? rmsnorm_saved8_bwd_kernel<3, 128> : block == 512 ? rmsnorm_saved8_bwd_kernel<2, 512> : rmsnorm_saved8_bwd_kernel<2, 256>;
    const size_t smem = (size_t)BWD_STAGES * vpl * 40 * block;
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return (int)e;
    e = launch_pdl(kern, n, block, smem, st, g, c, ldq, scale, scale_row, scale_group, rstd, wp, a, (bf16*)dx, part, T, D, tpr);
  }
  if (e != cudaSuccess || (!dw_add && !dw_out)) return (int)e;
  return (int)launch_pdl(sum_parts_kernel, (D + 31) / 32, 1024, 0, st, part, n, D, dw_add, (bf16*)dw_out);
}

// The activation of a dense fp32 [gate | up] projection, and the projection in 8 bits (rows of ldq >= 2 F bytes) by 64 columns of each half.
TPLR_API int tplr_swiglu_saved8(const float* gu, void* act, void* q, ll ldq, float* scale, ll scale_row, ll scale_group, ll T, int F,
                                void* stream) {
  TPLR_ENTER();
  if (T <= 0) return 0;
  if (F <= 0 || ldq < 2LL * F) return (int)cudaErrorInvalidValue;
  const ll groups = T * ((F + GROUP - 1) / GROUP);
  return (int)launch_pdl(swiglu_saved8_kernel, waves((groups + 7) / 8, 16), 256, 0, (cudaStream_t)stream, gu, (bf16*)act, (int8_t*)q, ldq,
                         scale, scale_row, scale_group, T, F);
}

// Its backward: dact dense fp32 [T, F] -> dgu = [dgate | dup] (dense bf16) and the activation again.
TPLR_API int tplr_swiglu_saved8_bwd(const float* dact, const void* q, ll ldq, const float* scale, ll scale_row, ll scale_group, void* dgu,
                                    void* act, ll T, int F, void* stream) {
  TPLR_ENTER();
  if (T <= 0) return 0;
  if (F <= 0) return (int)cudaErrorInvalidValue;
  return (int)launch_pdl(swiglu_saved8_bwd_kernel, waves((T * F + 255) / 256, 16), 256, 0, (cudaStream_t)stream, dact, (const int8_t*)q, ldq,
                         scale, scale_row, scale_group, (bf16*)dgu, (bf16*)act, T, F);
}

extern "C" ll tplr_gemm2_q8_workspace(int M, int N, int K);
extern "C" int tplr_gemm2_q8(const void* X, const void* W, const float* sx, const float* sw, void* C, int* ws, int M, int N, int K, ll ldx, ll ldw,
                             ll ldc, int out_fp32, unsigned int* status, void* stream);
extern "C" int tplr_gemm_q8_stream(const void* X, const void* W, const float* sx, const float* sw, void* C, int T, int N, int K, ll ldx, ll ldw,
                                   ll ldc, int out_fp32, unsigned int* status, void* stream);

// Which kernel multiplies 8-bit rows: up to 8 tokens the one that loads the weight into registers, up to 64 (or with a longer K) the weight's
// rows as the tensor core's long side with K cut over clusters, more on CTA pairs.  Microseconds, the three in that order, inner dimension x
// channels, at 8 | 32 | 64 tokens, weights of 500 MB in turn as the layers of a model take theirs: 2048 x 2048 2.8, 4.1, 7.3 | -, 5.1, 7.4 | -, 7.0, 7.7;
// 4096 x 6144 7.0, 8.8, 14.6 | -, 9.8, 11.1 | -, 12.1, 11.4; 2048 x 16384 9.4, 10.0, 15.0 | -, 10.8, 13.4 | -, 13.3, 13.2; 8192 x 2048 7.4, 7.3, 10.8 | -,
// 8.1, 10.0 | -, 9.8, 10.4; 14336 x 4096 -, 13.6, 20.9 | -, 13.9, 18.1 | -, 15.8, 18.9.  One weight again and again, out of L2, the order is the same
// (2048 x 16384: 7.1, 6.9, 13.2 | -, 7.6, 11.2 | -, 10.5, 10.6).  At 128 tokens, out of L2: the second 10.4 to 19.6, pairs 7.9 to 19.8.  The bytes of the
// weight alone take 5.1 us at 2048 x 16384 and 9.0 at 14336 x 4096.
static bool few_tokens(int T, int K) { return T <= FEW && K <= 8192; }
static bool streamed(int T) { return T <= 64; }

// int32 elements of the workspace that tplr_gemm_q8 takes for this size (0: none).
TPLR_API ll tplr_gemm_q8_workspace(int T, int N, int K) { return streamed(T) ? 0 : tplr_gemm2_q8_workspace(T, N, K); }

// y[T, N] = sx[t] * sw[n] * (x w^T) for int8 rows x [T, K] and w [N, K] on 16-byte boundaries, y bf16 or fp32 with row stride ldy.  The
// bytes of a row from K to the next 16-byte boundary may be read and count for nothing.  ws: tplr_gemm_q8_workspace elements, 16-byte
// aligned.
TPLR_API int tplr_gemm_q8(const void* x, const void* w, const float* sx, const float* sw, void* y, void* ws, int T, int N, int K, ll ldx, ll ldw,
                          ll ldy, int out_fp32, unsigned int* status, void* stream) {
  TPLR_ENTER();
  if (T <= 0 || N <= 0) return 0;
  if (K <= 0 || K > 131072 || (ldx | ldw) % 16 || (((uintptr_t)x | (uintptr_t)w) & 15)) return (int)cudaErrorInvalidValue;
  if (few_tokens(T, K)) {
    auto few = K % 16 ? (out_fp32 ? gemm_q8_few<float, false, true> : gemm_q8_few<bf16, false, true>)
                      : (out_fp32 ? gemm_q8_few<float, false, false> : gemm_q8_few<bf16, false, false>);
    return few(x, w, sx, sw, y, T, N, K, ldx, ldw, ldy, stream);
  }
  if (streamed(T)) return tplr_gemm_q8_stream(x, w, sx, sw, y, T, N, K, ldx, ldw, ldy, out_fp32, status, stream);
  return tplr_gemm2_q8(x, w, sx, sw, y, (int*)ws, T, N, K, ldx, ldw, ldy, out_fp32, status, stream);
}

// tplr_quantize_rows (one scale a row) of bf16 x and tplr_gemm_q8 in one launch, the same bits; y bf16.  -111: more tokens or values than a
// CTA holds, or rows that are not whole 16-byte pieces.
TPLR_API int tplr_linear_q8_few(const void* x, const void* w, const float* sw, void* y, int T, int N, int K, ll ldx, ll ldw, ll ldy, void* stream) {
  TPLR_ENTER();
  if (T <= 0 || N <= 0) return 0;
  if (T > FEW || K <= 0 || (ll)T * K > HELD_MOST || K % 8 || ldx % 8 || ldw % 16 || !whole_pieces(x, w)) return -111;
  int share = 256;
  while (share * T > 256) share /= 2;
  if ((K + 15) / 16 * 2 > share * HELD_PIECES) return -111;
  return gemm_q8_few<bf16, true, false>(x, w, nullptr, sw, y, T, N, K, ldx, ldw, ldy, stream);
}
