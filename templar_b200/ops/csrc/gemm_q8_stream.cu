// Product of few tokens with an 8-bit weight (sm_100a): the weight's bytes, read once, are what it costs.
//
//   y[t, n] = sx[t] * sw[n] * sum_k x[t, k] w[n, k]        T up to 64
//
// The weight takes the tensor core's long side: a CTA's tile is 128 output channels (rows of w, lanes of tensor memory) by all the
// tokens (8 to 64 columns), so no instruction multiplies rows that are not there, as a 256-row tile of tokens would.  A ring of up to
// 221 KB per SM is in flight all the time.  Where the blocks of 128 channels leave SMs idle, K is cut over the two to eight CTAs of a
// cluster; each sends the int32 sums of a token to the CTA that owns it, 16 bytes a store into its shared memory, and the owners add
// and scale: the sum of integers is the same in any order, and no workspace or second launch is needed.
// Weights in turn, so that each comes from memory: 32 x 4096 x 6144 (two CTAs a block) 9.8 us, 32 x 14336 x 4096 (four) 13.9, 64 x 2048 x 16384
// (one) 13.3: 2.5 to 4.2 TB/s of weight; one weight again and again, out of L2: 7.6, 9.6 and 10.5.  3 us of each are launch, barriers, tensor memory, first
// loads and the last sums.  With the owners loading from the others' memory instead, one word at a time, 128 tokens of 2048 x 2048 took
// 49 us, 10.4 in this form; from 65 on CTA pairs are as fast or faster.
// No load carries a cluster-multicast qualifier.  Every wait is bounded; on expiry TPLR_ST_WAIT_TIMEOUT is set and all roles return.
#include "quant.cuh"
#include "tcgen05.cuh"

namespace {
using namespace tplr_tc;
typedef long long ll;

constexpr int ROWS = 128, KB = 128, W_STAGE = ROWS * KB, SMEM = 225 * 1024, MAX_STAGES = 13, THREADS = 192, MAX_TOKENS = 64, MAX_SPLIT = 8;

struct StreamParams {
  CUtensorMap tmW, tmX;
  const float *sx, *sw;
  void* y;
  ll ldy;
  int T, N, K, tn;             // tn: columns of the tile, T rounded up to 8, 16, 32 or 64
  int split, k_per;            // CTAs of a cluster, k blocks of each
  int n_stages;
  int mine;                    // tokens whose sums meet in one CTA of a cluster, a multiple of 4
  int fp32;
  unsigned int* status;
};

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t mapa(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  return a;
}
__device__ __forceinline__ void st_cluster4(uint32_t a, const uint32_t* v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void store(const StreamParams& p, int t, int n, float v) {
  if (p.fp32) reinterpret_cast<float*>(p.y)[t * p.ldy + n] = v;
  else reinterpret_cast<__nv_bfloat16*>(p.y)[t * p.ldy + n] = __float2bfloat16(v);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, DescBase a, uint32_t a_off16, DescBase b, uint32_t b_off16, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %5, p;\n\t}"
      ::"r"(tmem_d), "r"(a.lo + a_off16), "r"(a.hi), "r"(b.lo + b_off16), "r"(b.hi), "r"(idesc), "r"(accumulate) : "memory");
}

__global__ void __launch_bounds__(THREADS, 1) gemm_q8_stream_kernel(const __grid_constant__ StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t bar_full[MAX_STAGES], bar_empty[MAX_STAGES], bar_done;
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = p.split > 1 ? cluster_ctarank() : 0;
  const int n0 = blockIdx.x / p.split * ROWS;
  const int x_stage = p.tn * KB, n_stages = p.n_stages;
  const int k_all = (p.K + KB - 1) / KB, kb0 = (int)rank * p.k_per, k_blocks = min(p.k_per, k_all - kb0);
  const uint32_t tmem_cols = p.tn < 32 ? 32u : (uint32_t)p.tn;
  volatile int* abort_flag = &s_abort;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < MAX_STAGES; ++s) { mbar_init(smem_u32(&bar_full[s]), 1); mbar_init(smem_u32(&bar_empty[s]), 1); }
    mbar_init(smem_u32(&bar_done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (threadIdx.x == 32) { prefetch_map(&p.tmW); prefetch_map(&p.tmX); }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem_base)), "r"(tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  if (p.split > 1) cluster_sync_all();             // the others' shared memory is there
  tcgen05_fence_after();
  grid_wait();
  grid_release();
  const uint32_t tmem = s_tmem_base, sW = smem_u32(smem), sX = sW + n_stages * W_STAGE;

  if (warp == 0) {
    // ----------------------------- producer ------------------------------------------
    const bool leader = elect_one();
    uint32_t s = 0, ph = 0, it = 0;
    for (int kb = 0; kb < k_blocks; ++kb, ++it) {
      if (!mbar_wait_warp(smem_u32(&bar_empty[s]), ph ^ 1u, abort_flag)) break;
      if (leader) {
        const uint32_t fb = smem_u32(&bar_full[s]);
        mbar_expect_tx(fb, W_STAGE + x_stage);
        tma_load_2d(sW + s * W_STAGE, &p.tmW, fb, (kb0 + kb) * KB, n0);
        tma_load_2d(sX + s * x_stage, &p.tmX, fb, (kb0 + kb) * KB, 0);
      }
      if (++s == (uint32_t)n_stages) { s = 0; ph ^= 1u; }
    }
    if (leader) {                    // every armed stage has landed before the CTA may retire or reuse the ring
      Drain drain;
      for (uint32_t back = 0; back < (uint32_t)n_stages && back < it; ++back) {
        const uint32_t j = it - 1 - back;
        drain.wait(smem_u32(&bar_full[j % n_stages]), (j / n_stages) & 1);
      }
    }
  } else if (warp == 1) {
    // ----------------------------- issuer --------------------------------------------
    const bool leader = elect_one();
    const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.tn >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
    const DescBase dW = desc_base(sW, 16, 1024), dX = desc_base(sX, 16, 1024);
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int kb = 0; kb < k_blocks; ++kb) {
      if (!(ok = mbar_wait_warp(smem_u32(&bar_full[s]), ph, abort_flag))) break;
      tcgen05_fence_after();
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_i8(tmem, dW, s * (W_STAGE >> 4) + kk * 2, dX, s * ((uint32_t)x_stage >> 4) + kk * 2, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
        umma_commit(smem_u32(&bar_empty[s]));
      }
      if (++s == (uint32_t)n_stages) { s = 0; ph ^= 1u; }
    }
    if (ok && leader) umma_commit(smem_u32(&bar_done));
  }
  // ----------------------------- sums out of tensor memory -----------------------------
  // A lane has a channel.  One CTA a block of channels: straight to y, token after token.  Several: `mine` consecutive tokens to each CTA
  // of the cluster, four of a channel in 16 bytes: [sender][four tokens][channel][4] behind the ring.
  const int c = (warp & 3) * 32 + lane, n = n0 + c, first = p.split > 1 ? (int)rank * p.mine : 0;
  const uint32_t part = sX + n_stages * x_stage, part_cta = (uint32_t)p.mine * ROWS * 4u;
  float sn = 0.f, st[2] = {};
  bool plain = true;                               // every product of this warp's scales is a normal number or zero
  auto value = [&](uint32_t sum, float t) { return plain ? (float)(int)sum * (t * sn) : scaled_far((int)sum, t, sn); };
  if (warp >= 2) {
    sn = n < p.N ? p.sw[n] : 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (first + j * 32 + lane < p.T) st[j] = p.sx[first + j * 32 + lane];
    const ScaleRange r0 = scale_range(st[0]), r1 = scale_range(st[1]);
    plain = __all_sync(0xffffffffu, in_range(r0, sn) && in_range(r1, sn));
    const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_done), 0, abort_flag));
    tcgen05_fence_after();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (!ok || j * 32 >= p.T) break;
      uint32_t r[32];
      tmem_ld32(tmem + j * 32 + ((uint32_t)((warp & 3) * 32) << 16), r);
      if (p.split > 1) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const int t = j * 32 + e, owner = t / p.mine;
          if (t < p.T) st_cluster4(mapa(part + rank * part_cta + (uint32_t)((t - owner * p.mine) * ROWS + c * 4) * 4u, (uint32_t)owner), r + e);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float t = __shfl_sync(0xffffffffu, st[j], e);
          if (j * 32 + e < p.T && n < p.N) store(p, j * 32 + e, n, value(r[e], t));
        }
      }
    }
  }
  __syncwarp();
  tcgen05_fence_before();
  if (p.split > 1) {
    cluster_sync_all();
    if (warp >= 2) {
      for (int e = 0; e < p.mine && first + e < p.T; e += 4) {     // 32 tokens at most: two CTAs or more
        int sum[4] = {};
#pragma unroll 4
        for (int k = 0; k < p.split; ++k) {
          int v[4];
          asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                       : "r"(part + (uint32_t)k * part_cta + (uint32_t)(e * ROWS + c * 4) * 4u));
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] += v[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float t = __shfl_sync(0xffffffffu, st[0], e + i);
          if (first + e + i < p.T && n < p.N) store(p, first + e + i, n, value((uint32_t)sum[i], t));
        }
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
  }
  if (threadIdx.x == 0 && s_abort && p.status) atomicOr(p.status, TPLR_ST_WAIT_TIMEOUT);
}
}  // namespace

// tplr_gemm2_q8 for T <= 64 tokens.
TPLR_API int tplr_gemm_q8_stream(const void* X, const void* W, const float* sx, const float* sw, void* C, int T, int N, int K, ll ldx, ll ldw,
                                 ll ldc, int out_fp32, unsigned int* status, void* stream) {
  TPLR_ENTER();
  if (T <= 0 || N <= 0 || K <= 0) return 0;
  if (T > MAX_TOKENS || K > 131072 || (ldx % 16) || (ldw % 16) || (((uintptr_t)X | (uintptr_t)W) & 15)) return -101;
  StreamParams p = {};
  p.tn = T <= 8 ? 8 : T <= 16 ? 16 : T <= 32 ? 32 : 64;
  if (!make_map_u8(&p.tmW, W, K, N, ldw, KB, ROWS) || !make_map_u8(&p.tmX, X, K, T, ldx, KB, p.tn)) return -102;
  p.sx = sx; p.sw = sw; p.y = C; p.ldy = ldc; p.T = T; p.N = N; p.K = K; p.fp32 = out_fp32; p.status = status;
  const int blocks = (N + ROWS - 1) / ROWS, k_all = (K + KB - 1) / KB;
  cudaError_t e = cudaFuncSetAttribute(gemm_q8_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1] = pdl_attr();
  // the largest split whose clusters are all resident at once: a second wave costs more than the wider cut gains
  int split = 1;
  for (int s = 2; s <= MAX_SPLIT && s <= k_all; s *= 2) {
    static int resident[MAX_SPLIT + 1] = {};
    if (resident[s] == 0) {
      attr[0].val.clusterDim.x = (unsigned)s;
      cfg.gridDim = dim3((unsigned)(tplr_sm_count() / s * s)); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM;
      cfg.attrs = attr; cfg.numAttrs = 1;
      int n = 0;
      if ((e = cudaOccupancyMaxActiveClusters(&n, gemm_q8_stream_kernel, &cfg)) != cudaSuccess) return (int)e;
      resident[s] = n > 0 ? n : -1;
    }
    if (blocks <= resident[s]) split = s;
  }
  p.k_per = (k_all + split - 1) / split;
  p.split = (k_all + p.k_per - 1) / p.k_per;       // every CTA has work
  p.mine = (T + p.split - 1) / p.split;
  p.mine = p.split > 1 ? (p.mine + 3) / 4 * 4 : T;
  const int part = p.split > 1 ? p.split * p.mine * ROWS * 4 : 0;
  p.n_stages = (SMEM - 1024 - part) / (W_STAGE + p.tn * KB);
  if (p.n_stages > MAX_STAGES) p.n_stages = MAX_STAGES;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  cfg.gridDim = dim3((unsigned)(blocks * p.split)); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM;
  cfg.stream = (cudaStream_t)stream; cfg.attrs = attr; cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, gemm_q8_stream_kernel, p);
}
