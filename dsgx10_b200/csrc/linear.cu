// Dense INT4-g32 matrix-vector products for 1..16 rows: out[m][n] = sum_k x[m][k] W[n][k], W = (u - z) s, f32 sums; the
// residual added, or with a second matrix silu(x W^T) * (x W_up^T).  (The expert kernels' weight blocks, decode_int4.cu.)
//
// Bound: the weights are read once (0.578 bytes a weight), so HBM; the conversion of the nibbles in registers is the next
// limit (int4_pair.cuh).  Work is cut in units of 16 output rows (SwiGLU: 8 gate + 8 up) and a unit in pairs of 8 x 512
// blocks.  A CTA owns a run of units and its 16 stream warps take the run's block pairs in turn, each through a private
// ring of bulk copies: every SM streams from one contiguous run whatever N and K are, no warp owns more than a block pair
// at a time, and the launch ends within one unit on every SM.  A warp's sums of a block pair go to shared memory; one more
// warp adds a unit's partial sums in ascending k and writes the outputs, so that the stream never waits for a reduction.
//
// K over a cluster: with C > 1 (1, 2, 4 or 8 CTAs) the ranks of a cluster take consecutive runs of K of the same units.  The
// activations of M rows are held in shared memory for a rank's own run only, and a matrix with few units still occupies
// every SM.  A rank's partial sums of a unit go to the unit's owner (unit modulo C) through distributed shared memory, and the
// owner adds the ranks.
//
// The order of a sum is the same for every cluster size: K's blocks fall into eight runs (block nb r / 8 on), a run is summed
// in ascending order from zero, and the runs are joined as a binary tree, ((r0 + r1) + (r2 + r3)) + ((r4 + r5) + (r6 + r7)),
// of which a rank holds a whole subtree.  So a row's bits do not depend on the rows beside it or on their number.
#include <atomic>

#include "common.cuh"
#include "int4_pair.cuh"
#include "kernels.h"

namespace dsgx {

namespace {

constexpr int kSlotsOwned = 2;   // a rank's receive buffers for units that the cluster has in flight
constexpr int kMaxCluster = 8;
constexpr int kRuns = 8;         // the parts of K whose sums are joined as a tree
constexpr size_t kSmemMax = 227 * 1024;

// W stream warps, P partial sums in flight; S sets of four tokens
template <int S_, int W_, int NST_, int P_>
struct LinVar {
  static constexpr int S = S_, W = W_, NST = NST_, P = P_;
  static constexpr int kThreads = (W + 1) * 32;
  static constexpr int kPart = 256 * S;  // bytes of a block pair's (or a rank's) sums: [S][32 lanes][2] f32
  static constexpr size_t kFixed = (size_t)W * NST * kPairStage + (size_t)P * kPart + 128;
  static size_t smem(int M, int kblocks, int C) {
    return kFixed + (C > 1 ? (size_t)kSlotsOwned * kMaxCluster * kPart : 0) + (size_t)kblocks * M * 1024 + 32 +
           (W * NST + kSlotsOwned * (1 + kMaxCluster)) * 8 + P * 4 + 64;
  }
};

DSGX_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
DSGX_DEV uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
DSGX_DEV void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
DSGX_DEV void remote_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
DSGX_DEV void st_remote(uint32_t addr, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(v.x), "f"(v.y) : "memory");
}
// bounded wait with the cluster's scope (the barrier's arrivals come from other CTAs)
DSGX_DEV bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (clock64() - t0 > kWaitCycles) return false;
  }
}
DSGX_DEV float2 add2(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }
DSGX_DEV int ld_shared_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}
DSGX_DEV void st_shared_release(int* p, int v) {
  asm volatile("st.release.cta.shared::cta.s32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}

template <class V>
__global__ void __launch_bounds__(V::kThreads, 1) k_linear_int4(const LinearParams p) {
  constexpr int S = V::S, W = V::W, NST = V::NST, P = V::P, kPart = V::kPart;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = p.cluster;
  const uint32_t rank = C > 1 ? cluster_rank() : 0;
  const int cl = blockIdx.x / C, ncl = gridDim.x / C;
  // this cluster's units and this rank's blocks of K
  const int u0 = (int)((long long)p.units * cl / ncl), u1 = (int)((long long)p.units * (cl + 1) / ncl);
  const int b0 = p.nb * (int)rank / C, nbk = p.nb * ((int)rank + 1) / C - b0;

  uint8_t* ring = smem;
  uint8_t* part = ring + (size_t)W * NST * kPairStage;                 // [P][S][32][2] f32
  uint8_t* recv = part + (size_t)P * kPart;                            // [kSlotsOwned][C][S][32][2] f32
  uint8_t* xt = recv + (C > 1 ? (size_t)kSlotsOwned * kMaxCluster * kPart : 0);
  uint8_t* zero = xt + (size_t)p.xblocks * p.M * 1024;                  // 32 bytes
  uint64_t* bars = reinterpret_cast<uint64_t*>(zero + 32);
  uint64_t* rfull = bars + W * NST;                                    // [kSlotsOwned] every rank's sums are in my buffer
  uint64_t* rfree = rfull + kSlotsOwned;                               // [owner][kSlotsOwned] that owner's buffer may be written
  int* cnt = reinterpret_cast<int*>(rfree + kMaxCluster * kSlotsOwned);  // [P] block pairs summed of a unit in flight
  int* done = cnt + P;                                                 // block pairs whose unit has been added up
  int* fail = done + 1;                                                // a bounded wait ran out

  if (warp < W && lane == 0)
    for (int s = 0; s < NST; ++s) mbar_init(bars + warp * NST + s, 1);
  if (threadIdx.x == W * 32) {
    for (int s = 0; s < kSlotsOwned; ++s) mbar_init(rfull + s, 32 * C);
    for (int s = 0; s < kMaxCluster * kSlotsOwned; ++s) mbar_init(rfree + s, 1);
    *done = 0, *fail = 0;
  }
  for (int i = threadIdx.x; i < P; i += V::kThreads) cnt[i] = 0;
  if (threadIdx.x < 8) reinterpret_cast<uint32_t*>(zero)[threadIdx.x] = 0;
  mbar_fence_init();
  __syncwarp();
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  pdl_launch_dependents();

  const int total = (u1 - u0) * nbk;  // this CTA's block pairs
  const size_t strip = (size_t)p.nb * kQBlk;
  const bool glu = p.w_up != nullptr;

  // ---- the first weights are requested before the activations are there (they do not depend on the launches before) ------
  uint8_t* myring = ring + (size_t)warp * NST * kPairStage;
  uint64_t* mybar = bars + warp * NST;
  uint32_t issued = 0;
  int pj = warp;
  const uint64_t pol = policy_evict_first();
  auto issue = [&]() {
    const int u = u0 + pj / nbk, b = b0 + pj % nbk;
    const uint8_t *a, *c;
    if (glu) {
      a = p.w + (size_t)u * strip, c = p.w_up + (size_t)u * strip;
    } else {
      a = p.w + (size_t)(2 * u) * strip;
      c = 2 * u + 1 < p.n8 ? a + strip : a;  // (an odd number of strips: the last unit's second half is not written)
    }
    uint8_t* st = myring + (issued % NST) * kPairStage;
    uint64_t* bar = mybar + issued % NST;
    mbar_expect_tx(bar, kPairBytes);
    bulk_g2s_hint(st, a + (size_t)b * kQBlk, kQBlk, bar, pol);
    bulk_g2s_hint(st + kQBlk, c + (size_t)b * kQBlk, kQBlk, bar, pol);
    ++issued, pj += W;
  };
  if (warp < W && lane == 0)
    for (int s = 0; s < NST && pj < total; ++s) issue();

  // ---- this rank's activations ------------------------------------------------------------------------------------------
  pdl_wait();
  {
    const bool vec = p.x_vec != 0;
    for (int i = threadIdx.x; i < nbk * 32 * p.M; i += V::kThreads) {
      const int kg = i / p.M, r = i % p.M;
      uint4 o[2];
      tile_group(o, p.x + (size_t)r * p.ldx, b0 * 512 + 16 * kg, p.K, vec);
      uint4* d = reinterpret_cast<uint4*>(xt + (size_t)i * 32);
      d[0] = o[0], d[1] = o[1];
    }
  }
  __syncthreads();

  if (warp < W) {
    // ---- stream warps ---------------------------------------------------------------------------------------------------
    XCols<S> cols;
    xcols_int4<S>(cols, xt, p.M, zero, lane, [&](int s, int j) { return 4 * s + j < p.M ? 4 * s + j : -1; });
    uint32_t consumed = 0;
    for (int j = warp; j < total; j += W) {
      const uint32_t si = consumed % NST;
      if (!mbar_wait(mybar + si, (consumed / NST) & 1)) {
        *fail = 1;
        break;
      }
      float acc[S][2];
#pragma unroll
      for (int s = 0; s < S; ++s) acc[s][0] = acc[s][1] = 0.f;
      XCols<S> xc = cols;
#pragma unroll
      for (int s = 0; s < S; ++s) xc.p[s] += (size_t)(j % nbk) * 8 * xc.step[s];
      const uint8_t* st = myring + si * kPairStage;
      int4_pair<S>(acc, st, st + kQBlk, xc, lane);
      ++consumed;
      __syncwarp();
      if (lane == 0 && pj < total) issue();
      // the sums into the partial buffer, once the buffer's last unit has been added up
      if (j >= ld_shared_acquire(done) + P) {
        const long long t0 = clock64();
        bool ok = true;
        while (ok && j >= ld_shared_acquire(done) + P) ok = clock64() - t0 < kWaitCycles;
        if (!ok) {
          *fail = 1;
          break;
        }
      }
      float2* d = reinterpret_cast<float2*>(part + (size_t)(j % P) * kPart) + lane;
#pragma unroll
      for (int s = 0; s < S; ++s) d[32 * s] = make_float2(acc[s][0], acc[s][1]);
      __threadfence_block();
      __syncwarp();
      if (lane == 0) atomicAdd(cnt + (j / nbk) % P, 1);
    }
    if (lane == 0)  // (only after a wait that ran out: no copy is left in flight)
      for (; consumed < issued; ++consumed) mbar_wait(mybar + consumed % NST, (consumed / NST) & 1);
  } else {
    // ---- the adding warp ------------------------------------------------------------------------------------------------
    const int g = lane >> 2, t = lane & 3;
    bool ok = true;
    for (int i = 0; i < u1 - u0 && ok; ++i) {
      const int* c = cnt + i % P;
      if (ld_shared_acquire(c) < nbk) {
        const long long t0 = clock64();
        while (ok && ld_shared_acquire(c) < nbk) ok = clock64() - t0 < kWaitCycles;
        if (!ok) break;
      }
      // this rank's runs of K (kRuns / C of the eight), each in ascending order, joined pairwise
      float2 a[S], lv[3][S];
      int b = 0;
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        if (r < kRuns / C) {
          const int e = p.nb * ((int)rank * (kRuns / C) + r + 1) / kRuns - b0;
#pragma unroll
          for (int s = 0; s < S; ++s) a[s] = make_float2(0.f, 0.f);
          for (; b < e; ++b) {
            const float2* d = reinterpret_cast<const float2*>(part + (size_t)((i * nbk + b) % P) * kPart) + lane;
#pragma unroll
            for (int s = 0; s < S; ++s) a[s] = add2(a[s], d[32 * s]);
          }
          int l = 0;
#pragma unroll
          for (int k = r; k & 1; k >>= 1, ++l)
#pragma unroll
            for (int s = 0; s < S; ++s) a[s] = add2(lv[l][s], a[s]);
          if (l < 3)
#pragma unroll
            for (int s = 0; s < S; ++s) lv[l][s] = a[s];
        }
      }
      __syncwarp();
      if (lane == 0) {
        cnt[i % P] = 0;
        st_shared_release(done, (i + 1) * nbk);
      }
      if (C > 1) {
        // to the unit's owner, once it has let go of the unit that had the buffer before; the owner adds the ranks in order
        const int owner = i % C, slot = (i / C) % kSlotsOwned, turn = i / C / kSlotsOwned;
        if (turn > 0 && !mbar_wait_cluster(rfree + owner * kSlotsOwned + slot, (turn - 1) & 1)) {
          ok = false;
          break;
        }
        const uint32_t to = map_rank(smem_u32(recv) + (uint32_t)((slot * kMaxCluster + (int)rank) * kPart + lane * 8), owner);
#pragma unroll
        for (int s = 0; s < S; ++s) st_remote(to + 256 * s, a[s]);
        remote_arrive(map_rank(smem_u32(rfull + slot), owner));
        if (owner != (int)rank) continue;
        if (!mbar_wait_cluster(rfull + slot, turn & 1)) {
          ok = false;
          break;
        }
        const float2* d = reinterpret_cast<const float2*>(recv + (size_t)slot * kMaxCluster * kPart) + lane;
        constexpr int kStep = kPart / 8;  // the ranks' sums, joined pairwise like the runs
        auto rank_pair = [&](int r, int s) { return add2(d[r * kStep + 32 * s], d[(r + 1) * kStep + 32 * s]); };
#pragma unroll
        for (int s = 0; s < S; ++s) {
          a[s] = rank_pair(0, s);
          if (C >= 4) a[s] = add2(a[s], rank_pair(2, s));
          if (C >= 8) a[s] = add2(a[s], add2(rank_pair(4, s), rank_pair(6, s)));
        }
        __syncwarp();
        if (lane < C) remote_arrive(map_rank(smem_u32(rfree + rank * kSlotsOwned + slot), lane));
      }
      const int unit = u0 + i;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int m = 4 * s + t;
        if (m < p.M) {
          if (glu) {
            const int n = 8 * unit + g;
            if (n < p.N) {
              const float h = __fmul_rn(silu(a[s].x), a[s].y);
              if (p.out_f32) reinterpret_cast<float*>(p.out)[(size_t)m * p.ldo + n] = h;
              else reinterpret_cast<__nv_bfloat16*>(p.out)[(size_t)m * p.ldo + n] = __float2bfloat16_rn(h);
            }
          } else {
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              const int n = 16 * unit + 8 * hi + g;
              if (n < p.N) {
                float y = hi ? a[s].y : a[s].x;
                if (p.res) y = __fadd_rn(y, __bfloat162float(p.res[(size_t)m * p.ldr + n]));
                if (p.out_f32) reinterpret_cast<float*>(p.out)[(size_t)m * p.ldo + n] = y;
                else reinterpret_cast<__nv_bfloat16*>(p.out)[(size_t)m * p.ldo + n] = __float2bfloat16_rn(y);
              }
            }
          }
        }
      }
    }
    if (!ok) *fail = 1;
  }
  // (a rank's shared memory is written by the others: nobody leaves before all are done)
  __syncwarp();
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  if (threadIdx.x == 0 && *fail && p.status) atomicCAS(p.status, 0, (int)DSGX_ERR_DEVICE_WAIT);
}

int device_index() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? dev & 63 : 0;
}
// clusters of C CTAs that the device runs at once (asked once per kernel, device and C; the shared memory is given at its most)
template <class V>
cudaError_t resident_clusters(int C, int* n) {
  static std::atomic<int> known[64][kMaxCluster + 1];
  static std::atomic<bool> set[64];
  const int dev = device_index();
  if (!set[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(k_linear_int4<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax);
    if (e != cudaSuccess) return e;
    set[dev].store(true, std::memory_order_release);
  }
  if (C == 1) {
    *n = sm_count();
    return cudaSuccess;
  }
  int v = known[dev][C].load();
  if (!v) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sm_count() / C * C), cfg.blockDim = dim3(V::kThreads), cfg.dynamicSmemBytes = kSmemMax;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    cudaError_t e = cudaOccupancyMaxActiveClusters(&v, k_linear_int4<V>, &cfg);
    if (e != cudaSuccess) return e;
    if (v < 1) return cudaErrorInvalidConfiguration;
    known[dev][C].store(v);
  }
  *n = v;
  return cudaSuccess;
}

// The cluster size: the one whose busiest SM streams the fewest block pairs (ceil(units / clusters) x ceil(blocks / C)),
// among those whose activations fit shared memory; a larger cluster has to save an eighth to be worth its exchange.
template <class V>
cudaError_t launch(LinearParams p, cudaStream_t st, bool* fits) {
  int best = 0, clusters = 1;
  long long best_cost = 0;
  for (int C = 1; C <= kMaxCluster && C <= p.nb; C *= 2) {
    const int kb = (p.nb + C - 1) / C;
    if (V::smem(p.M, kb, C) > kSmemMax) continue;
    int n = 0;
    cudaError_t e = resident_clusters<V>(C, &n);
    if (e != cudaSuccess) return e;
    const long long cost = (long long)((p.units + n - 1) / n) * kb;
    if (!best || cost * 8 <= best_cost * 7) best = C, best_cost = cost, clusters = n;
  }
  *fits = best != 0;
  if (!best) return cudaSuccess;
  p.cluster = best, p.xblocks = (p.nb + best - 1) / best;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.units < clusters ? p.units : clusters) * best), cfg.blockDim = dim3(V::kThreads);
  cfg.dynamicSmemBytes = V::smem(p.M, p.xblocks, best), cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = best, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = best > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k_linear_int4<V>, p);
}

}  // namespace

// One launch for M rows, or *fits = false where their activations do not fit shared memory.
cudaError_t launch_linear_int4(const LinearParams& p, cudaStream_t st, bool* fits) {
  if (p.M <= 4) return launch<LinVar<1, 16, 2, 64>>(p, st, fits);
  if (p.M <= 8) return launch<LinVar<2, 16, 2, 32>>(p, st, fits);
  return launch<LinVar<4, 12, 2, 24>>(p, st, fits);
}

}  // namespace dsgx
