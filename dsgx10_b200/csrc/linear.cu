// Dense INT4-g32 matrix-vector products for 1..16 rows: out[m][n] = sum_k x[m][k] W[n][k], W = (u - z) s, f32 sums; the
// residual added, or with a second matrix silu(x W^T) * (x W_up^T).
//
// Bound: the weights are read once (0.578 bytes a weight), so HBM: 131072 x 4096 takes 58 us for one row and 59 for four, 83 %
// and 81 % of a copy's rate; the copies alone, with nothing computed, take 50.  What is lost beside the launch and the first
// blocks' latency (3.6 us together, all of a small matrix's time) is the conversion and the products (int4_mma.cuh): with
// eight rows (69 us) the schedulers issue every other cycle, none of the pipes is above half, and a warp waits for its own
// chain of loads, MMAs and f32 operations; fewer stream warps lose more (thirteen 70 us), more have no registers.
//
// Work is cut in units of 16 output rows (SwiGLU: 8 gate + 8 up), a unit along K in 1, 2, 4 or 8 tasks, a task in blocks of 16
// rows x 512 k.  A CTA owns a run of units and its stream warps take the run's tasks in turn, each through a private ring of bulk
// copies (one a block), so that every SM streams one contiguous run and the launch ends within a task on every SM.  One warp
// fills all the rings (a copy takes its issuer 130 to 250 cycles; each warp for itself: 12288 x 6144 pair, one row 20.7 us
// instead of 19.5); a task's sums go to shared memory, and one more warp joins the tasks of a unit and writes the outputs, so
// that the stream never waits for a reduction.
//
// Rows 9..16: the clusters of a pair take eight rows and the rest over the same units, the second reads them from L2.  (One
// cluster for all sixteen, two columns of MMAs a weight, took 45 us instead of 38 for 32768 x 4096: its activations leave room
// for eleven warps only, and its loads of them double.)
//
// Weight layout (k_linear_prepare makes it from the experts' 8-row blocks): the blocks of a unit one after the other, 4736
// bytes each.  [8 spans of 64 k][32 lanes][four words]: row g of the first strip and of the second in the span's first group of
// 32, then both in its second; a word = the 8 nibbles k = 32 group + 8 t + 0..7 of lane 4 g + t (nibbles i and i + 4 meet in one
// f16 pair).  [4 x 128 k][8 g][eight bf16 scales: (strip, group) by (first span, second span)].  [8 g][4 x 128 k][the eight zero
// points' nibbles in that order].
// In the experts' blocks a lane's 16 bytes mix two groups in every MMA, so their scales have to go onto the weights (and
// round them) or the MMAs' columns be halved (block_int4.cu: twice the MMAs and activation loads from five rows on; 131072 x
// 4096 and eight rows took 87 us that way).  Here an MMA stays inside one group, its f32 sums take the scale, and all eight
// columns are rows of x.
//
// K over a cluster: with C > 1 (2, 4 or 8 CTAs) the ranks of a cluster take consecutive parts of K of the same units.  The
// activations of M rows are held in shared memory for a rank's own part only, and a matrix with few units still occupies
// every SM.  A rank's sums of a unit go to the unit's owner (unit modulo C) through distributed shared memory; the owner's
// adding warp joins them a few units later, when the others' have arrived.
//
// The order of a sum is the same for every division of the work: K's blocks fall into eight runs (block nb r / 8 on), a run
// is summed in ascending order from zero, and the runs are joined as a binary tree, ((r0 + r1) + (r2 + r3)) + ((r4 + r5) + (r6 +
// r7)), of which a task and a rank hold whole subtrees.  So a row's bits do not depend on the rows beside it or their number.
#include <atomic>

#include "common.cuh"
#include "int4_mma.cuh"
#include "kernels.h"

namespace dsgx {

namespace {

constexpr int kSlotsOwned = 4;   // a rank's receive buffers: units of its own that the cluster has in flight
constexpr int kMaxCluster = 8;
constexpr int kRuns = 8;         // the parts of K whose sums are joined as a tree
constexpr size_t kSmemMax = 227 * 1024;

constexpr int kUnitBlk = 4736;   // 16 rows x 512 k

// W stream warps with NST ring stages each, NP warps that fill the rings, P tasks' sums in flight (a power of two); kCol: four
// rows at most (unit_block4)
template <bool kCol_, int W_, int NP_, int NST_, int P_>
struct LinVar {
  static constexpr int W = W_, NP = NP_, NST = NST_, P = P_;
  static constexpr bool kCol = kCol_;
  static constexpr int kThreads = (W + 1 + NP) * 32;
  static constexpr int kPart = 512;  // bytes of a task's (or a rank's) sums: [32 lanes][4] f32
  static size_t smem(int M, int kblocks, int C) {
    return (size_t)W * NST * kUnitBlk + (size_t)P * kPart + (C > 1 ? (size_t)kSlotsOwned * C * kPart : 0) +
           (size_t)kblocks * (M * 1024 + even(M) * 68) + (kCol ? 256 : 0) + (2 * W * NST + kSlotsOwned * (1 + kMaxCluster)) * 8 + P * 4 + 16 + 128;
  }
  __host__ __device__ static int even(int M) { return (M + 1) & ~1; }
};

// The products of one block, times 2^(E - 24): blk = a lane's four sums (first strip's row g with rows 2 t and 2 t + 1 of x, then
// the second strip's), the spans' first and second groups apart.  st: the stage; x, sx: this lane's activations and group
// sums at the block's first span; span, sspan: bytes from one span to the next.
DSGX_DEV void unit_block8(float (&blk)[4][2], uint32_t st, uint32_t x, uint32_t span, uint32_t sx, uint32_t sspan, int lane) {
  const int g = lane >> 2;
  const uint4 zq = lds_v4(st + 4608 + 16 * g);
  const uint32_t* zw = &zq.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) blk[i][0] = blk[i][1] = 0.f;
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    const uint4 sc = lds_v4(st + 4096 + 128 * jj + 16 * g);
    const uint32_t* sw = &sc.x;
    const uint32_t ze = zw[jj] & 0x0F0F0F0Fu, zo = (zw[jj] >> 4) & 0x0F0F0F0Fu;  // first span's four, second span's four
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint4 w = lds_v4(st + 512 * (2 * jj + q) + 16 * lane), sm = lds_v4(sx);  // (sums: of both groups, the lane's two rows each)
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // the span's two groups
        const uint32_t wa = c ? w.z : w.x, wb = c ? w.w : w.y, wa8 = wa >> 8, wb8 = wb >> 8;
        const float za = minus_zero(q ? zo : ze, 2 * c), zb = minus_zero(q ? zo : ze, 2 * c + 1);
        const float fa = q ? scale_hi(sw[2 * c]) : scale_lo(sw[2 * c]), fb = q ? scale_hi(sw[2 * c + 1]) : scale_lo(sw[2 * c + 1]);
        const uint4 xv = lds_v4(x ^ (c ? 64u : 0u));
        float d[4];
        mma_f16_zero(d, wa & kNib0, wb & kNib0, wa & kNib1, wb & kNib1, xv.x, xv.y);
        mma_f16(d, wa8 & kNib0, wb8 & kNib0, wa8 & kNib1, wb8 & kNib1, xv.z, xv.w);
        const float s0 = __uint_as_float(c ? sm.z : sm.x), s1 = __uint_as_float(c ? sm.w : sm.y);
        blk[0][c] = fmaf(fa, fmaf(za, s0, d[0]), blk[0][c]), blk[1][c] = fmaf(fa, fmaf(za, s1, d[1]), blk[1][c]);
        blk[2][c] = fmaf(fb, fmaf(zb, s0, d[2]), blk[2][c]), blk[3][c] = fmaf(fb, fmaf(zb, s1, d[3]), blk[3][c]);
      }
      x += span, sx += sspan;
    }
  }
}

// The same for up to four rows, with the same bits: column 2 r + c of B is row r in the MMAs of a span's group c and zeros in the
// other group's, so a lane ends with row t's two group sums side by side and packed operations finish them: 46 instructions
// 64 k instead of 60.  x0, x1: where the lane finds group 0's and group 1's activations (zeros: step 0); sx: row t's sums.
DSGX_DEV void unit_block4(float2 (&blk)[2], uint32_t st, uint32_t x0, uint32_t x1, uint32_t step0, uint32_t step1, uint32_t sx, uint32_t sspan,
                          int lane) {
  const int g = lane >> 2;
  const uint4 zq = lds_v4(st + 4608 + 16 * g);
  const uint32_t* zw = &zq.x;
  blk[0] = blk[1] = make_float2(0.f, 0.f);
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    const uint4 sc = lds_v4(st + 4096 + 128 * jj + 16 * g);
    const uint32_t ze = zw[jj] & 0x0F0F0F0Fu, zo = (zw[jj] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint4 w = lds_v4(st + 512 * (2 * jj + q) + 16 * lane), xa = lds_v4(x0), xb = lds_v4(x1);
      const float2 sum = lds_f2(sx);
      x0 += step0, x1 += step1, sx += sspan;
      const uint32_t a8 = w.x >> 8, b8 = w.y >> 8, c8 = w.z >> 8, d8 = w.w >> 8, z = q ? zo : ze;
      float d[4];
      mma_f16_zero(d, w.x & kNib0, w.y & kNib0, w.x & kNib1, w.y & kNib1, xa.x, xa.y);
      mma_f16(d, a8 & kNib0, b8 & kNib0, a8 & kNib1, b8 & kNib1, xa.z, xa.w);
      mma_f16(d, w.z & kNib0, w.w & kNib0, w.z & kNib1, w.w & kNib1, xb.x, xb.y);
      mma_f16(d, c8 & kNib0, d8 & kNib0, c8 & kNib1, d8 & kNib1, xb.z, xb.w);
      const float2 za = make_float2(minus_zero(z, 0), minus_zero(z, 2)), zb = make_float2(minus_zero(z, 1), minus_zero(z, 3));
      const float2 fa = q ? make_float2(scale_hi(sc.x), scale_hi(sc.z)) : make_float2(scale_lo(sc.x), scale_lo(sc.z));
      const float2 fb = q ? make_float2(scale_hi(sc.y), scale_hi(sc.w)) : make_float2(scale_lo(sc.y), scale_lo(sc.w));
      blk[0] = fma2(fa, fma2(za, sum, make_float2(d[0], d[1])), blk[0]);
      blk[1] = fma2(fb, fma2(zb, sum, make_float2(d[2], d[3])), blk[1]);
    }
  }
}

// ---- the weights' own layout, once at load ------------------------------------------------------------------------------
// One CTA a block: strips a and b of a unit (b null: an odd number of strips, zeros) at one 512-k block.
__global__ void __launch_bounds__(256) k_linear_prepare(const uint8_t* __restrict__ w, const uint8_t* __restrict__ w_up, int n8, int nb,
                                                        uint8_t* __restrict__ out) {
  const size_t blk = blockIdx.x;
  const int u = (int)(blk / nb), b = (int)(blk % nb);
  const size_t strip = (size_t)nb * kQBlk;
  const uint8_t* src[2];
  src[0] = (w_up ? w + (size_t)u * strip : w + (size_t)(2 * u) * strip) + (size_t)b * kQBlk;
  src[1] = w_up ? w_up + (size_t)u * strip + (size_t)b * kQBlk : 2 * u + 1 < n8 ? src[0] + strip : nullptr;
  uint8_t* o = out + blk * kUnitBlk;
  {  // thread: span, lane; the word of (strip, group c): 8 nibbles k = 32 c + 8 t of the span
    const int sp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t v[4];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int m = 0; m < 2; ++m)  // in the 8-row block: unit sp / 2, lane 4 g + 2 c + t / 2, half sp % 2, word t % 2
        v[2 * c + m] = src[m] ? *reinterpret_cast<const uint32_t*>(src[m] + 512 * (sp >> 1) + 16 * (4 * g + 2 * c + (t >> 1)) + 8 * (sp & 1) + 4 * (t & 1)) : 0u;
    *reinterpret_cast<uint4*>(o + 512 * sp + 16 * lane) = make_uint4(v[0], v[1], v[2], v[3]);
  }
  {  // thread: one scale (128-k part jj, row g, group c, strip m, span q)
    const int jj = threadIdx.x >> 6, g = (threadIdx.x >> 3) & 7, c = (threadIdx.x >> 2) & 1, m = (threadIdx.x >> 1) & 1, q = threadIdx.x & 1;
    reinterpret_cast<uint16_t*>(o + 4096)[threadIdx.x] =
        src[m] ? *reinterpret_cast<const uint16_t*>(src[m] + 2048 + 32 * g + 16 * c + 2 * (2 * jj + q)) : (uint16_t)0;
  }
  if (threadIdx.x < 128) {  // thread: one byte of zero points (row g, part jj, group c, strip m): first span low, second high
    const int g = threadIdx.x >> 4, jj = (threadIdx.x >> 2) & 3, c = (threadIdx.x >> 1) & 1, m = threadIdx.x & 1;
    o[4608 + threadIdx.x] = src[m] ? src[m][2304 + 8 * g + 4 * c + jj] : (uint8_t)0;
  }
}

// Runs behind k_linear_prepare: the product requests weights before it waits for the launch in front of it, so that launch is not
// to be the one that wrote them.
__global__ void k_linear_prepared() {}

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
// 16 bytes into another CTA's shared memory, counted by that CTA's barrier (no release that would wait for the round trip)
DSGX_DEV void st_remote(uint32_t addr, float4 v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "f"(v.x),
               "f"(v.y), "f"(v.z), "f"(v.w), "r"(bar)
               : "memory");
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
DSGX_DEV float4 add4(float4 a, float4 b) {
  return make_float4(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y), __fadd_rn(a.z, b.z), __fadd_rn(a.w, b.w));
}
template <class V>
__global__ void __launch_bounds__(V::kThreads, 1) k_linear_int4(const LinearParams p) {
  constexpr int W = V::W, NP = V::NP, NST = V::NST, P = V::P, kPart = V::kPart;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int C = p.cluster;
  const uint32_t rank = C > 1 ? cluster_rank() : 0;
  // this cluster's rows (more than eight: the clusters of a pair take eight and the rest, over the same units), its units and
  // this rank's blocks of K
  const int part_m = p.M > 8 ? (int)(blockIdx.x / C) & 1 : 0, m0 = 8 * part_m, M = p.M > 8 ? (part_m ? p.M - 8 : 8) : p.M;
  const int cl = blockIdx.x / C >> (p.M > 8), ncl = gridDim.x / C >> (p.M > 8);
  const int u0 = (int)((long long)p.units * cl / ncl), u1 = (int)((long long)p.units * (cl + 1) / ncl);
  const int b0 = p.nb * (int)rank / C, nbk = p.nb * ((int)rank + 1) / C - b0;

  uint8_t* ring = smem;
  uint8_t* part = ring + (size_t)W * NST * kUnitBlk;                   // [P][32][4] f32
  uint8_t* recv = part + (size_t)P * kPart;                            // [kSlotsOwned][C][32][4] f32
  uint8_t* xt = recv + (C > 1 ? (size_t)kSlotsOwned * C * kPart : 0);  // [spans][M rows][128 B]
  const int Me = V::even(M);
  float* xsum = reinterpret_cast<float*>(xt + (size_t)p.xblocks * M * 1024);  // [spans][row pairs][2 groups][2 rows]
  float* xscale = xsum + (size_t)p.xblocks * Me * 16;                           // [blocks][rows]: 2^(12 - E)
  uint8_t* zero = smem + (((xscale + (size_t)p.xblocks * Me) - reinterpret_cast<float*>(smem)) * 4 + 127) / 128 * 128;  // kCol: 128 zeros
  uint64_t* bars = reinterpret_cast<uint64_t*>(V::kCol ? zero + 128 : reinterpret_cast<uint8_t*>(xscale + (size_t)p.xblocks * Me));
  uint64_t* freed = bars + W * NST;                                    // a stage has been read
  uint64_t* rfull = freed + W * NST;                                    // [kSlotsOwned] every rank's sums are in my buffer
  uint64_t* rfree = rfull + kSlotsOwned;                               // [owner][kSlotsOwned] that owner's buffer may be written
  int* cnt = reinterpret_cast<int*>(rfree + kMaxCluster * kSlotsOwned);  // [P] tasks summed of a unit in flight
  int* done = cnt + P;                                                 // tasks whose unit has been added up
  int* fail = done + 1;                                                // a bounded wait ran out

  if (warp < W && lane == 0)
    for (int s = 0; s < NST; ++s) mbar_init(bars + warp * NST + s, 1), mbar_init(freed + warp * NST + s, 1);
  if (threadIdx.x == W * 32) {
    for (int s = 0; s < kSlotsOwned; ++s) mbar_init(rfull + s, 1), mbar_expect_tx(rfull + s, C * kPart);
    for (int s = 0; s < kMaxCluster * kSlotsOwned; ++s) mbar_init(rfree + s, 1);
    *done = 0, *fail = 0;
  }
  for (int i = threadIdx.x; i < P; i += V::kThreads) cnt[i] = 0;
  if (V::kCol && threadIdx.x < 32) reinterpret_cast<uint32_t*>(zero)[threadIdx.x] = 0;
  mbar_fence_init();
  __syncwarp();
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  pdl_launch_dependents();

  const int lq = p.lq, Q = 1 << lq, RPT = (kRuns / C) >> lq;  // tasks a unit (this rank's part), runs a task
  const int total = (u1 - u0) << lq;                          // this CTA's tasks
  const int r0 = (int)rank * (kRuns / C);                     // this rank's first run
  const bool glu = p.glu != 0;
  // a warp's next task: one place on in every round of W tasks (blocks that do not divide by eight make every other run longer,
  // and an even number of warps would give half of them all the long ones: 6144 x 6144 and one row took 9.1 us)
  auto next_task = [&](int j, int& place) { return ++place < W ? j + W + 1 : (place = 0, j + 1); };

  if (warp > W) {
    // ---- the producers: lane l of warp W + 1 + q fills stream warp NP l + q's ring as its stages are freed.  The first weights are
    // requested before the activations are there: they do not depend on the launches before
    const int w = NP * lane + (warp - W - 1);
    uint8_t* myring = ring + (size_t)w * NST * kUnitBlk;
    uint64_t *mybar = bars + w * NST, *myfreed = freed + w * NST;
    const uint64_t pol = policy_evict_first();
    uint32_t issued = 0;
    int pj = w, place = w, pb = 0, pe = 0;  // the task and its next and last block
    const uint8_t* pa = nullptr;
    bool more = w < W, begun = false;
    long long t0 = clock64();
    for (;;) {
      while (more && pb == pe) {  // the next task with a block in it (K shorter than eight blocks: some runs are empty)
        if (pj >= total) {
          more = false;
          break;
        }
        const int u = u0 + (pj >> lq), r = r0 + (pj & (Q - 1)) * RPT;
        pb = p.nb * r / kRuns, pe = p.nb * (r + RPT) / kRuns, pj = next_task(pj, place);
        pa = p.w + ((size_t)u * p.nb + pb) * kUnitBlk;
      }
      if (!__any_sync(0xffffffffu, more)) break;
      const uint32_t slot = issued % NST;
      const bool go = more && (issued < (uint32_t)NST || mbar_test_wait(myfreed + slot, (issued / NST - 1) & 1));
      if (go) {
        mbar_expect_tx(mybar + slot, kUnitBlk);
        bulk_g2s_hint(myring + slot * kUnitBlk, pa, kUnitBlk, mybar + slot, pol);
        ++issued, ++pb, pa += kUnitBlk;
      }
      if (__any_sync(0xffffffffu, go)) {
        t0 = clock64();
      } else if (!begun) {  // the rings are full: the time that the launches in front take is not this launch's
        pdl_wait();
        begun = true, t0 = clock64();
      } else {
        if (*reinterpret_cast<volatile int*>(fail) || clock64() - t0 > kWaitCycles) break;
        __nanosleep(20);
      }
    }
    if (__any_sync(0xffffffffu, more)) {  // given up: no copy is left in flight
      *fail = 1;
      for (uint32_t n = issued > (uint32_t)NST ? issued - NST : 0; w < W && n < issued; ++n) mbar_wait(mybar + n % NST, (n / NST) & 1);
    }
  } else {
  // ---- this rank's activations ------------------------------------------------------------------------------------------
  pdl_wait();
  // tile: [span of 64 k][row][the span's 8 pieces of 8 f16], a piece = the k a lane's word covers, in the words' nibble order;
  // eight columns: odd rows with the span's two groups exchanged, so that two rows' reads of one group do not meet in the
  // banks.  The groups' sums: a row's two side by side (kCol), or two rows' of a group.
  const uint32_t span = M * 128, sspan = Me * 8;
  for (int i = warp; i < nbk * M; i += W + 1) {
    const int b = i / M, r = i - b * M;
    uint32_t w[8];
    load_16<false>(w, p.x + (size_t)(m0 + r) * p.ldx, (b0 + b) * 512 + 16 * lane, p.K, p.x_vec != 0);
    stage_row<V::kCol ? 4 : 8>(w, xt + (size_t)b * 8 * span + r * 128, span, !V::kCol && (r & 1),
                               xsum + (size_t)b * 16 * Me + (V::kCol ? 2 * r : (r >> 1) * 4 + (r & 1)), sspan, xscale + b * Me + r, lane);
  }
  asm volatile("bar.sync 1, %0;" ::"n"((W + 1) * 32) : "memory");

  if (warp < W) {
    // ---- stream warps ---------------------------------------------------------------------------------------------------
    const int g = lane >> 2, t = lane & 3;
    const uint32_t ring_at = smem_u32(ring + (size_t)warp * NST * kUnitBlk);
    uint64_t *mybar = bars + warp * NST, *myfreed = freed + warp * NST;
    // the lane's column of B is row g of x, or (kCol) row g / 2 in group g % 2; rows past M repeat the last, their sums go unused
    const int half = g & 1, r = min(V::kCol ? g >> 1 : g, M - 1), me = V::kCol ? min(t, M - 1) : min(t, Me / 2 - 1);
    const uint32_t xl = smem_u32(xt) + r * 128 + (V::kCol ? 64 * half + t * 16 : (t * 16) ^ ((r & 1) * 64));
    const uint32_t xz = V::kCol ? smem_u32(zero) + 64 * half + t * 16 : 0u;  // zeros for the other group
    const uint32_t sl = smem_u32(xsum) + me * (V::kCol ? 8 : 16), fl = smem_u32(xscale) + me * (V::kCol ? 4 : 8);
    uint32_t consumed = 0;
    bool ok = true;
    for (int j = warp, place = warp; j < total && ok; j = next_task(j, place)) {
      const int rt = r0 + (j & (Q - 1)) * RPT;
      float acc[4], lv[3][4];  // the run's sums; the subtrees that wait for their right halves
      int b = p.nb * rt / kRuns;
      for (int r = 0; r < RPT; ++r) {
        const int e = p.nb * (rt + r + 1) / kRuns;
        acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
        for (; b < e; ++b) {
          const uint32_t si = consumed % NST;
          if (!mbar_wait(mybar + si, (consumed / NST) & 1)) {
            ok = false;
            break;
          }
          const int lb = b - b0;
          const uint32_t st = ring_at + si * kUnitBlk, xb = xl + lb * 8 * span, sb = sl + lb * 8 * sspan;
          // the block's sums times 2^(24 - E), in two steps that cannot leave f32's range by themselves
          if constexpr (V::kCol) {
            float2 blk[2];
            unit_block4(blk, st, half ? xz : xb, half ? xb : xz, half ? 0 : span, half ? span : 0, sb, sspan, lane);
            const float f = lds_f(fl + lb * Me * 4);
            acc[0] = fmaf(__fadd_rn(blk[0].x, blk[0].y) * 4096.f, f, acc[0]), acc[2] = fmaf(__fadd_rn(blk[1].x, blk[1].y) * 4096.f, f, acc[2]);
          } else {
            float blk[4][2];
            unit_block8(blk, st, xb, span, sb, sspan, lane);
            const float2 f = lds_f2(fl + lb * Me * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(__fadd_rn(blk[i][0], blk[i][1]) * 4096.f, i & 1 ? f.y : f.x, acc[i]);
          }
          ++consumed;
          __syncwarp();
          if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(myfreed + si)) : "memory");
        }
        if (!ok) break;
        // run r closes as many waiting subtrees as it has trailing ones
        auto fold = [&](float (&l)[4]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = __fadd_rn(l[i], acc[i]);
        };
        auto keep = [&](float (&l)[4]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) l[i] = acc[i];
        };
        if (!(r & 1)) {
          keep(lv[0]);
        } else {
          fold(lv[0]);
          if ((r & 3) != 3) {
            keep(lv[1]);
          } else {
            fold(lv[1]);
            if (r == 7) fold(lv[2]);
            else keep(lv[2]);
          }
        }
      }
      // the sums into the partial buffer, once the unit that had the place has been added up
      if (ok) ok = wait_shared_ge(done, j - P + 1, 100);
      if (!ok) break;
      reinterpret_cast<float4*>(part + (size_t)(j & (P - 1)) * kPart)[lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      __threadfence_block();
      __syncwarp();
      if (lane == 0) atomicAdd(cnt + ((j >> lq) & (P - 1)), 1);
    }
    if (!ok) *fail = 1;
  } else {
    // ---- the adding warp ------------------------------------------------------------------------------------------------
    const int g = lane >> 2, t = lane & 3, n = u1 - u0, lc = p.lc;
    const int lag = C > 1 ? C * (kSlotsOwned / 2) : 0;  // an owner joins the ranks' sums this many units later
    float4 a;
    auto join = [&](const float4* d, int parts) {  // parts sums (1, 2, 4 or 8), as a tree
      auto two = [&](int i) { return add4(d[i * (kPart / 16)], d[(i + 1) * (kPart / 16)]); };
      if (parts == 1) a = d[0];
      else if (parts == 2) a = two(0);
      else if (parts == 4) a = add4(two(0), two(2));
      else a = add4(add4(two(0), two(2)), add4(two(4), two(6)));
    };
    auto put = [&](int m, int c, float y) {
      if (p.out_f32) reinterpret_cast<float*>(p.out)[(size_t)m * p.ldo + c] = y;
      else reinterpret_cast<__nv_bfloat16*>(p.out)[(size_t)m * p.ldo + c] = __float2bfloat16_rn(y);
    };
    auto write = [&](int unit) {
      const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int e = 0; e < (V::kCol ? 1 : 2); ++e) {
        if ((V::kCol ? t : 2 * t + e) >= M) continue;
        const int m = m0 + (V::kCol ? t : 2 * t + e);
        if (glu) {
          const int c = 8 * unit + g;
          if (c < p.N) put(m, c, __fmul_rn(silu(v[e]), v[2 + e]));
        } else {
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const int c = 16 * unit + 8 * hi + g;
            if (c < p.N) put(m, c, p.res ? __fadd_rn(v[2 * hi + e], __bfloat162float(p.res[(size_t)m * p.ldr + c])) : v[2 * hi + e]);
          }
        }
      }
    };
    bool ok = true;
    for (int i = 0; i < n + lag && ok; ++i) {
      if (i < n) {
        int* c = cnt + (i & (P - 1));
        if (!(ok = wait_shared_ge(c, Q, 40))) break;
        join(reinterpret_cast<const float4*>(part + (size_t)((i << lq) & (P - 1)) * kPart) + lane, Q);
        __syncwarp();
        if (lane == 0) {
          *c = 0;
          st_shared_release(done, (i + 1) << lq);
        }
        if (C == 1) {
          write(u0 + i);
        } else {  // to the unit's owner, once it has let go of the unit that had the buffer before
          const int owner = i & (C - 1), slot = (i >> lc) % kSlotsOwned, turn = (i >> lc) / kSlotsOwned;
          if (turn > 0 && !mbar_wait_cluster(rfree + owner * kSlotsOwned + slot, (turn - 1) & 1)) {
            ok = false;
            break;
          }
          const uint32_t bar = map_rank(smem_u32(rfull + slot), owner);
          const uint32_t to = map_rank(smem_u32(recv) + (uint32_t)((slot * C + (int)rank) * kPart + lane * 16), owner);
          st_remote(to, a, bar);
        }
      }
      const int o = i - lag;
      if (C > 1 && o >= 0 && o < n && (o & (C - 1)) == (int)rank) {
        const int slot = (o >> lc) % kSlotsOwned, turn = (o >> lc) / kSlotsOwned;
        if (!mbar_wait_cluster(rfull + slot, turn & 1)) {
          ok = false;
          break;
        }
        join(reinterpret_cast<const float4*>(recv + (size_t)slot * C * kPart) + lane, C);
        if (lane == 0) mbar_expect_tx(rfull + slot, C * kPart);  // (for the unit that takes the buffer next)
        __syncwarp();
        if (lane < C) remote_arrive(map_rank(smem_u32(rfree + rank * kSlotsOwned + slot), lane));
        write(u0 + o);
      }
    }
    if (!ok) *fail = 1;
  }
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
// clusters of C CTAs that the device runs at once, 0: none of that size (asked once per kernel, device and C; the shared memory is given
// at its most)
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
    if (cudaOccupancyMaxActiveClusters(&v, k_linear_int4<V>, &cfg) != cudaSuccess) (void)cudaGetLastError(), v = 0;
    else known[dev][C].store(v > 0 ? v : v = -1);
  }
  *n = v > 0 ? v : 0;
  return cudaSuccess;
}

// The division of a launch: a cluster size C (1, 2, 4, 8) and 14 or 11 stream warps (fewer leave more shared memory to the
// activations).  What is compared is the busiest SM's block count, ceil(units / clusters) ceil(blocks / C), where eleven warps
// stream a tenth slower and a cluster's exchange costs a quarter (12288 x 6144 pair, eight rows: 26 us with eleven warps
// alone, 31 us with more in clusters of two).
struct Division {
  long long cost = 0;
  int C = 0, clusters = 0;
};
template <class V>
cudaError_t divide(const LinearParams& p, Division* best, bool* mine) {
  const int rows = p.M > 8 ? 8 : p.M, pair = p.M > 8 ? 2 : 1;
  for (int C = 1; C <= kMaxCluster && C <= p.nb; C *= 2) {
    const int kb = (p.nb + C - 1) / C;
    if (V::smem(rows, kb, C) > kSmemMax) continue;
    int n = 0;
    cudaError_t e = resident_clusters<V>(C, &n);
    if (e != cudaSuccess) return e;
    if (n < 1) continue;  // (the other sizes still serve)
    n = n / pair > 0 ? n / pair : 1;
    const long long cost = (long long)((p.units + n - 1) / n) * kb * (V::W > 11 ? 20 : 22) * (C > 1 ? 5 : 4);
    if (!best->C || cost < best->cost) *best = Division{cost, C, n}, *mine = true;
  }
  return cudaSuccess;
}

template <class V>
cudaError_t launch(LinearParams p, const Division& d, cudaStream_t st) {
  const int C = d.C, per_cta = (p.units + d.clusters - 1) / d.clusters, rows = p.M > 8 ? 8 : p.M;
  p.cluster = C, p.lc = C == 8 ? 3 : C == 4 ? 2 : C == 2 ? 1 : 0, p.xblocks = (p.nb + C - 1) / C, p.lq = 0;
  // Tasks a unit: as few as leave every stream warp of a CTA three tasks (the last task of a launch is idle time of the
  // others), at most one a block or a run.
  while ((2 << p.lq) <= kRuns / C && (2 << p.lq) <= p.xblocks && (per_cta << p.lq) < 3 * V::W) ++p.lq;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.units < d.clusters ? p.units : d.clusters) * C * (p.M > 8 ? 2 : 1)), cfg.blockDim = dim3(V::kThreads);
  cfg.dynamicSmemBytes = V::smem(rows, p.xblocks, C), cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = C, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = C > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k_linear_int4<V>, p);
}

}  // namespace

// One launch for M rows, or *fits = false where a row's activations do not fit shared memory.
template <bool kCol>
static cudaError_t launch_rows(const LinearParams& p, cudaStream_t st, bool* fits) {
  using Wide = LinVar<kCol, 14, 1, 2, 32>;
  using Narrow = LinVar<kCol, 11, 1, 2, 32>;
  Division d;
  bool wide = false, narrow = false;
  cudaError_t e = divide<Wide>(p, &d, &wide);
  if (e == cudaSuccess) e = divide<Narrow>(p, &d, &narrow);
  *fits = d.C != 0;
  if (e != cudaSuccess || !*fits) return e;
  return narrow ? launch<Narrow>(p, d, st) : launch<Wide>(p, d, st);
}
cudaError_t launch_linear_int4(const LinearParams& p, cudaStream_t st, bool* fits) {
  return p.M <= 4 ? launch_rows<true>(p, st, fits) : launch_rows<false>(p, st, fits);
}

size_t linear_bytes(int N, int K, bool glu) {
  const size_t n8 = ((size_t)N + 7) / 8, nb = ((size_t)K + 511) / 512;
  return (glu ? n8 : (n8 + 1) / 2) * nb * kUnitBlk;
}
cudaError_t launch_linear_prepare(const uint8_t* w, const uint8_t* w_up, int N, int K, uint8_t* out, cudaStream_t st) {
  const int n8 = (N + 7) / 8, nb = (K + 511) / 512;
  const cudaError_t e = launch_k(k_linear_prepare, dim3((unsigned)((w_up ? n8 : (n8 + 1) / 2) * (long long)nb)), dim3(256), 0, st, false, w,
                                 w_up, n8, nb, out);
  return e != cudaSuccess ? e : launch_k(k_linear_prepared, dim3(1), dim3(32), 0, st, false);
}

}  // namespace dsgx
