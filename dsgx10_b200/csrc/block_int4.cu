// A whole INT4-g32 (or BF16) MoE layer for 1..8 rows in one launch: router logits, routing, the picked experts' gate / up with
// SwiGLU, down, the bf16 shared expert, the weighted sum in ascending expert id, the residual, the rounding.
//
// Bound: the weights of the distinct picked experts are read once, so HBM.  One CTA a SM, launched cooperatively (all resident
// together, so CTAs may wait for one another; every wait is bounded and a run-out is recorded in the workspace).  Of a
// CTA's warps W stream weights, each from a ring of bulk copies that three more fill for all, one joins their sums and one
// keeps track of what the other CTAs have done; whoever is free turns activations into the MMAs' operands.
//
//   front    every CTA but the last M: the router's logit slices (route.cuh's order).  The last M CTAs route a row each; the
//            last of them builds the step's table: the picked experts in ascending id with the rows that picked them.
//   shared   meanwhile the other CTAs stream the shared expert's gate and up matrices, which need no routing.
//   up       a CTA owns a run of (expert, 8 channels) units, shorter where it has streamed more of the shared expert.
//   down     the shared expert's tiles first (its h is ready early), then a run of (expert, 16 channels) units as soon as the
//            expert's h is complete; their weights are already in the rings.
//   combine  after a grid-wide count: every element adds its row's picks, the shared expert and the residual.
//
// Measured (a captured chain, more weights than L2 holds): 168 experts of 6144 x 2048, eight picks a row and the shared expert, one
// row 59.5 us (254 MB, 4.3 TB/s; four launches 76), four rows 146 us (717 MB, 4.9 TB/s; 231), eight rows 258 us (434); 1024 x 512
// and 16 experts, one row: 21 us, all of it the chain of six grid-wide steps (four launches 18).  About 16 us pass until routed
// weights stream; from then on 85 % of a copy's rate, the warps' chains of loads, MMAs and f32 operations next to HBM.
//
// Work items.  A unit (16 weight rows) is cut along K in tasks of about two 512-k blocks, dealt to the stream warps in turn
// across units and phases; a task's sums go to shared memory and the joining warp adds a unit's tasks in ascending k.  The cut
// depends on H and I alone, so a row's bits do not depend on the other rows.
//
// An INT4 block is used as the experts' format has it (decode_int4.cu).  Its lanes mix two groups of 32 in every MMA (lane 4 g +
// t holds k = 64 q + 16 t + 0..15 of row g: lanes t = 0, 1 one group, t = 2, 3 the next), so the eight columns of B are (row of
// x, half) pairs: column 2 r + h holds row r's values in the lanes of half h and zeros in the others, lane (g, t) ends with
// both groups' sums of row t and two packed multiply-adds finish 64 k (scale, zero point: int4_mma.cuh).  Four rows of x a
// set of MMAs; an expert that more rows picked takes two sets.  Only the rows that picked an expert are computed for it.
//
// Gate, up and the down sums stay f32, and so does h until it is an MMA operand: f16 with a power of two a 512-k block, as the INT4
// products take x (eleven bits, at most 2^-11 of the value; h in bf16 made the layer's error against 64 bits 0.0021 of its
// outputs instead of 0.0017, which the outputs' own rounding is, and took 145.1 us for four rows of 168 experts instead of 146.1,
// 253 for eight instead of 258).  A bf16 matrix meets it as two bf16 parts whose sum it is (pair_b16).
#include <atomic>
#include <cstddef>
#include <type_traits>

#include "common.cuh"
#include "decode_common.cuh"
#include "int4_mma.cuh"
#include "kernels.h"
#include "route.cuh"

namespace dsgx {

constexpr int kMaxEnt = kMaxRows * kMaxTopK;

// A picked expert: its matrices, the rows that picked it (n of them, ascending, a byte each).
struct alignas(16) BlockEnt {
  const uint8_t *g, *u, *d;
  unsigned long long rows;
  int n;
  int pad[3];
};
struct alignas(16) BlockTab {
  int nslots, npick, pad[2];
  int pick[kMaxRows][kMaxTopK];   // a row's picks in ascending expert id: slot | its place among the slot's rows << 8
  float w[kMaxRows][kMaxTopK];
  BlockEnt ent[kMaxEnt];          // (last: only as many as the step can have picked are read)
};
static_assert(sizeof(BlockEnt) == 48 && sizeof(BlockTab) % 16 == 0, "copied in 16-byte pieces");

struct BlockSync {
  int cnt_lp, cnt_rt, tab_ready, cnt_done, cnt_exit, pad[3];
  int cnt_h[kMaxEnt + 1];  // gate/up units of a slot that are in memory
};

namespace {

constexpr int kStage = 2 * kQBlk;        // a ring stage: an INT4 block pair (a pair of bf16 blocks, 4096 B, fits)
constexpr int kFront = 300 * 1024;       // bytes an SM streams from the end of the logits until the table is known (7 us)
constexpr int kP = 16;                   // tasks' sums in flight
constexpr int kPart = 512;               // bytes of a task's sums: [2 sets][32 lanes][2] f32
constexpr int kShared = kMaxEnt;         // the shared expert's place among the h, y and counters
constexpr int kMaxSegs = kMaxEnt + 4;
constexpr size_t kSmemMax = 227 * 1024;

// Signals to other CTAs: releases of what this thread has written or has seen written behind a barrier of its CTA or warp.
DSGX_DEV void red_release(int* p, int v) { asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory"); }
DSGX_DEV void st_release(int* p, int v) { asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory"); }
DSGX_DEV int atom_add_acq_rel(int* p, int v) {
  int o;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(o) : "l"(p), "r"(v) : "memory");
  return o;
}
DSGX_DEV void arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
// mbar_wait without the suspended try: the joining warp's wake-up is on every unit's path
DSGX_DEV bool mbar_spin(uint64_t* bar, uint32_t parity) {
  if (mbar_test_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_test_wait(bar, parity))
    if (clock64() - t0 > kWaitCycles) return false;
  return true;
}
// bounded poll until *p >= target (decode_common.cuh's poll_ge with a shorter sleep: these waits are on the critical path)
DSGX_DEV bool poll_near(const int* p, int target) {
  if (ld_acquire(p) >= target) return true;
  const long long t0 = clock64();
  while (ld_acquire(p) < target) {
    __nanosleep(32);
    if (clock64() - t0 > kWaitCycles) return false;
  }
  return true;
}

// g / (1 + e^-g) by the fast exponential and division: within 100 x 2^-23 = 2^-16.3 of the value for |g| up to 80, and h's rounding to
// eleven bits, 2^-11, comes next (expf and an IEEE division in the joining warp: 168 experts, four rows 146.3 -> 147.2 us)
DSGX_DEV float quick_silu(float g) { return __fdividef(g, 1.f + __expf(-g)); }

// A CTA's run of units of one phase.
struct Seg {
  int down, b16, slot, rows;  // slot: of a down run (an up run covers several); rows: of the activation tile
  int u0, n;                  // units; an up run's unit u: slot u / (I / 8)
  int tasks, base;            // tasks of the run; tasks before it
};

DSGX_DEV int tasks_of(int nb) { return nb <= 1 ? 1 : nb / 2 < 8 ? nb / 2 : 8; }  // tasks a unit

// ---- the tile of activations: [nb x 8 spans][rows][128 B], then group sums [spans][rows][2], then scales [nb][rows]
__host__ __device__ inline size_t tile_bytes(int K, int rows) { return ((size_t)K / 512 * rows * (1024 + 64 + 4) + 127) & ~(size_t)127; }
struct Tile {
  uint8_t* x;
  float *sum, *scale;
  DSGX_DEV Tile(uint8_t* base, int nb, int rows) : x(base), sum(reinterpret_cast<float*>(base + (size_t)nb * rows * 1024)), scale(sum + (size_t)nb * rows * 16) {}
};

// One INT4 block pair: acc[s][strip] += (.x, .y: the two halves of the groups) row g of strip a / b times the lane's row t of set s,
// times 2^(E - 24).
template <int S>
DSGX_DEV void pair_int4(float2 (&acc)[S][2], uint32_t st, const uint32_t (&x_at)[S], const uint32_t (&step)[S], const uint32_t (&sum_at)[S],
                        uint32_t sstep, int lane) {
  const int g = lane >> 2;
  const uint2 za = lds_v2(st + 2304 + 8 * g), zb = lds_v2(st + kQBlk + 2304 + 8 * g);  // the halves' eight zero points each
  const uint4 sa0 = lds_v4(st + 2048 + 32 * g), sa1 = lds_v4(st + 2048 + 32 * g + 16);
  const uint4 sb0 = lds_v4(st + kQBlk + 2048 + 32 * g), sb1 = lds_v4(st + kQBlk + 2048 + 32 * g + 16);
  const uint32_t *a0 = &sa0.x, *a1 = &sa1.x, *b0 = &sb0.x, *b1 = &sb1.x;
  uint32_t x[S], sm[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    x[s] = x_at[s], sm[s] = sum_at[s];
    acc[s][0] = acc[s][1] = make_float2(0.f, 0.f);
  }
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    const uint4 va = lds_v4(st + 512 * jj + 16 * lane), vb = lds_v4(st + kQBlk + 512 * jj + 16 * lane);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t al = q ? va.z : va.x, ah = q ? va.w : va.y, bl = q ? vb.z : vb.x, bh = q ? vb.w : vb.y;
      const uint32_t al8 = al >> 8, ah8 = ah >> 8, bl8 = bl >> 8, bh8 = bh >> 8;
      const float2 mza = make_float2(minus_zero(q ? za.x >> 4 & 0x0F0F0F0Fu : za.x & 0x0F0F0F0Fu, jj), minus_zero(q ? za.y >> 4 & 0x0F0F0F0Fu : za.y & 0x0F0F0F0Fu, jj));
      const float2 mzb = make_float2(minus_zero(q ? zb.x >> 4 & 0x0F0F0F0Fu : zb.x & 0x0F0F0F0Fu, jj), minus_zero(q ? zb.y >> 4 & 0x0F0F0F0Fu : zb.y & 0x0F0F0F0Fu, jj));
      const float2 fa = q ? make_float2(scale_hi(a0[jj]), scale_hi(a1[jj])) : make_float2(scale_lo(a0[jj]), scale_lo(a1[jj]));
      const float2 fb = q ? make_float2(scale_hi(b0[jj]), scale_hi(b1[jj])) : make_float2(scale_lo(b0[jj]), scale_lo(b1[jj]));
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint4 x0 = lds_v4(x[s]), x1 = lds_v4(x[s] + 16);
        const float2 sum = lds_f2(sm[s]);
        x[s] += step[s], sm[s] += sstep;
        float d[4];
        mma_f16_zero(d, al & kNib0, bl & kNib0, al & kNib1, bl & kNib1, x0.x, x0.y);
        mma_f16(d, al8 & kNib0, bl8 & kNib0, al8 & kNib1, bl8 & kNib1, x0.z, x0.w);
        mma_f16(d, ah & kNib0, bh & kNib0, ah & kNib1, bh & kNib1, x1.x, x1.y);
        mma_f16(d, ah8 & kNib0, bh8 & kNib0, ah8 & kNib1, bh8 & kNib1, x1.z, x1.w);
        acc[s][0] = fma2(fa, fma2(mza, sum, make_float2(d[0], d[1])), acc[s][0]);
        acc[s][1] = fma2(fb, fma2(mzb, sum, make_float2(d[2], d[3])), acc[s][1]);
      }
    }
  }
}

// Two f16 values as two bf16 parts each, hi + lo = the value (eight bits and the three or fewer left)
DSGX_DEV void split_f16(uint32_t& hi, uint32_t& lo, uint32_t w) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(v.y), "f"(v.x));
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(__fadd_rn(v.y, -scale_hi(hi))), "f"(__fadd_rn(v.x, -scale_lo(hi))));
}
// a lane's 16 bytes of two strips with 16 bytes of the tile (both in nibble order's pairs)
DSGX_DEV void mma_b16_words(float (&d)[4], const uint4& a, const uint4& b, const uint4& x) {
  mma_bf16(d, __byte_perm(a.x, a.z, 0x5410), __byte_perm(b.x, b.z, 0x5410), __byte_perm(a.x, a.z, 0x7632), __byte_perm(b.x, b.z, 0x7632), x.x, x.y);
  mma_bf16(d, __byte_perm(a.y, a.w, 0x5410), __byte_perm(b.y, b.w, 0x5410), __byte_perm(a.y, a.w, 0x7632), __byte_perm(b.y, b.w, 0x7632), x.z, x.w);
}
// One bf16 block pair (128 k) on a bf16 tile, or (f16) on an f16 one with two MMAs for one (twice the tile, split beforehand, would
// leave no room for its rows): all eight columns are rows of x (column n: row n / 2 + 4 (n & 1), so that a lane ends with rows t
// and t + 4).  used(): the stage has been read, before its last products, so that the split keeps no copy waiting (32 BF16 experts of
// 6144 x 2048, four rows: 264 us instead of 268, eight 354 instead of 360; 257 and 343 with h in bf16).
template <class F>
DSGX_DEV void pair_b16(float (&d)[4], uint32_t st, uint32_t x, uint32_t span, bool f16, int lane, F used) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t a = st + 1024 * q + 16 * lane;
    const uint4 a0 = lds_v4(a), a1 = lds_v4(a + 512), b0 = lds_v4(a + kQBlk), b1 = lds_v4(a + kQBlk + 512);
    if (q) used();
    uint4 x0 = lds_v4(x), x1 = lds_v4(x + 16);
    x += span;
    if (f16) {
      uint4 lo;
      split_f16(x0.x, lo.x, x0.x), split_f16(x0.y, lo.y, x0.y), split_f16(x0.z, lo.z, x0.z), split_f16(x0.w, lo.w, x0.w);
      mma_b16_words(d, a0, b0, lo);
      split_f16(x1.x, lo.x, x1.x), split_f16(x1.y, lo.y, x1.y), split_f16(x1.z, lo.z, x1.z), split_f16(x1.w, lo.w, x1.w);
      mma_b16_words(d, a1, b1, lo);
    }
    mma_b16_words(d, a0, b0, x0);
    mma_b16_words(d, a1, b1, x1);
  }
}

// ---- the division of a phase's units over the CTAs.  n shared units of cost cs over the first Gs CTAs, then N routed ones of cost c
// so that all G CTAs end alike; none begins its routed units before a time worth `front` has passed.  N is known with the table
// only, and every CTA waits for its bounds then: everything else is worked out before, one multiplication and a correction are left.
DSGX_DEV int shared_begin(int i, int n, int Gs) { return (int)((unsigned)(n * min(i, Gs)) / (unsigned)Gs); }
struct Deal {
  int i, G, c, many;
  long long used, rest, D;  // used: G times the cost of what CTAs before i do otherwise; rest: of all; D = c G
  double inv;
  DSGX_DEV Deal(int i_, int c_, int n, int cs, int Gs, int G_, int front) : i(i_), G(G_), c(c_) {
    const int a = n / Gs, few = max(cs * a, front), all_extra = n - a * Gs;  // a CTA has a or a + 1 shared units
    const int extra = shared_begin(i, n, Gs) - a * min(i, Gs);
    many = max(cs * (a + 1), front);
    used = ((long long)few * (i - extra) + (long long)many * extra - (i > Gs ? (long long)(few - front) * (i - Gs) : 0)) * G;
    rest = (long long)few * (G - all_extra) + (long long)many * all_extra - (long long)(few - front) * (G - Gs);
    D = (long long)c * G, inv = 1. / (double)D;
  }
  // where CTA i's run begins
  DSGX_DEV int begin(int N) const {
    if (i <= 0) return 0;
    if (i >= G) return N;
    const long long total = (long long)N * c + rest;
    const bool even = total < (long long)G * 2 * many;  // (few routed units: an even deal)
    const long long num = even ? (long long)N * i * c : total * i - used;
    if (num <= 0) return 0;
    long long q = (long long)((double)num * inv);  // floor(num / D): off by at most one
    const long long r = num - q * D;
    q += r < 0 ? -1 : r >= D ? 1 : 0;
    return (int)min((long long)N, q);
  }
};

// One (expert, 1024 k) slice of the router logits for rows [m0, m1): decode_common.cuh's logit_slice_task, sum for sum, with two
// rows' loads in flight (row after row, eight rows took 7 us).
DSGX_DEV void logit_rows(const __nv_bfloat16* __restrict__ x, const float* __restrict__ wr, int m0, int m1, int H, int E, int e, int sl,
                         float* __restrict__ lpart, int lane) {
  float4 wv[8];
  logit_slice_weights(wr, H, e, sl, lane, wv);
  const int base = sl * 1024, nit = min(1024, H - base) / 128;
  for (int m = m0; m < m1; m += 2) {
    uint2 xv[2][8];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        xv[c][i] = i < nit && m + c < m1 ? __ldg(reinterpret_cast<const uint2*>(x + (size_t)(m + c) * H + base + 128 * i + 4 * lane)) : make_uint2(0, 0);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < nit) {
          a = fmaf(bf16_bits_to_f(xv[c][i].x & 0xffffu), wv[i].x, a), a = fmaf(bf16_bits_to_f(xv[c][i].x >> 16), wv[i].y, a);
          a = fmaf(bf16_bits_to_f(xv[c][i].y & 0xffffu), wv[i].z, a), a = fmaf(bf16_bits_to_f(xv[c][i].y >> 16), wv[i].w, a);
        }
      a = warp_sum(a);
      if (lane == 0 && m + c < m1) lpart[((size_t)sl * kMaxRows + m + c) * E + e] = a;
    }
  }
}

// ---- the table, by the first 64 threads of a CTA, a thread a pick, written straight to global memory.  An expert's picks and the
// experts picked are bit masks in shared memory (zero at the start), so that a slot is a count of bits.
struct alignas(16) TabSmem {
  uint32_t of[512][2];  // the picks of an expert
  uint32_t any[16];     // the experts that were picked
  int idx[kMaxEnt];
  int bad;
  int pick[kMaxTopK];   // one row's picks and weights, from the routing
  float w[kMaxTopK];
};
static_assert(sizeof(TabSmem) <= kP * kPart, "in the place of the tasks' sums");
DSGX_DEV void build_block_tab(BlockTab* out, TabSmem& sm, const BlockParams& p) {
  constexpr int kNone = 0x7fffffff;
  const int i = threadIdx.x, np = p.M * p.topk;
  const bool in = i < np;
  int e = in ? (p.M == 1 ? sm.pick[i] : __ldcg(p.idx + i)) : kNone;
  const float w = in ? (p.M == 1 ? sm.w[i] : __ldcg(p.w + i)) : 0.f;
  const bool bad_id = in && (e < 0 || e >= p.E);
  if (bad_id) e = kNone;
  uint4 d[3];  // off, s2, fmt of the expert's three descriptors
  if (e != kNone) {
#pragma unroll
    for (int m = 0; m < 3; ++m) d[m] = __ldg(reinterpret_cast<const uint4*>(p.desc + (size_t)e * 3 + m));
    atomicOr(&sm.of[e][i >> 5], 1u << (i & 31));
    atomicOr(&sm.any[e >> 5], 1u << (e & 31));
  }
  sm.idx[i] = e;
  asm volatile("bar.sync 3, 64;" ::: "memory");
  // (rolled loops: this code runs once a launch, its instructions come from memory)
  int upto = (i & 31) < 16 ? __popc(sm.any[i & 15]) : 0;  // distinct experts up to the lane's word
  const int own = upto;
#pragma unroll 1
  for (int o = 1; o < 16; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if ((i & 31) >= o) upto += v;
  }
  const int n = __shfl_sync(0xffffffffu, upto, 15);
  int slot = __shfl_sync(0xffffffffu, upto - own, e >> 5 & 15);
  unsigned long long of = 0;
  if (e != kNone) slot += __popc(sm.any[e >> 5] & ((1u << (e & 31)) - 1u)), of = *reinterpret_cast<const unsigned long long*>(sm.of[e]);
  const bool first = e != kNone && __ffsll((long long)of) - 1 == i;
  uint32_t mask = 0;  // the rows that picked the expert
  const uint32_t picks = (1u << p.topk) - 1u;
#pragma unroll 1
  for (int r = 0; r < p.M; ++r, of >>= p.topk)
    if ((uint32_t)of & picks) mask |= 1u << r;
  const int row = in ? i / p.topk : 0;
  int place = 0;  // the pick's place in its row's ascending order
#pragma unroll 1
  for (int j = 0; j < p.topk; ++j) place += sm.idx[row * p.topk + j] < e;
  int bad = bad_id ? DSGX_ERR_ARG : 0;
  if (first) {
    if (d[0].w != p.fmt || d[1].w != p.fmt || d[2].w != p.fmt || ((d[0].x | d[1].x | d[2].x) & 255)) bad = DSGX_ERR_FORMAT;  // (bulk copies fault)
    BlockEnt en;
    en.g = p.pool + ((uint64_t)d[0].x | (uint64_t)d[0].y << 32), en.u = p.pool + ((uint64_t)d[1].x | (uint64_t)d[1].y << 32);
    en.d = p.pool + ((uint64_t)d[2].x | (uint64_t)d[2].y << 32);
    en.rows = 0, en.n = 0, en.pad[0] = en.pad[1] = en.pad[2] = 0;
#pragma unroll 1
    for (uint32_t left = mask; left; left &= left - 1) en.rows |= (unsigned long long)(__ffs((int)left) - 1) << (8 * en.n++);
    out->ent[slot] = en;
  }
  if (in) {
    out->pick[row][place] = slot | __popc(mask & ((1u << row) - 1u)) << 8;
    out->w[row][place] = w;
  }
  bad = (int)__reduce_max_sync(0xffffffffu, (unsigned)bad);
  if (i == 32) sm.bad = bad;
  asm volatile("bar.sync 3, 64;" ::: "memory");
  if (i == 0) {
    bad = max(bad, sm.bad);
    if (bad) atomicCAS(p.status, 0, bad);
    out->nslots = bad ? 0 : n, out->npick = bad ? 0 : p.topk;
    st_release(&p.sync->tab_ready, 1);
  }
}

// W stream warps with NST ring stages each, the joining warp, the control warp and NP producers, sixteen together (the routing
// wants a thread an expert).  S: sets of four rows that the code has room for.
template <int S_, int W_, int NST_, int NP_>
struct BlkVar {
  static constexpr int S = S_, W = W_, NST = NST_, NP = NP_, kThreads = 512;
  // W <= kP: a warp at task j has written j - W, so the unit of j - W - kP, and with it that of j - 2 kP, is joined: the parity waits
  // on a place never meet one that is two uses behind
  static_assert(W + 2 + NP == 16 && W <= kP, "warps");
};

template <class V>
__global__ void __launch_bounds__(V::kThreads, 1) k_block(const BlockParams p) {
  constexpr int kStreamW = V::W, NST = V::NST, S = V::S, kThreads = V::kThreads, kLogitW = kStreamW + 1;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = gridDim.x, cta = blockIdx.x;
  const int nbH = p.H / 512, nbI = p.I / 512, upp = p.I / 8, NT = p.H / 16, QH = tasks_of(nbH), QI = tasks_of(nbI);
  uint8_t* ring = smem;
  uint8_t* part = ring + (size_t)kStreamW * NST * kStage;
  BlockTab& tab = *reinterpret_cast<BlockTab*>(part + kP * kPart);
  uint8_t* tiles = reinterpret_cast<uint8_t*>(&tab + 1);  // [nbuf] activation tiles
  uint8_t* zero = tiles + (size_t)p.nbuf * p.tile + 16;   // 32 bytes, off the banks that the tile's lines use
  uint64_t* bars = reinterpret_cast<uint64_t*>(zero + 48);
  uint64_t* freed = bars + kStreamW * NST;                // [kStreamW][NST] a stage has been used
  uint64_t* seg_open = freed + kStreamW * NST;             // [kMaxSegs] the segment's activations exist and their tile is free
  uint64_t* tile_full = seg_open + kMaxSegs;              // [kMaxSegs] they are in the tile (an arrival a row and block)
  uint64_t* tile_free = tile_full + kMaxSegs;             // [kMaxSegs] no stream warp reads them any more
  uint64_t* tabbar = tile_free + kMaxSegs;                // the table and all segments are known
  uint64_t* full = tabbar + 2;                            // [kP] a task's sums are in their place
  uint64_t* emptied = full + kP;                          // [kP] its unit has been joined
  Seg* segs = reinterpret_cast<Seg*>(emptied + kP);
  int* first_blk = reinterpret_cast<int*>(segs + kMaxSegs);  // [2][12] a task's first block, of K = H and of K = I
  int* claim = first_blk + 24;                            // [kMaxSegs] rows and blocks that a warp has taken on
  int* s_nseg = claim + kMaxSegs;
  int* s_fail = s_nseg + 1;
  int* s_tick = s_nseg + 2;
  BlockSync* sy = p.sync;

  if (warp < kStreamW && lane == 0)
    for (int s = 0; s < NST; ++s) mbar_init(bars + warp * NST + s, 1), mbar_init(freed + warp * NST + s, 1);
  for (int i = threadIdx.x; i < kMaxSegs; i += kThreads) mbar_init(seg_open + i, 1), mbar_init(tile_free + i, kStreamW), claim[i] = 0;
  if (threadIdx.x < kP) mbar_init(full + threadIdx.x, 1), mbar_init(emptied + threadIdx.x, 1);
  if (threadIdx.x < 8) reinterpret_cast<uint32_t*>(zero)[threadIdx.x] = 0;
  if (threadIdx.x <= 8) first_blk[threadIdx.x] = nbH * (int)threadIdx.x / QH, first_blk[12 + threadIdx.x] = nbI * (int)threadIdx.x / QI;

  const bool has_sh = p.sh_d != nullptr;
  const int Gs = G - p.M;  // the CTAs that do not route
  const bool router = cta >= Gs;
  // the run that needs no routing: the shared expert's gate and up
  const int a0 = has_sh && !router ? shared_begin(cta, upp, Gs) : 0, a1 = has_sh && !router ? shared_begin(cta + 1, upp, Gs) : 0;
  if (router) {  // (build_block_tab)
    TabSmem& ts = *reinterpret_cast<TabSmem*>(part);
    ts.of[threadIdx.x][0] = ts.of[threadIdx.x][1] = 0u;
    if (threadIdx.x < 16) ts.any[threadIdx.x] = 0u;
  }
  if (threadIdx.x == 0) {
    mbar_init(tabbar, 1);
    *s_nseg = 0, *s_fail = 0;
    segs[0] = Seg{0, 1, kShared, p.M, a0, a1 - a0, (a1 - a0) * QH, 0};
    mbar_init(tile_full, p.M * nbH);
    if (a1 > a0) mbar_init(tile_full + 1, p.M * nbH);  // (the down segments' are set when they are known, each once)
  }
  mbar_fence_init();
  __syncthreads();

  // ---- a stream warp's way through the tasks of a segment, without divisions (W tasks on: some units and a part of one)
  const int duH = kStreamW / QH, dqH = kStreamW % QH, duI = kStreamW / QI, dqI = kStreamW % QI;
  struct Cursor {
    int i, u, q, slot;  // task, unit (of the slot, in an up run of the routed experts), task of the unit
  };
  auto enter = [&](Cursor& c, const Seg& s, int w) {
    const int Q = s.down ? QI : QH;
    c.i = (int)((unsigned)(w + kStreamW - s.base % kStreamW) % kStreamW);
    c.u = s.u0 + c.i / Q, c.q = c.i % Q, c.slot = s.slot;
    if (!s.down && s.slot != kShared) c.slot = c.u / upp, c.u -= c.slot * upp;
  };
  auto next = [&](Cursor& c, const Seg& s) {
    c.i += kStreamW, c.u += s.down ? duI : duH, c.q += s.down ? dqI : dqH;
    const int Q = s.down ? QI : QH;
    if (c.q >= Q) c.q -= Q, ++c.u;
    if (!s.down && s.slot != kShared)
      while (c.u >= upp) c.u -= upp, ++c.slot;
  };
  const int nb_first = a1 > a0 ? 1 : 0;  // segments whose units are known without the table

  // ---- a segment's activation tile: the shared expert's x, the routed experts' x, then the down segments in the first tile's place
  auto tile_at = [&](int k) { return tiles + (k <= nb_first ? (k == nb_first ? (p.nbuf - 1) * p.tile : 0) : (k - nb_first - 1) % p.nbuf_down * p.tile_down); };
  // every warp that waits for a segment takes on some of its rows and blocks first
  auto prepare = [&](int k, bool b16, int down, int slot, int rows) {
    if (!mbar_wait(seg_open + k, 0, 20)) return false;
    const int nb = down ? nbI : nbH, K = down ? p.I : p.H, items = nb * rows;
    const Tile tile(tile_at(k), nb, rows);
    const uint32_t span = rows * 128;
    for (;;) {
      int i = 0;
      if (lane == 0) i = atomicAdd(claim + k, 1);
      i = __shfl_sync(0xffffffffu, i, 0);
      if (i >= items) return true;
      const int b = i / rows, r = i - b * rows;
      uint8_t* xt = tile.x + (size_t)b * 8 * span + r * 128;
      uint32_t w[8];
      if (!down) load_16<true>(w, p.x + (size_t)r * K, b * 512 + 16 * lane, K, true);
      if (down) {
        const float4* src = reinterpret_cast<const float4*>(p.h + ((size_t)slot * kMaxRows + r) * K + b * 512 + 16 * lane);
        float2 v[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 u = __ldcg(src + c);
          v[2 * c] = make_float2(u.x, u.y), v[2 * c + 1] = make_float2(u.z, u.w);
        }
        stage_row_f32(v, !b16, xt, span, tile.sum + (size_t)b * 16 * rows + 2 * r, rows * 8, tile.scale + b * rows + r, lane);
      } else if (b16) {
        uint4 o[2];
        nibble_order(o, w);
        uint4* d = reinterpret_cast<uint4*>(xt + (size_t)(lane >> 2) * span + (lane & 3) * 32);
        d[0] = o[0], d[1] = o[1];
      } else {
        stage_row<4>(w, xt, span, false, tile.sum + (size_t)b * 16 * rows + 2 * r, rows * 8, tile.scale + b * rows + r, lane);
      }
      __threadfence_block();
      __syncwarp();
      if (lane == 0) arrive(tile_full + k);
    }
  };

  if (router) {
    // ---- a row each; the last one to be routed builds the table -------------------------------------------------------------
    RouteSmem& rs = *reinterpret_cast<RouteSmem*>(ring);  // (nothing is streamed yet)
    TabSmem& ts = *reinterpret_cast<TabSmem*>(part);
    const int row = cta - Gs, KS = (p.H + 1023) / 1024, nt = (p.E + 31) & ~31, ng = max(nt, 64);
    auto sync = [&]() { asm volatile("bar.sync 4, %0;" ::"r"(ng) : "memory"); };
    if (threadIdx.x == 0) arrive(seg_open);
    if ((int)threadIdx.x >= ng) {  // (the routed experts' x meanwhile; after the routing, these CTAs began to stream 5 us late)
      prepare(0, p.b16, 0, 0, p.M);
    } else {
      for (int i = threadIdx.x; i < p.E * 3; i += ng) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.desc + i));
      if (threadIdx.x == 0) *s_tick = poll_near(&sy->cnt_lp, Gs) ? 1 : 0;
      sync();
      const bool ok = *s_tick != 0;
      sync();
      if (ok) {
        if ((int)threadIdx.x < nt)
          route_row_cta(p.rp, p.lpart + (size_t)row * p.E, KS, (size_t)kMaxRows * p.E, p.bias, rs, nullptr, p.idx + row * p.topk,
                        p.w + row * p.topk, p.M == 1 ? ts.pick : nullptr, ts.w, CtaPart{nt, 2});
        if (warp == 0) {  // (warp 0 wrote the picks)
          __syncwarp();
          if (lane == 0) *s_tick = p.M > 1 ? atom_add_acq_rel(&sy->cnt_rt, 1) : 0;
        }
        sync();
        if (*s_tick == p.M - 1 && threadIdx.x < 64) build_block_tab(p.tab, ts, p);
      } else if (threadIdx.x == 0) {
        *s_fail = 1;
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (bulk copies write the routing's scratch next)
    __syncthreads();
  } else if (warp < kLogitW) {
    // ---- the router's logit slices, one warp a (expert, 1024 k); a CTA reports when all of its are in memory.  (The rings
    // filled first: 2.4 us later logits and not a microsecond gained on the shared expert.) ------------------------------------
    const int KS = (p.H + 1023) / 1024, ntask = p.E * KS;
    // (more warps than slices: a slice's rows over several warps)
    const int parts = min(p.M, max(1, kLogitW * Gs / ntask)), per = (p.M + parts - 1) / parts;
    for (int i = warp * Gs + cta; i < ntask * parts; i += kLogitW * Gs) {
      const int slice = i / parts, m = (i - slice * parts) * per;
      logit_rows(p.x, p.wr, m, min(p.M, m + per), p.H, p.E, slice / KS, slice % KS, p.lpart, lane);
    }
    asm volatile("bar.sync 1, %0;" ::"n"((kLogitW + V::NP) * 32) : "memory");
    if (threadIdx.x == 0) red_release(&sy->cnt_lp, 1);
  } else if (warp > kStreamW + 1) {
    asm volatile("bar.sync 1, %0;" ::"n"((kLogitW + V::NP) * 32) : "memory");  // (the producers begin when the logits are done)
  }

  if (warp < kStreamW) {
    // ---- stream warps --------------------------------------------------------------------------------------------------------
    const uint32_t ring_at = smem_u32(ring + (size_t)warp * NST * kStage);
    uint64_t *mybar = bars + warp * NST, *myfreed = freed + warp * NST;
    uint32_t consumed = 0;
    bool ok = true;
    auto stage_ready = [&]() {
      const uint32_t si = consumed % NST;
      if (!mbar_wait(mybar + si, (consumed / NST) & 1)) ok = false;
      return ring_at + si * kStage;
    };
    auto stage_used = [&]() {
      __syncwarp();
      if (lane == 0) arrive(myfreed + consumed % NST);
      ++consumed;
    };

    for (int k = 0; ok; ++k) {
      if (k <= nb_first && !prepare(k, k < nb_first || p.b16, 0, 0, p.M)) {  // (x needs no table)
        ok = false;
        break;
      }
      if (k >= nb_first) {  // (the units do, from here on)
        if (k == nb_first && !mbar_wait(tabbar, 0, 20)) ok = false;
        if (!ok || *s_fail || k >= *s_nseg) break;
      }
      const Seg s = segs[k];
      if ((k > nb_first && !prepare(k, s.b16, 1, s.slot, s.rows)) || !mbar_wait(tile_full + k, 0, 20)) {
        ok = false;
        break;
      }
      const int Q = s.down ? QI : QH, nb = s.down ? nbI : nbH;
      const Tile tile(tile_at(k), nb, s.rows);
      const uint32_t span = s.rows * 128, x0 = smem_u32(tile.x), z0 = smem_u32(zero);
      Cursor c;
      enter(c, s, warp);
      // where this lane finds the slot's rows: set e's column in the tile (zeros: step 0), its row's sums and scales
      int slot = -1, n = s.rows;
      uint32_t xr[S], step[S], sr[S], fr[S];
      auto rows_of = [&](unsigned long long rows) {
        auto row = [&](int j) { return (int)(rows >> (8 * min(j, n - 1)) & 0xff); };
        if (s.b16) {
          xr[0] = x0 + row((g >> 1) + 4 * (g & 1)) * 128 + t * 32;
#pragma unroll
          for (int e = 0; e < S; ++e) fr[e] = smem_u32(tile.scale) + row(4 * e + t) * 4;
          return;
        }
#pragma unroll
        for (int e = 0; e < S; ++e) {
          const int col = 4 * e + (g >> 1), me = row(4 * e + t);
          const bool on = (t >> 1) == (g & 1) && col < n;
          xr[e] = on ? x0 + row(col) * 128 + t * 32 : z0, step[e] = on ? span : 0u;
          sr[e] = smem_u32(tile.sum) + me * 8, fr[e] = smem_u32(tile.scale) + me * 4;
        }
      };
      if constexpr (S > 1) rows_of(0x0706050403020100ull);
      for (; c.i < s.tasks && ok; next(c, s)) {
        // an up run's expert: only the rows that picked it (with one set, one call of rows_of for all: a row of 168 experts 59.8 ->
        // 58.9 us; with two, 2 % slower)
        if constexpr (S > 1) {
          if (!s.down && s.slot != kShared && c.slot != slot) slot = c.slot, n = tab.ent[slot].n, rows_of(tab.ent[slot].rows);
        } else if (c.slot != slot) {
          slot = c.slot;
          const bool some = !s.down && slot != kShared;
          if (some) n = tab.ent[slot].n;
          rows_of(some ? tab.ent[slot].rows : 0x0706050403020100ull);
        }
        const int* fb = first_blk + (s.down ? 12 : 0) + c.q;
        const int b0 = fb[0], b1 = fb[1];
        float acc[S][2];  // [rows t, t + 4][strip]
#pragma unroll
        for (int e = 0; e < S; ++e) acc[e][0] = acc[e][1] = 0.f;
        if (s.b16) {
          for (int b = b0; b < b1 && ok; ++b) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            for (int q = 0; q < 4; ++q) {
              const uint32_t st = stage_ready();
              if (!ok) break;
              pair_b16(d, st, xr[0] + (8 * b + 2 * q) * span, span, s.down, lane, stage_used);
            }
#pragma unroll
            for (int e = 0; e < S; ++e) {
              const float f = s.down ? lds_f(fr[e] + b * (s.rows * 4)) * 0x1p-12f : 1.f;  // (h: times 2^-E)
              acc[e][0] = fmaf(d[e], f, acc[e][0]), acc[e][1] = fmaf(d[2 + e], f, acc[e][1]);
            }
          }
        } else {
          auto run = [&](auto sets) {
            constexpr int N = decltype(sets)::value;
            for (int b = b0; b < b1; ++b) {
              uint32_t xb[N], st_[N], sb[N];
              float f[N];
#pragma unroll
              for (int e = 0; e < N; ++e) {
                xb[e] = xr[e] + b * 8 * step[e], st_[e] = step[e], sb[e] = sr[e] + b * (s.rows * 64);
                f[e] = lds_f(fr[e] + b * (s.rows * 4));
              }
              const uint32_t st = stage_ready();
              if (!ok) break;
              float2 blk[N][2];
              pair_int4<N>(blk, st, xb, st_, sb, s.rows * 8, lane);
              stage_used();
#pragma unroll
              for (int e = 0; e < N; ++e) {  // times 2^(24 - E), in two steps that cannot leave f32's range by themselves
                acc[e][0] = fmaf(__fadd_rn(blk[e][0].x, blk[e][0].y) * 4096.f, f[e], acc[e][0]);
                acc[e][1] = fmaf(__fadd_rn(blk[e][1].x, blk[e][1].y) * 4096.f, f[e], acc[e][1]);
              }
            }
          };
          if (S > 1 && n > 4) run(std::integral_constant<int, S>());
          else run(std::integral_constant<int, 1>());
        }
        if (!ok) break;
        const unsigned j = s.base + c.i, place = j % kP;
        if (j >= kP && !(ok = mbar_wait(emptied + place, (j / kP - 1) & 1))) break;
        float2* d = reinterpret_cast<float2*>(part + place * kPart) + lane;
#pragma unroll
        for (int e = 0; e < S; ++e) d[32 * e] = make_float2(acc[e][0], acc[e][1]);
        __syncwarp();
        if (lane == 0) arrive(full + place);
      }
      if (ok && lane == 0) arrive(tile_free + k);
    }
    if (!ok) *s_fail = 1;
  } else if (warp == kStreamW) {
    // ---- the joining warp: a unit's tasks in ascending k, then SwiGLU or the picks' outputs -----------------------------------
    bool ok = true;
    for (int k = 0; ok; ++k) {
      if (k >= nb_first) {
        if (k == nb_first && !mbar_wait(tabbar, 0, 20)) ok = false;
        if (!ok || *s_fail || k >= *s_nseg) break;
      }
      const Seg s = segs[k];
      const int Q = s.down ? QI : QH;
      const bool inter = s.slot == kShared && p.sh_bgu;
      // the unit's slot, and its number among the slot's units
      int slot = s.slot, u = s.u0, reported = 0;
      if (!s.down && s.slot != kShared) slot = u / upp, u -= slot * upp;
      int n = slot == kShared ? p.M : tab.ent[slot].n;
      unsigned j = s.base;
      for (int i = 0; i < s.n && ok; ++i, j += Q, ++u) {
        if (!s.down && s.slot != kShared && u == upp) u = 0, n = tab.ent[++slot].n;
        const unsigned at = j + lane;  // lane q < Q: the unit's task q
        const bool there = lane >= Q || mbar_spin(full + at % kP, at / kP & 1);
        if (!(ok = __all_sync(0xffffffffu, there))) break;
        __syncwarp();
        float2 v[S], d[8][S];
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
          for (int e = 0; e < S; ++e)
            if (q < Q) d[q][e] = (reinterpret_cast<const float2*>(part + ((j + q) % kP) * kPart) + lane)[32 * e];
#pragma unroll
        for (int e = 0; e < S; ++e) {
          v[e] = d[0][e];
#pragma unroll
          for (int q = 1; q < 8; ++q)
            if (q < Q) v[e] = make_float2(__fadd_rn(v[e].x, d[q][e].x), __fadd_rn(v[e].y, d[q][e].y));
        }
        __syncwarp();
        if (lane < Q) arrive(emptied + at % kP);
        if (s.down) {
          float* y = p.y + ((size_t)slot * kMaxRows + t) * p.H + 16 * u + g;
#pragma unroll
          for (int e = 0; e < S; ++e)
            if (4 * e + t < n) y[(size_t)4 * e * p.H] = v[e].x, y[(size_t)4 * e * p.H + 8] = v[e].y;
          continue;
        }
        float* h = p.h + ((size_t)slot * kMaxRows + t) * p.I + 8 * u;
        if (inter) {
          // interleaved rows: strip rows 2 i and 2 i + 1 are gate and up of a channel (first strip: channels 0-3, second: 4-7)
#pragma unroll
          for (int e = 0; e < S; ++e) {
            const float ua = __shfl_down_sync(0xffffffffu, v[e].x, 4), ub = __shfl_down_sync(0xffffffffu, v[e].y, 4);
            if (!(g & 1) && 4 * e + t < n) {
              h[(size_t)4 * e * p.I + (g >> 1)] = __fmul_rn(quick_silu(v[e].x), ua);
              h[(size_t)4 * e * p.I + 4 + (g >> 1)] = __fmul_rn(quick_silu(v[e].y), ub);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < S; ++e)
            if (4 * e + t < n) h[(size_t)4 * e * p.I + g] = __fmul_rn(quick_silu(v[e].x), v[e].y);
        }
        // the run's units of a slot are reported together: h is read when all of the slot's are there
        if (i + 1 == s.n || (s.slot != kShared && u + 1 == upp)) {
          __syncwarp();
          if (lane == 0) red_release(&sy->cnt_h[slot], i + 1 - reported);
          reported = i + 1;
        }
      }
    }
    if (ok && !*s_fail) {
      __syncwarp();
      if (lane == 0) red_release(&sy->cnt_done, 1);
    } else {
      *s_fail = 1;
    }
  } else if (warp > kStreamW + 1) {
    // ---- the producers: a lane fills one stream warp's ring as its stages are freed (a warp that fills its own spends 650 to 1000 of
    // 4400 cycles a stage on it, all of them in its way: 168 experts and four rows took 177 us instead of 151)
    const int w = V::NP * lane + (warp - kStreamW - 2);
    uint8_t* myring = ring + (size_t)w * NST * kStage;
    uint64_t *mybar = bars + w * NST, *myfreed = freed + w * NST;
    const uint64_t pol = policy_evict_first();
    uint32_t issued = 0;
    int nknown = nb_first, ps = 0, pslot = -1, pb = 0, pe = 0, pc = 0;
    bool all_known = false, inside = false, more = w < kStreamW;
    Cursor cur{0, 0, 0, 0};
    Seg sg = segs[0];
    const uint8_t *pa = nullptr, *pz = nullptr, *base_a = nullptr, *base_z = nullptr;
    long long t0 = clock64();
    while (__any_sync(0xffffffffu, more)) {
      bool moved = false;
      // the next task with a block to fetch, if its segment is known
      if (more && pb == pe) {
        if (inside) next(cur, sg);
        if (inside && cur.i >= sg.tasks) ++ps, inside = false;
        if (!inside) {
          if (ps >= nknown && !all_known && mbar_test_wait(tabbar, 0)) all_known = true, nknown = *s_nseg;
          if (ps < nknown) sg = segs[ps], inside = true, pslot = -1, enter(cur, sg, w), moved = true;
          else if (all_known) more = false;
        }
        if (more && inside && cur.i < sg.tasks) {
          const int nb = sg.down ? nbI : nbH;
          const uint32_t blk = sg.b16 ? 4 * kHBlk : kQBlk;  // bytes of 8 rows x 512 k
          if (cur.slot != pslot) {
            pslot = cur.slot;
            if (sg.down) {
              base_a = pslot == kShared ? p.sh_d : tab.ent[pslot].d, base_z = base_a + (size_t)nb * blk;
            } else if (pslot == kShared) {
              base_a = p.sh_bgu ? p.sh_bgu : p.sh_g, base_z = p.sh_bgu ? base_a + (size_t)nb * blk : p.sh_u;
            } else {
              base_a = tab.ent[pslot].g, base_z = tab.ent[pslot].u;
            }
          }
          const int* fb = first_blk + (sg.down ? 12 : 0) + cur.q;
          pb = fb[0], pe = fb[1], pc = 0;
          const bool both = sg.down || (pslot == kShared && p.sh_bgu);  // the unit's two strips follow each other in one matrix
          const size_t off = (size_t)((both ? 2 * cur.u : cur.u) * nb + pb) * blk;
          pa = base_a + off, pz = base_z + off, moved = true;
        }
      }
      if (more && pb < pe) {
        const uint32_t slot = issued % NST;
        if (issued < (uint32_t)NST || mbar_test_wait(myfreed + slot, (issued / NST - 1) & 1)) {
          const uint32_t bytes = sg.b16 ? kHBlk : kQBlk;
          uint8_t* st = myring + slot * kStage;
          mbar_expect_tx(mybar + slot, 2 * bytes);
          bulk_g2s_hint(st, pa, bytes, mybar + slot, pol);
          bulk_g2s_hint(st + kQBlk, pz, bytes, mybar + slot, pol);
          ++issued, pa += bytes, pz += bytes, moved = true;
          if (!sg.b16 || ++pc == 4) ++pb, pc = 0;
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
        t0 = clock64();
      } else {
        if (*reinterpret_cast<volatile int*>(s_fail) || clock64() - t0 > kWaitCycles) break;
        __nanosleep(20);
      }
    }
    if (__any_sync(0xffffffffu, more)) {  // given up: no copy is left in flight
      *s_fail = 1;
      for (uint32_t n = issued > (uint32_t)NST ? issued - NST : 0; w < kStreamW && n < issued; ++n) mbar_wait(mybar + n % NST, (n / NST) & 1);
    }
    __syncwarp();
  } else {
    // ---- the control warp: opens the segments, the table when it is there ------------------------------------------------------
    auto open_seg = [&](int k) {
      if (lane == 0) arrive(seg_open + k);
      __syncwarp();
    };
    bool ok = true;
    // x: in bf16 for the shared expert, as their format wants it for the routed ones
    for (int k = 0; k <= nb_first && ok; ++k) {
      if (k > 0 && p.nbuf == 1) ok = mbar_wait(tile_free, 0, 20);
      if (!router) open_seg(k);
      if (ok) ok = prepare(k, k < nb_first || p.b16, 0, 0, p.M);
    }
    // the table, and from it this CTA's segments.  Costs of 8 rows x 512 k in 64 bytes; lanes 0 and 1: this CTA's and the next one's
    // first up unit, 2 and 3: down
    const int cI = p.b16 ? 4 * kHBlk / 64 : kQBlk / 64, cS = 4 * kHBlk / 64, nsh = has_sh ? upp : 0, nd = has_sh ? NT : 0;
    const bool up = lane < 2;
    const Deal deal(cta + (lane & 1), cI, up ? nsh : nd, cS, up ? Gs : G, G, up ? kFront / (64 * nbH) : 0);
    const int s0 = shared_begin(cta, nd, G), s1 = shared_begin(cta + 1, nd, G);
    int got = 0;
    if (lane == 0) got = ok && !*s_fail && poll_near(&sy->tab_ready, 1);
    ok = __shfl_sync(0xffffffffu, got, 0) != 0;
    __syncwarp();  // (a shuffle orders no memory: what lane 0 has acquired is the other lanes' from here on)
    if (ok) {
      const int n16 = (int)(offsetof(BlockTab, ent) + min(p.M * p.topk, kMaxEnt) * sizeof(BlockEnt)) / 16;
      for (int i0 = lane; i0 < n16; i0 += 128) {
        uint4 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (i0 + 32 * c < n16) v[c] = __ldcg(reinterpret_cast<const uint4*>(p.tab) + i0 + 32 * c);
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (i0 + 32 * c < n16) reinterpret_cast<uint4*>(&tab)[i0 + 32 * c] = v[c];
      }
      __syncwarp();
      const int at = deal.begin(tab.nslots * (up ? upp : NT));
      const int u0 = __shfl_sync(0xffffffffu, at, 0), u1 = __shfl_sync(0xffffffffu, at, 1);
      const int d0 = __shfl_sync(0xffffffffu, at, 2), d1 = __shfl_sync(0xffffffffu, at, 3);
      if (lane == 0) {
        int nseg = nb_first, base = (a1 - a0) * QH;
        segs[nseg++] = Seg{0, p.b16, 0, p.M, u0, u1 - u0, (u1 - u0) * QH, base}, base += (u1 - u0) * QH;
        if (s1 > s0) {
          mbar_init(tile_full + nseg, p.M * nbI);
          segs[nseg++] = Seg{1, 1, kShared, p.M, s0, s1 - s0, (s1 - s0) * QI, base}, base += (s1 - s0) * QI;
        }
        for (int d = d0, slot = d0 / NT; d < d1; ++slot) {
          const int e = min(d1, (slot + 1) * NT), n = tab.ent[slot].n;
          mbar_init(tile_full + nseg, n * nbI);
          segs[nseg++] = Seg{1, p.b16, slot, n, d - slot * NT, e - d, (e - d) * QI, base}, base += (e - d) * QI;
          d = e;
        }
        *s_nseg = nseg;
      }
      __threadfence_block();
    } else {
      *s_fail = 1;
    }
    __syncwarp();
    if (lane == 0) arrive(tabbar);
    __syncwarp();
    const int nseg = ok ? *s_nseg : 0;
    for (int k = nb_first + 1; ok && k < nseg; ++k) {
      // the tile: the first tile's place (one tile: once the routed experts' x is done with), then the segments' before
      const int j = k - nb_first - 1, before = j >= p.nbuf_down ? k - p.nbuf_down : p.nbuf == 1 ? nb_first : nb_first - 1;
      if (before >= 0) ok = mbar_wait(tile_free + before, 0, 20);
      int there = 0;  // the slot's h, once all of its units are in memory
      if (lane == 0) there = ok && poll_near(&sy->cnt_h[segs[k].slot], upp);
      ok = __shfl_sync(0xffffffffu, there, 0) != 0;
      if (ok) {
        open_seg(k);
        ok = prepare(k, segs[k].b16, 1, segs[k].slot, segs[k].rows);
      }
    }
    if (!ok) *s_fail = 1;
  }

  // ---- every CTA's outputs are in memory: a row's picks in ascending expert id, the shared expert, the residual, one rounding
  __syncthreads();
  if (threadIdx.x == 0 && !*s_fail && !poll_near(&sy->cnt_done, G)) *s_fail = 1;
  __syncthreads();
  if (!*s_fail) {
    const int H4 = p.H / 4, items = p.M * H4;
    const int i0 = (int)((long long)items * cta / G), i1 = (int)((long long)items * (cta + 1) / G);
    for (int i = i0 + threadIdx.x; i < i1; i += kThreads) {
      const int m = i / H4, c = 4 * (i - m * H4);
      float4 v[kMaxTopK], sh = make_float4(0.f, 0.f, 0.f, 0.f);
      uint2 r = make_uint2(0u, 0u);
#pragma unroll
      for (int j = 0; j < kMaxTopK; ++j)
        if (j < tab.npick) {
          const int at = tab.pick[m][j];
          v[j] = __ldcg(reinterpret_cast<const float4*>(p.y + ((size_t)(at & 0xff) * kMaxRows + (at >> 8)) * p.H + c));
        }
      if (has_sh) sh = __ldcg(reinterpret_cast<const float4*>(p.y + ((size_t)kShared * kMaxRows + m) * p.H + c));
      if (p.res) r = *reinterpret_cast<const uint2*>(p.res + (size_t)m * p.H + c);
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kMaxTopK; ++j)
        if (j < tab.npick) {
          const float w = tab.w[m][j];
          a.x = fmaf(w, v[j].x, a.x), a.y = fmaf(w, v[j].y, a.y), a.z = fmaf(w, v[j].z, a.z), a.w = fmaf(w, v[j].w, a.w);
        }
      a.x = __fadd_rn(__fadd_rn(a.x, sh.x), bf16_bits_to_f(r.x & 0xffffu)), a.y = __fadd_rn(__fadd_rn(a.y, sh.y), bf16_bits_to_f(r.x >> 16));
      a.z = __fadd_rn(__fadd_rn(a.z, sh.z), bf16_bits_to_f(r.y & 0xffffu)), a.w = __fadd_rn(__fadd_rn(a.w, sh.w), bf16_bits_to_f(r.y >> 16));
      *reinterpret_cast<uint2*>(p.out + (size_t)m * p.H + c) = pack_bf16x4(a.x, a.y, a.z, a.w);
    }
  }
  if (threadIdx.x == 0 && *s_fail) atomicCAS(p.status, 0, (int)DSGX_ERR_DEVICE_WAIT);
  // ---- the last CTA to leave resets the counters ------------------------------------------------------------------------------
  __syncthreads();
  if (threadIdx.x == 0) *s_tick = atomicAdd(&sy->cnt_exit, 1);
  __syncthreads();
  if (*s_tick == G - 1) {
    for (int i = threadIdx.x; i < kMaxEnt + 1; i += kThreads) sy->cnt_h[i] = 0;
    if (threadIdx.x == 0) sy->cnt_lp = 0, sy->cnt_rt = 0, sy->tab_ready = 0, sy->cnt_done = 0, sy->cnt_exit = 0;
  }
}

template <class V>
size_t block_smem(size_t tile, int nbuf) {
  return (size_t)V::W * V::NST * kStage + kP * kPart + sizeof(BlockTab) + nbuf * tile + 64 + (2 * V::W * V::NST + 3 * kMaxSegs + 2 + 2 * kP) * 8 +
         kMaxSegs * (sizeof(Seg) + 4) + 24 * 4 + 4 * 4 + 16;
}
size_t block_tile(int H, int I, int M) {
  return tile_bytes(H, M) > tile_bytes(I, M) ? tile_bytes(H, M) : tile_bytes(I, M);
}

template <class V>
cudaError_t launch(const BlockParams& p, cudaStream_t st) {
  static std::atomic<bool> done[64];  // (per device; two host threads may both set the attribute: harmless)
  int dev = 0;
  cudaGetDevice(&dev);
  if (!done[dev & 63].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(k_block<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax);
    if (e != cudaSuccess) return e;
    done[dev & 63].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count()), cfg.blockDim = dim3(V::kThreads), cfg.dynamicSmemBytes = block_smem<V>(p.tile, p.nbuf), cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeCooperative, at[0].val.cooperative = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_block<V>, p);
}
// (twelve stream warps with two producers, where they fit: one row of 168 experts 58.2 us instead of 58.9, four rows 147 instead of 145)
template <int S>
using Var = BlkVar<S, 11, 2, 3>;

size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace

size_t block_ws_bytes(int H, int I) {
  return 256 + al256(sizeof(BlockSync)) + al256(sizeof(BlockTab)) + al256((size_t)((H + 1023) / 1024) * kMaxRows * 512 * 4) +
         al256((size_t)(kMaxEnt + 1) * kMaxRows * I * 4) + al256((size_t)(kMaxEnt + 1) * kMaxRows * H * 4);
}

// The rows of one launch: as many of M as the activations' shared memory holds (every row's weights are streamed once a launch).
int block_rows(int H, int I, int M) {
  int r = M < kMaxRows ? M : kMaxRows;
  while (r > 1 && block_smem<Var<2>>(block_tile(H, I, r), 1) > kSmemMax) r = (r + 1) / 2;
  return block_smem<Var<2>>(block_tile(H, I, r), 1) > kSmemMax || sm_count() < 2 * kMaxRows ? 0 : r;
}

cudaError_t launch_block_int4(BlockParams p, void* ws, cudaStream_t st) {
  char* w = reinterpret_cast<char*>(ws);
  p.status = reinterpret_cast<int*>(w), w += 256;
  p.sync = reinterpret_cast<BlockSync*>(w), w += al256(sizeof(BlockSync));
  p.tab = reinterpret_cast<BlockTab*>(w), w += al256(sizeof(BlockTab));
  p.lpart = reinterpret_cast<float*>(w), w += al256((size_t)((p.H + 1023) / 1024) * kMaxRows * 512 * 4);
  p.h = reinterpret_cast<float*>(w), w += al256((size_t)(kMaxEnt + 1) * kMaxRows * p.I * 4);
  p.y = reinterpret_cast<float*>(w);
  // Two tiles where they fit: the routed experts' activations are prepared while the shared expert's are in use.
  p.tile = block_tile(p.H, p.I, p.M), p.tile_down = tile_bytes(p.I, p.M), p.nbuf_down = 2 * p.tile_down <= p.tile ? 2 : 1;
  p.nbuf = block_smem<Var<2>>(p.tile, 2) <= kSmemMax ? 2 : 1;
  // One set of rows in the code where that is enough: one row of 168 experts 59.8 -> 58.9 us, of 2048 x 1024 29.6 -> 28.5, four rows
  // of 168 experts 148.5 -> 145.
  return p.M > 4 ? launch<Var<2>>(p, st) : launch<Var<1>>(p, st);
}

}  // namespace dsgx
