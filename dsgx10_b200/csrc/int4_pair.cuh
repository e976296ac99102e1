// The inner product of the 4-bit operators (linear.cu, block_int4.cu): a pair of 8-row INT4-g32 blocks (512 k each) against the
// rows of a bf16 activation tile, and the same for bf16 blocks.
//
// W[n][k] = (u - z) s with one bf16 scale s and one nibble z a group of 32 along K.  u - z is a whole number of at most 15,
// so it is exact in bf16; the scale is applied to the group's f32 sum, so W itself is never rounded.
//
// How a group's sum is had from m16n8k16 MMAs although the blocks' lanes mix two groups in every MMA (lane 4 g + t holds
// k = 64 q + 16 t + 0..15 of row g, so lanes t = 0, 1 hold one group of 32 and t = 2, 3 the next): the eight columns of B are
// (token, half) pairs.  Column 2 r + h holds token r's activations in the lanes of half h and zeros in the others, so column
// 2 r + h of D is the sum over group h alone, and lane (g, t) ends with both sums of token t: two fused multiply-adds with
// the row's two scales finish 64 k.  Four tokens an MMA instead of eight, but the weights' conversion (the part that bounds
// these kernels: 28 logic and 16 subtract instructions for 32 weights a lane) loses its multiply by the scale, and a
// token's bits depend neither on the other tokens nor on their number.
#pragma once
#include "common.cuh"
#include "decode_common.cuh"

namespace dsgx {

constexpr int kQBlk = 2368;                          // an INT4 block: 8 rows x 512 k
constexpr int kHBlk = 2048;                          // a bf16 block: 8 rows x 128 k
constexpr int kPairBytes = 2 * kQBlk;
constexpr int kPairStage = (kPairBytes + 127) & ~127;  // (two bf16 blocks, 4096 B, fit)

// shared memory by 32-bit addresses (a generic pointer costs 64-bit arithmetic in the inner loop)
DSGX_DEV uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
DSGX_DEV uint32_t lds_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
// nibbles i and i + 4 of a word minus the zero point, as bf16x2 (zz = 128 + z in both halves): 0x4300 | u is 128 + u
DSGX_DEV uint32_t nib_pair(uint32_t w, int i, uint32_t zz) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w >> (4 * i)), "r"(0x000F000Fu), "r"(0x43004300u));  // (w & m) | c
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&zz));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// c += a b on both halves of a register pair
DSGX_DEV void fma2(float2& c, float2 a, float2 b) {
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%0, %1};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "+f"(c.x), "+f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}
DSGX_DEV void mma_bf16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Where a lane finds its column's activations.  The tile: [K / 64 spans][rows][4 groups][16 bf16 in tile_pos order], so that the
// four lanes of a column read 32-byte steps of one 128-byte line (rows inside the groups cost four-way bank conflicts:
// 8 rows 213 us against 101 on 131072 x 4096).  Set s holds the tokens 4 s .. 4 s + 3.  Lanes of the other half, and columns
// without a token, read 32 bytes of zeros (step 0) that lie 16 bytes off a multiple of 32: the banks the others leave free.
template <int S>
struct XCols {
  uint32_t p[S];     // shared-memory address
  uint32_t step[S];  // bytes from one 64-k span to the next
};
// tok(s, j): the tile row of the j-th token of set s, negative: none
template <int S, class F>
DSGX_DEV void xcols_int4(XCols<S>& x, uint32_t tile, int rows, uint32_t zero, int lane, F tok) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int r = tok(s, g >> 1);
    const bool on = r >= 0 && (t >> 1) == (g & 1);
    x.p[s] = on ? tile + (r * 4 + t) * 32 : zero;
    x.step[s] = on ? 4u * rows * 32 : 0u;
  }
}

// acc[s][0 / 1] += row g of strip a / b times token 4 s + t over the 512 k of one block pair, the two halves of the groups
// apart (.x, .y); st: the pair's stage, strip b kQBlk after strip a; x at the block's first k
template <int S>
DSGX_DEV void int4_pair(float2 (&acc)[S][2], uint32_t st, XCols<S> x, int lane) {
  constexpr int QI = 1, UNR = S == 1 ? 4 : 1;
  const int g = lane >> 2, h = (lane >> 1) & 1;
  const uint32_t az = st + 2304 + 8 * g + 4 * h;
  const uint32_t za = lds_u32(az), zb = lds_u32(az + kQBlk);
  const uint32_t zae = za & 0x0F0F0F0Fu, zao = (za >> 4) & 0x0F0F0F0Fu;
  const uint32_t zbe = zb & 0x0F0F0F0Fu, zbo = (zb >> 4) & 0x0F0F0F0Fu;
  uint32_t av = st + 16 * lane, as = st + 2048 + 32 * g, zsel = 0x4040u;  // bytes (nibble jj, 0x43, nibble jj, 0x43): 128 + z twice
#pragma unroll UNR
  for (int jj = 0; jj < 4; ++jj) {
    const uint4 va = lds_v4(av), vb = lds_v4(av + kQBlk);
    const uint32_t sa0 = lds_u32(as), sa1 = lds_u32(as + 16), sb0 = lds_u32(as + kQBlk), sb1 = lds_u32(as + kQBlk + 16);
#pragma unroll
    for (int q0 = 0; q0 < 2; q0 += QI) {
      uint32_t wa[QI][8], wb[QI][8];
      uint4 x0[QI][S], x1[QI][S];
      float d[QI][S][4];
#pragma unroll
      for (int c = 0; c < QI; ++c) {
        const int q = q0 + c;
        const uint32_t zza = __byte_perm(q ? zao : zae, 0x43434343u, zsel), zzb = __byte_perm(q ? zbo : zbe, 0x43434343u, zsel);
        const uint32_t al = q ? va.z : va.x, ah = q ? va.w : va.y, bl = q ? vb.z : vb.x, bh = q ? vb.w : vb.y;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          x0[c][s] = lds_v4(x.p[s]), x1[c][s] = lds_v4(x.p[s] + 16);
          x.p[s] += x.step[s];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          wa[c][i] = nib_pair(al, i, zza), wa[c][4 + i] = nib_pair(ah, i, zza);
          wb[c][i] = nib_pair(bl, i, zzb), wb[c][4 + i] = nib_pair(bh, i, zzb);
        }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int c = 0; c < QI; ++c)
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const uint4& xv = m < 2 ? x0[c][s] : x1[c][s];
            const uint32_t b0 = m & 1 ? xv.z : xv.x, b1 = m & 1 ? xv.w : xv.y;
            if (m == 0) mma_bf16_zero(d[c][s], wa[c][0], wb[c][0], wa[c][1], wb[c][1], b0, b1);
            else mma_bf16(d[c][s], wa[c][2 * m], wb[c][2 * m], wa[c][2 * m + 1], wb[c][2 * m + 1], b0, b1);
          }
#pragma unroll
      for (int c = 0; c < QI; ++c) {
        const bool q = q0 + c;
        const float2 fa = q ? make_float2(__uint_as_float(sa0 & 0xffff0000u), __uint_as_float(sa1 & 0xffff0000u))
                            : make_float2(__uint_as_float(sa0 << 16), __uint_as_float(sa1 << 16));
        const float2 fb = q ? make_float2(__uint_as_float(sb0 & 0xffff0000u), __uint_as_float(sb1 & 0xffff0000u))
                            : make_float2(__uint_as_float(sb0 << 16), __uint_as_float(sb1 << 16));
#pragma unroll
        for (int s = 0; s < S; ++s) {
          fma2(acc[s][0], fa, make_float2(d[c][s][0], d[c][s][1]));
          fma2(acc[s][1], fb, make_float2(d[c][s][2], d[c][s][3]));
        }
      }
    }
    av += 512, as += 4, zsel += 0x0101u;
  }
}

// 16 values of row r of x from column k0 on, in tile_pos order, zeros from column K on: the tile's 32 bytes of a (group, row)
DSGX_DEV void tile_group(uint4 (&o)[2], const __nv_bfloat16* row, int k0, int K, bool vec) {
  uint32_t w[8];
  if (vec && k0 + 16 <= K) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(row + k0)), b = __ldg(reinterpret_cast<const uint4*>(row + k0 + 8));
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = k0 + 2 * i;
      const uint32_t lo = k < K ? p[k] : 0u, hi = k + 1 < K ? p[k + 1] : 0u;
      w[i] = lo | hi << 16;
    }
  }
  // words (v0 v1)(v2 v3)(v4 v5)(v6 v7) -> (v0 v4)(v1 v5)(v2 v6)(v3 v7), both halves of the group
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t* d = &o[j].x;
    d[0] = __byte_perm(w[4 * j], w[4 * j + 2], 0x5410), d[1] = __byte_perm(w[4 * j], w[4 * j + 2], 0x7632);
    d[2] = __byte_perm(w[4 * j + 1], w[4 * j + 3], 0x5410), d[3] = __byte_perm(w[4 * j + 1], w[4 * j + 3], 0x7632);
  }
}

}  // namespace dsgx
