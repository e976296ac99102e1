// Pieces of the 4-bit operators (linear.cu, block_int4.cu): nibbles as f16 MMA operands, the activation tile they meet, and the
// shared-memory handshakes between their warps.
//
// W[n][k] = (u - z) s with one bf16 scale s and one nibble z a group of 32 along K.  A nibble u in the low byte of a half-word
// is, as it stands, the f16 subnormal u 2^-24 (bits 0-3) or u 2^-20 (bits 4-7), and the MMA takes subnormals exactly: a word of
// eight weights costs four ANDs and one shift and no arithmetic (the bf16 form, 128 + u minus 128 + z, cost three shifts,
// four logic operations and four subtractions; 131072 x 4096 and one row went from 69 to 64 us).  The scale and the zero
// point meet a group's f32 sum, s (sum u x - z sum x), so W itself is never rounded.
//
// x goes to f16 for that.  Per row and block of 512 k a power of two 2^E brings the largest magnitude into [2^14, 2^15), where
// bf16's eight bits are exact down to 2^-31 of it and smaller values round by at most 2^-39 of the largest.  Values at odd k meet
// a nibble in bits 4-7 and are taken times 2^-4: for them it is 2^-27 and 2^-35, still below an f32 sum's last bit.  Whatever is
// infinite or NaN in a row makes the whole row NaN.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace dsgx {

constexpr int kQBlk = 2368;  // an INT4 block: 8 rows x 512 k
constexpr int kHBlk = 2048;  // a bf16 block: 8 rows x 128 k

// shared memory by 32-bit addresses (a generic pointer costs 64-bit arithmetic in the inner loop)
DSGX_DEV uint4 lds_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
DSGX_DEV uint2 lds_v2(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
DSGX_DEV float2 lds_f2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a));
  return v;
}
DSGX_DEV float lds_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
DSGX_DEV int ld_shared_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}
DSGX_DEV void st_shared_release(int* p, int v) {
  asm volatile("st.release.cta.shared::cta.s32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
// bounded wait until a word of shared memory has reached v
DSGX_DEV bool wait_shared_ge(const int* p, int v, unsigned sleep_ns) {
  if (ld_shared_acquire(p) >= v) return true;
  const long long t0 = clock64();
  while (ld_shared_acquire(p) < v) {
    if (sleep_ns) __nanosleep(sleep_ns);
    if (clock64() - t0 > kWaitCycles) return false;
  }
  return true;
}

// D[16x8] = A[16x16] B[16x8], f16 operands, f32 accumulate (lanes as mma_bf16), and the accumulating form
DSGX_DEV void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
DSGX_DEV void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// a b + c on both halves of a register pair
DSGX_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

DSGX_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

DSGX_DEV float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
DSGX_DEV __nv_bfloat162 abs_bf16x2(uint32_t w) {
  w &= 0x7FFF7FFFu;
  return *reinterpret_cast<const __nv_bfloat162*>(&w);
}

constexpr uint32_t kNib0 = 0x000F000Fu, kNib1 = 0x00F000F0u;  // nibbles 0 and 4 of a word; 1 and 5 (2, 6 and 3, 7 after a shift by 8)
// minus the zero point in byte b of a word of them: 0x4B0000zz is 2^23 + z
DSGX_DEV float minus_zero(uint32_t zeros, int b) { return 8388608.f - __uint_as_float(__byte_perm(zeros, 0x4B000000u, 0x7440u + b)); }
DSGX_DEV float scale_lo(uint32_t v) { return __uint_as_float(v << 16); }
DSGX_DEV float scale_hi(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// 16 bf16 values of a row from column k on (zeros from K on) as eight words.  kCg: written by other SMs during this kernel.
template <bool kCg>
DSGX_DEV void load_16(uint32_t (&w)[8], const __nv_bfloat16* row, int k, int K, bool vec) {
  if (vec && k + 16 <= K) {
    const uint4* p = reinterpret_cast<const uint4*>(row + k);
    const uint4 a = kCg ? __ldcg(p) : __ldg(p), b = kCg ? __ldcg(p + 1) : __ldg(p + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = k + 2 * i < K ? p[k + 2 * i] : 0u, hi = k + 2 * i + 1 < K ? p[k + 2 * i + 1] : 0u;
      w[i] = lo | hi << 16;
    }
  }
}
// words (v0 v1)(v2 v3)(v4 v5)(v6 v7) -> (v0 v4)(v1 v5)(v2 v6)(v3 v7), the order nibbles i and i + 4 meet, both halves of 16 values
DSGX_DEV void nibble_order(uint4 (&o)[2], const uint32_t (&w)[8]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t* d = &o[j].x;
    d[0] = __byte_perm(w[4 * j], w[4 * j + 2], 0x5410), d[1] = __byte_perm(w[4 * j], w[4 * j + 2], 0x7632);
    d[2] = __byte_perm(w[4 * j + 1], w[4 * j + 3], 0x5410), d[3] = __byte_perm(w[4 * j + 1], w[4 * j + 3], 0x7632);
  }
}

// One row's 512 k of a block into the activation tile, by one warp (w: a lane's 16 k): f16 times 2^E; the groups' sums times
// 2^(E - 24); 2^(12 - E).  xt: the row's 128-byte line in the block's first span of 64 k, the next span's `span` bytes on; flip:
// its two groups exchanged; sx: the row's first group sum, GB bytes to the span's second, `sspan` to the next span.
template <int GB>
DSGX_DEV void stage_row(const uint32_t (&w)[8], uint8_t* xt, uint32_t span, bool flip, float* sx, uint32_t sspan, float* scale, int lane) {
  // the largest magnitude (bf16 bits order like numbers; a NaN loses against a number) of the row's 512 values
  __nv_bfloat162 m2 = abs_bf16x2(w[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m2 = __hmax2(m2, abs_bf16x2(w[i]));
  const uint32_t mb = *reinterpret_cast<const uint32_t*>(&m2);
  uint32_t top = __reduce_max_sync(0xffffffffu, max(mb & 0xffffu, mb >> 16));
  if (top >= 0x7F80u) {  // an infinity, or nothing but NaN: the largest finite one
    top = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = w[i] & 0x7FFFu, hi = w[i] >> 16 & 0x7FFFu;
      top = max(top, max(lo < 0x7F80u ? lo : 0u, hi < 0x7F80u ? hi : 0u));
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  const int E = top >= 0x80u ? min(14 + 127 - (int)(top >> 7), 126) : 126;  // (subnormal or zero: as small as it gets)
  const float2 f = make_float2(__uint_as_float((uint32_t)(E + 127) << 23), __uint_as_float((uint32_t)(E - 4 + 127) << 23));
  uint32_t h[8];
  float2 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = mul2(make_float2(scale_lo(w[i]), scale_hi(w[i])), f);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[i]) : "f"(v[i].y), "f"(v[i].x));
  }
#pragma unroll
  for (int n = 4; n > 0; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = add2(v[i], v[i + n]);
  float sum = fmaf(v[0].y, 16.f, v[0].x);
  sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 1));
  uint4 o[2];
  nibble_order(o, h);
  uint4* d = reinterpret_cast<uint4*>(xt + (size_t)(lane >> 2) * span + (((lane & 3) * 32) ^ (flip ? 64 : 0)));
  d[0] = o[0], d[1] = o[1];
  if (!(lane & 1)) *reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sx) + (size_t)(lane >> 2) * sspan + GB * (lane >> 1 & 1)) = sum * 0x1p-24f;
  if (lane == 0) *scale = __uint_as_float((uint32_t)(12 - E + 127) << 23);
}

// The same for 16 f32 values (k = 2 i, 2 i + 1 in v[i]) that are to become a product's f16 operands: 2^E as above, then one
// rounding to f16's eleven bits (fewer below 2^-28 of the block's largest, at odd k with `nib` below 2^-24), and the groups' sums
// are those of the rounded values.  nib: the weights are nibbles (odd k times 2^-4).
DSGX_DEV void stage_row_f32(float2 (&v)[8], bool nib, uint8_t* xt, uint32_t span, float* sx, uint32_t sspan, float* scale, int lane) {
  auto mag = [](float a) { return __float_as_uint(a) & 0x7FFFFFFFu; };
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, max(mag(v[i].x), mag(v[i].y)));
  top = __reduce_max_sync(0xffffffffu, top);
  if (top >= 0x7F800000u) {  // an infinity or a NaN: the largest finite one
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = mag(v[i].x), b = mag(v[i].y);
      top = max(top, max(a < 0x7F800000u ? a : 0u, b < 0x7F800000u ? b : 0u));
    }
    top = __reduce_max_sync(0xffffffffu, top);
  }
  const int E = top >= 0x800000u ? min(14 + 127 - (int)(top >> 23), 126) : 126;
  const float2 f = make_float2(__uint_as_float((uint32_t)(E + 127) << 23), __uint_as_float((uint32_t)(E - (nib ? 4 : 0) + 127) << 23));
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = mul2(v[i], f);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h[i]) : "f"(v[i].y), "f"(v[i].x));
    v[i] = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
  }
#pragma unroll
  for (int n = 4; n > 0; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = add2(v[i], v[i + n]);
  float sum = fmaf(v[0].y, 16.f, v[0].x);
  sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, 1));
  uint4 o[2];
  nibble_order(o, h);
  uint4* d = reinterpret_cast<uint4*>(xt + (size_t)(lane >> 2) * span + (lane & 3) * 32);
  d[0] = o[0], d[1] = o[1];
  if (!(lane & 1)) *reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sx) + (size_t)(lane >> 2) * sspan + 4 * (lane >> 1 & 1)) = sum * 0x1p-24f;
  if (lane == 0) *scale = __uint_as_float((uint32_t)(12 - E + 127) << 23);
}

}  // namespace dsgx
