// Device pieces the prompt-width operators share: rounding a block of 128 values to
// E4M3 with its scale.
#pragma once

#include "common.h"
#include "prompt_ops.h"

namespace mono {
namespace prompt {

constexpr float LEAST = 0x1p-96f;  // a block's largest magnitude counts as at least this

// A block's scale and what its values are multiplied and divided by on the way to codes.
struct BlockScale {
  float scale;  // a / 448
  float mant;   // a = mant 2^e, mant in [1/2, 1)
  float rcp;    // 1 / mant
  int shift;    // 9 - e
  bool finite;
};

// From the block's largest magnitude as f32 bits (a NaN's bits are above infinity's).
MONO_DEV BlockScale block_scale(uint32_t amax_bits) {
  BlockScale b;
  b.finite = amax_bits < 0x7f800000u;
  const float a = fmaxf(b.finite ? __uint_as_float(amax_bits) : 1.0f, LEAST);
  int e;
  b.mant = frexpf(a, &e);
  b.rcp = 1.0f / b.mant;
  b.shift = 9 - e;
  b.scale = b.finite ? a / FP8_MAX : __uint_as_float(0x7fc00000u);  // a block that is not finite: NaN
  return b;
}

// 448 v / a, correctly rounded but for a last bit where that is no tie: the quotient of
// two bf16 values is often exactly midway between two codes, and the product with a
// rounded reciprocal alone would send such a tie either way. One residual step makes a
// quotient that f32 can hold exact. v and a are scaled by a's exponent first, so nothing
// overflows and only what rounds to zero is lost.
MONO_DEV float to_code_range(float v, const BlockScale& b) {
  const float n = ldexpf(v, b.shift) * 0.875f;
  const float q = n * b.rcp;
  const float r = fmaf(-q, b.mant, n);
  return b.finite ? fminf(fmaxf(fmaf(r, b.rcp, q), -FP8_MAX), FP8_MAX) : 0.0f;
}

MONO_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// unsigned max over each 16 consecutive lanes
MONO_DEV uint32_t row_umax16(uint32_t v) {
  v = max(v, dpp_u<DPP_XOR1>(v));
  v = max(v, dpp_u<DPP_XOR2>(v));
  v = max(v, dpp_u<DPP_HALF_MIRROR>(v));
  return max(v, dpp_u<DPP_MIRROR>(v));
}

// Eight values of a block that 16 lanes hold together -> their codes; every lane of the
// 16 gets the block's scale.
MONO_DEV u32x2 quant8(const float (&v)[8], float& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
  const BlockScale b = block_scale(row_umax16(m));
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = to_code_range(v[i], b);
  scale = b.scale;
  return u32x2{fp8x4_pack(c[0], c[1], c[2], c[3]), fp8x4_pack(c[4], c[5], c[6], c[7])};
}

// Four of a lane's bytes, widened exactly to bf16.
MONO_DEV void widen4(uint32_t w, bf16x8& to, int at) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
  to[at] = a[0], to[at + 1] = a[1], to[at + 2] = b[0], to[at + 3] = b[1];
}

// A block's partial products, A[16 x 128] B[128 x 16]. The FP8 MFMA adds its 128 products
// with fewer than f32's bits (1.4e-5 of the result, measured on N(0, 1) values): too few
// for f32 outputs, whose codes are widened exactly to bf16 (6e-9) at half the rate.
template <bool F32>
MONO_DEV f32x4 mfma_block(const i32x8& a, const i32x8& b) {
  f32x4 p = {0.f, 0.f, 0.f, 0.f};
  if (!F32) return mfma_fp8(a, b, p);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    bf16x8 x, y;
    widen4((uint32_t)a[2 * q], x, 0);
    widen4((uint32_t)a[2 * q + 1], x, 4);
    widen4((uint32_t)b[2 * q], y, 0);
    widen4((uint32_t)b[2 * q + 1], y, 4);
    p = mfma_bf16(x, y, p);
  }
  return p;
}

MONO_DEV void load8(const uint16_t* p, float (&v)[8]) {
  const u32x4 u = ld_u32x4(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = u[i];
    v[2 * i] = bf16_lo(w);
    v[2 * i + 1] = bf16_hi(w);
  }
}
MONO_DEV void load8(const float* p, float (&v)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = a[i];
    v[4 + i] = b[i];
  }
}

MONO_DEV float half_to_f32(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
MONO_DEV uint32_t pack_halves(float a, float b) {
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
}

// The largest of four lane groups' values (lanes l, l ^ 16, l ^ 32, l ^ 48), in all of them.
MONO_DEV uint32_t groups_umax(uint32_t v) {
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(v, v, false, false));
  v = max(a[0], a[1]);
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(v, v, false, false));
  return max(b[0], b[1]);
}

// A lane's 16 of one place's 64 columns (tiles of 16 weight rows i, columns 16 i + 4 g + e of
// lane group g) as halves of a Parts block: the scale, and the values divided by it. The
// scale is that of the largest finite value, so a sum past f32's range is an infinity in its
// own column and costs the other 63 nothing. (The float maximum passes over a NaN, which
// stays one as a half.)
MONO_DEV float part_block(const f32x4 (&y)[4], u32x2 (&h)[4]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(fmaxf(top, fmaxf(fabsf(y[i][0]), fabsf(y[i][1]))), fmaxf(fabsf(y[i][2]), fabsf(y[i][3])));
  uint32_t m = groups_umax(__float_as_uint(top));
  if (__any(m >= 0x7f800000u)) {  // rare: the whole wave again without the infinities
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, abs_bits(y[i][j]) < 0x7f800000u ? fabsf(y[i][j]) : 0.f);
    m = groups_umax(__float_as_uint(top));
  }
  // 2^14 / 2^floor(log2 max)
  const int e = max((int)(m >> 23), 27);
  const float inv = __uint_as_float((uint32_t)(127 + 14 + 127 - e) << 23);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = u32x2{pack_halves(y[i][0] * inv, y[i][1] * inv), pack_halves(y[i][2] * inv, y[i][3] * inv)};
  return __uint_as_float((uint32_t)(e - 14) << 23);
}

// 16 rows of 64 two-byte values as the MFMA leaves them (lane r + 16 g: columns 16 i + 4 g ..
// + 3 of row r) stored as whole 128-byte rows, through 2 KB of LDS that are the wave's own:
// straight from the lanes a store would touch 32 bytes of each of 16 rows. `store(row,
// column, 16 bytes)`; the 16-byte pieces are swapped by row, so neither side meets a bank twice.
template <class F>
MONO_DEV void store_rows(uint8_t* buf, const u32x2 (&h)[4], F store) {
  const int lane = lane_id(), r = lane % 16, g = lane / 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<u32x2*>(buf + r * 128 + (((2 * i + g / 2) ^ (r & 7)) * 16) + (g & 1) * 8) = h[i];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int row = lane / 8 + 8 * k, unit = lane % 8;
    store(row, 8 * unit, *reinterpret_cast<const u32x4*>(buf + row * 128 + ((unit ^ (row & 7)) * 16)));
  }
}

// One place's row of a wave's 64 columns into Parts (16 places a call, place `first` + r).
MONO_DEV void store_part(uint8_t* buf, const Parts& p, int64_t first, int count, int col, const f32x4 (&y)[4]) {
  u32x2 h[4];
  const float s = part_block(y, h);
  const int lane = lane_id();
  if (lane < 16 && lane < count) p.s[(first + lane) * (p.ld / PART) + col / PART] = s;
  store_rows(buf, h, [&](int row, int c, u32x4 v) {
    if (row < count) *reinterpret_cast<u32x4*>(p.v + (first + row) * p.ld + col + c) = v;
  });
}

}  // namespace prompt
}  // namespace mono
