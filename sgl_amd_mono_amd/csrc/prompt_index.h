// Device pieces of the index vectors (keys that are appended, queries): f64 sums and
// butterflies over the 16 lanes that hold a vector, its roundings and its FP4 codes.
#pragma once

#include "proj_common.h"
#include "prompt_common.h"

namespace mono {
namespace prompt {

// (every lane has a source here, so nothing needs the register's old value)
template <int CTRL>
MONO_DEV uint32_t dpp_all(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
MONO_DEV double dpp_d(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t r = (uint64_t)dpp_all<CTRL>((uint32_t)u) | (uint64_t)dpp_all<CTRL>((uint32_t)(u >> 32)) << 32;
  return __builtin_bit_cast(double, r);
}
// the sum over each 16 lanes, the same in every one of them
MONO_DEV double row_sum_d(double v) {
  v += dpp_d<DPP_XOR1>(v);
  v += dpp_d<DPP_XOR2>(v);
  v += dpp_d<DPP_HALF_MIRROR>(v);
  return v + dpp_d<DPP_MIRROR>(v);
}
// lane i's value of lane i ^ 4 in each 16 lanes: banks of 4 lanes rotated by one bank, the
// odd ones forwards, the even ones backwards
MONO_DEV uint32_t xor4_u(uint32_t v) {
  const int up = (int)dpp_all<0x124>(v);  // row_ror:4: right for banks 1 and 3
  return (uint32_t)__builtin_amdgcn_update_dpp(up, (int)v, 0x12c, 0xf, 0x5, false);  // row_ror:12 over banks 0 and 2
}
constexpr int DPP_XOR8 = 0x128;  // row_ror:8
template <int X>
MONO_DEV double row_xor_d(double v) {
  if (X != 4) return dpp_d<X == 1 ? (int)DPP_XOR1 : X == 2 ? (int)DPP_XOR2 : DPP_XOR8>(v);
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)xor4_u((uint32_t)u) | (uint64_t)xor4_u((uint32_t)(u >> 32)) << 32);
}
// A butterfly between lanes X apart: a + b in the lane with the bit clear, a - b in its partner.
template <int X, int N>
MONO_DEV void lanes_butterfly(double (&y)[N], int sub) {
  const double sign = sub & X ? -1.0 : 1.0;
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = fma(sign, y[i], row_xor_d<X>(y[i]));
}
MONO_DEV void lane_butterfly(double (&y)[8], int x) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (!(i & x)) {
      const double a = y[i], b = y[i + x];
      y[i] = a + b;
      y[i + x] = a - b;
    }
}

// through f32, as torch casts (an opaque copy: the compiler would fuse the two roundings
// into one, by a longer sequence)
MONO_DEV float to_bf16(double v) {
  float f = (float)v;
  asm("" : "+v"(f));
  return bf16_round(f);
}

MONO_DEV uint32_t pack_bf16(double a, double b) {
  float x = (float)a, y = (float)b;
  asm("" : "+v"(x), "+v"(y));
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)x, (__bf16)y});
}

// the larger of each magnitude's bits over the 16 lanes of a token, over 4 lanes of it
MONO_DEV uint32_t quad_umax(uint32_t v) {
  v = max(v, dpp_u<DPP_XOR1>(v));
  return max(v, dpp_u<DPP_XOR2>(v));
}

MONO_DEV void load4(const uint16_t* p, float (&v)[4]) {
  const u32x2 w = *reinterpret_cast<const u32x2*>(p);
  const uint32_t a = w[0], b = w[1];
  v[0] = bf16_lo(a), v[1] = bf16_hi(a), v[2] = bf16_lo(b), v[3] = bf16_hi(b);
}
MONO_DEV void load4(const float* p, float (&v)[4]) {
  const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = w[i];
}

// Eight E2M1 codes without negative zeros: a sign bit stays where its code's magnitude is not zero.
MONO_DEV uint32_t no_negative_zero(uint32_t w) { return w & (((w & 0x77777777u) + 0x77777777u) | 0x77777777u); }

// Eight values of |q| <= 6 as E2M1 codes (the first in the low nibble), ties to even, no
// negative zero.
MONO_DEV uint32_t e2m1_pack8(const float (&q)[8]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.0f, 3);
  return no_negative_zero(w);
}

// The code of the scale of a block whose largest magnitude has the f32 bits hm: the smallest power of
// two that it divided by is at most 6; NaN's, 255, where it is not finite.
MONO_DEV uint32_t block_code(uint32_t hm) {
  return hm < 0x7f800000u ? proj::code_ceil(proj::mul_rn(fmaxf(__uint_as_float(hm), 6.0f * 0x1p-126f), 1.0f / 6.0f)) : 255u;
}

// The codes of a vector whose rotated values (dims 8 sub .. + 7, bf16 values) are y: Hadamard,
// x 128^-1/2, bf16, and E2M1 with a power-of-two scale for each 32 dims (4 lanes). FP4 has no
// NaN: a block that is not finite has zero codes and the scale format's NaN, 255.
MONO_DEV uint32_t index_codes(double (&y)[8], int sub, uint32_t& e8) {
  lane_butterfly(y, 1);
  lane_butterfly(y, 2);
  lane_butterfly(y, 4);
  lanes_butterfly<1>(y, sub);
  lanes_butterfly<2>(y, sub);
  lanes_butterfly<4>(y, sub);
  lanes_butterfly<8>(y, sub);
  float k[8];
  uint32_t hm = 0;
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    k[v] = to_bf16(y[v] * 0.08838834764831844055);  // 128^-1/2
    hm = max(hm, abs_bits(k[v]));
  }
  hm = quad_umax(hm);
  e8 = block_code(hm);
  const float ei = proj::pow2_of(254u - min(e8, 254u));
#pragma unroll
  for (int v = 0; v < 8; ++v) k[v] *= ei;
  return e8 < 255 ? e2m1_pack8(k) : 0u;
}

}  // namespace prompt
}  // namespace mono
