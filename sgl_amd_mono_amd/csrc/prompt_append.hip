// Appending a prompt's keys to the paged caches.
//
//   latent  bf16(kv_a g / sqrt(mean(kv_a^2) + eps)), pe = bf16(rope(kv_a[512:])), then
//           E4M3 with one power-of-two scale a token (or raw, clamped to +-448)
//   key     LayerNorm, rope on dims [0, 64), bf16, Hadamard / sqrt(128), bf16, E2M1 with
//           a power-of-two scale for each 32 dims
//
// Everything up to a rounding is formed in f64: an f32 sum's last bits would decide now
// and then which side of a 4-bit code's border a value falls on, and a token's row would
// depend on how its sums were ordered.
//
// 16 lanes take a token, four tokens a wave: every sum is four DPP steps inside a row of
// lanes, the Hadamard's strides 1, 2, 4 lie within a lane and 8 .. 64 between the row's
// lanes, and what a token computes once it computes in 16 lanes and not in 64.
//
// Measured: 32768 bf16 tokens 21.9 us (one wave a token, with LDS permutes and library
// square roots: 37), 3.5 TB/s of its 76 MB against the 4.9 of a large copy; the vector
// unit's f64 and the memory are about even. 1 token 3.9 us.
#include "prompt_common.h"
#include "proj_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 256;
constexpr double EPS = 1e-6;

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
template <int X>
MONO_DEV void lanes_butterfly(double (&y)[8], int sub) {
  const double sign = sub & X ? -1.0 : 1.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fma(sign, y[i], row_xor_d<X>(y[i]));
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

// 1 / sqrt(a), a > 0: the hardware's estimate (some 24 bits) and two Newton steps
MONO_DEV double rsqrt_d(double a) {
  double y = __builtin_amdgcn_rsq(a);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(0.5 * y, fma(-a * y, y, 1.0), y);
  return y;
}

// through f32, as torch casts (an opaque copy: the compiler would fuse the two roundings
// into one, by a longer sequence)
MONO_DEV float to_bf16(double v) {
  float f = (float)v;
  asm("" : "+v"(f));
  return bf16_round(f);
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

// v / 2^(e - 127) within the E4M3 range; what is not finite stays so (its code is NaN)
MONO_DEV float scaled_to_e4m3(float v, float inv) {
  const float q = v * inv;
  return abs_bits(v) < 0x7f800000u ? fminf(fmaxf(q, -FP8_MAX), FP8_MAX) : __uint_as_float(0x7fc00000u);
}

// Eight values of |q| <= 6 as E2M1 codes (the first in the low nibble), ties to even, no
// negative zero: a sign bit stays where its code's magnitude is not zero.
MONO_DEV uint32_t e2m1_pack8(const float (&q)[8]) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.0f, 3);
  return w & (((w & 0x77777777u) + 0x77777777u) | 0x77777777u);
}

template <class V>
__global__ __launch_bounds__(T) void k_append(mono_prompt_append_args a) {
  const int sub = threadIdx.x % 16;
  const int64_t i = (int64_t)blockIdx.x * (T / 16) + threadIdx.x / 16;
  // a lane group without a token to write computes the last token's and stores nothing
  const int64_t n = i < a.tokens ? i : a.tokens - 1;
  int req = a.req[n], pos = a.pos[n];
  bool live = i < a.tokens && req >= 0 && req < a.requests && pos >= 0 && pos < a.max_pos && pos / PAGE < a.pt_stride;
  req = live ? req : 0;
  pos = live ? pos : 0;
  const int page = a.page_table[(int64_t)req * a.pt_stride + pos / PAGE], t = pos % PAGE;
  live = live && page >= 0 && page < a.n_pages;
  if (!__any(live)) return;
  const V* kv = static_cast<const V*>(a.kv_a) + n * a.kv_stride;

  // lane `sub`: latents 8 (sub + 16 q) .. + 7, pe 4 sub .. + 3, index key dims 8 sub .. + 7
  float x[4][8], pe[4], k[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) load8(kv + 8 * (sub + 16 * q), x[q]);
  load4(kv + LATENT + 4 * sub, pe);
  {
    float lo[4], hi[4];
    const V* p = static_cast<const V*>(a.ik) + n * a.ik_stride + 8 * sub;
    load4(p, lo);
    load4(p + 4, hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = lo[e], k[4 + e] = hi[e];
  }
  const float* cos = a.rope_cos + (int64_t)pos * (PE / 2);
  const float* sin = a.rope_sin + (int64_t)pos * (PE / 2);

  double ss = 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fma((double)x[q][e], (double)x[q][e], ss);
  const double rk = rsqrt_d(fma(row_sum_d(ss), 1.0 / LATENT, EPS));
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float g[8];
    load8(static_cast<const uint16_t*>(a.g_kv) + 8 * (sub + 16 * q), g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[q][e] = to_bf16((double)x[q][e] * rk * (double)g[e]);
      m = max(m, abs_bits(x[q][e]));
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const double p0 = pe[2 * e], p1 = pe[2 * e + 1], c = cos[2 * sub + e], s = sin[2 * sub + e];
    pe[2 * e] = to_bf16(p0 * c - p1 * s);
    pe[2 * e + 1] = to_bf16(p0 * s + p1 * c);
    m = max(m, max(abs_bits(pe[2 * e]), abs_bits(pe[2 * e + 1])));
  }
  m = row_umax16(m);
  const uint32_t e = a.kv_scale ? proj::code_ceil(fmaxf(__uint_as_float(min(m, 0x7f7fffffu)), 1e-4f) / FP8_MAX) : 127u;
  const float inv = proj::pow2_of(254u - e);
  const int64_t slot = (int64_t)page * PAGE + t;
  uint8_t* row = static_cast<uint8_t*>(a.kv) + slot * (LATENT + PE);
  if (a.kv_scale && __all(m < 0x7f800000u)) {  // scaled and finite: within the range as it is
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int v = 0; v < 8; ++v) x[q][v] *= inv;
#pragma unroll
    for (int v = 0; v < 4; ++v) pe[v] *= inv;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int v = 0; v < 8; ++v) x[q][v] = scaled_to_e4m3(x[q][v], inv);
#pragma unroll
    for (int v = 0; v < 4; ++v) pe[v] = scaled_to_e4m3(pe[v], inv);
  }
  if (live) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<u32x2*>(row + 8 * (sub + 16 * q)) =
          u32x2{fp8x4_pack(x[q][0], x[q][1], x[q][2], x[q][3]), fp8x4_pack(x[q][4], x[q][5], x[q][6], x[q][7])};
    *reinterpret_cast<uint32_t*>(row + LATENT + 4 * sub) = fp8x4_pack(pe[0], pe[1], pe[2], pe[3]);
    if (sub == 0 && a.kv_scale) a.kv_scale[slot] = proj::pow2_of(e);
  }

  // the index key
  double y[8], sum = 0.0, sq = 0.0;
#pragma unroll
  for (int v = 0; v < 8; ++v) sum += (double)k[v];
  const double mean = row_sum_d(sum) * (1.0 / INDEX);
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    y[v] = (double)k[v] - mean;
    sq = fma(y[v], y[v], sq);
  }
  const double rs = rsqrt_d(fma(row_sum_d(sq), 1.0 / INDEX, EPS));
  float gi[8], bi[8];
  load8(a.g_ik + 8 * sub, gi);
  load8(a.b_ik + 8 * sub, bi);
#pragma unroll
  for (int v = 0; v < 8; ++v) y[v] = fma(y[v] * rs, (double)gi[v], (double)bi[v]);
  const bool turns = sub < PE / 8;
  float c4[4], s4[4];
  load4(cos + 4 * (sub % 8), c4);
  load4(sin + 4 * (sub % 8), s4);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const double c = turns ? c4[v] : 1.0f, s = turns ? s4[v] : 0.0f, y0 = y[2 * v], y1 = y[2 * v + 1];
    y[2 * v] = to_bf16(y0 * c - y1 * s);
    y[2 * v + 1] = to_bf16(y0 * s + y1 * c);
  }
  lane_butterfly(y, 1);
  lane_butterfly(y, 2);
  lane_butterfly(y, 4);
  lanes_butterfly<1>(y, sub);
  lanes_butterfly<2>(y, sub);
  lanes_butterfly<4>(y, sub);
  lanes_butterfly<8>(y, sub);
  uint32_t hm = 0;
#pragma unroll
  for (int v = 0; v < 8; ++v) {
    k[v] = to_bf16(y[v] * 0.08838834764831844055);  // 128^-1/2
    hm = max(hm, abs_bits(k[v]));
  }
  hm = quad_umax(hm);
  const bool finite = hm < 0x7f800000u;
  const uint32_t e8 = finite ? proj::code_ceil(proj::mul_rn(fmaxf(__uint_as_float(hm), 6.0f * 0x1p-126f), 1.0f / 6.0f)) : 255u;
  const float ei = proj::pow2_of(254u - min(e8, 254u));
#pragma unroll
  for (int v = 0; v < 8; ++v) k[v] *= ei;
  if (!live) return;
  // FP4 has no NaN: a block that is not finite gets the scale format's NaN
  const int64_t at = ((int64_t)page * 4 + sub / 4) * PAGE;
  *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.ikv) + (at + t) * 16 + 4 * (sub % 4)) = finite ? e2m1_pack8(k) : 0u;
  if (sub % 4 == 0) static_cast<uint8_t*>(a.iks)[at + t % 16 * 4 + t / 16] = (uint8_t)e8;
}

}  // namespace

hipError_t append(const mono_prompt_append_args& a, hipStream_t st) {
  const uint32_t grid = (uint32_t)((a.tokens + T / 16 - 1) / (T / 16));
  if (a.f32)
    k_append<float><<<grid, T, 0, st>>>(a);
  else
    k_append<uint16_t><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
