// Appending a prompt's keys to the paged caches. One wave a token: lane l holds latents
// 8 l .. 8 l + 7, rotated pair l (l < 32) and index key dims 2 l, 2 l + 1.
//
//   latent  bf16(kv_a g / sqrt(mean(kv_a^2) + eps)), pe = bf16(rope(kv_a[512:])), then
//           E4M3 with one power-of-two scale a token (or raw, clamped to +-448)
//   key     LayerNorm, rope on dims [0, 64), bf16, Hadamard / sqrt(128), bf16, E2M1 with
//           a power-of-two scale for each 32 dims
//
// Everything up to a rounding is formed in f64: an f32 sum's last bits would decide now
// and then which side of a 4-bit code's border a value falls on, and a token's row would
// depend on how its sums were ordered.
#include "prompt_common.h"
#include "proj_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 256, WV = T / WAVE;
constexpr double EPS = 1e-6;

template <int CTRL>
MONO_DEV double dpp_d(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t r = (uint64_t)dpp_u<CTRL>((uint32_t)u) | (uint64_t)dpp_u<CTRL>((uint32_t)(u >> 32)) << 32;
  return __builtin_bit_cast(double, r);
}
MONO_DEV double lane_d(double v, int l) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t r = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), l) << 32;
  return __builtin_bit_cast(double, r);
}
// the sum over the wave, the same in every lane
MONO_DEV double wave_sum_d(double v) {
  v += dpp_d<DPP_XOR1>(v);
  v += dpp_d<DPP_XOR2>(v);
  v += dpp_d<DPP_HALF_MIRROR>(v);
  v += dpp_d<DPP_MIRROR>(v);
  return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}

// through f32, as torch casts (an opaque copy: the compiler would fuse the two roundings
// into one, by a longer sequence)
MONO_DEV float to_bf16(double v) {
  float f = (float)v;
  asm("" : "+v"(f));
  return bf16_round(f);
}

MONO_DEV void load2(const uint16_t* p, float& a, float& b) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  a = bf16_lo(w);
  b = bf16_hi(w);
}
MONO_DEV void load2(const float* p, float& a, float& b) {
  const f32x2 v = *reinterpret_cast<const f32x2*>(p);
  a = v[0];
  b = v[1];
}

// v / 2^(e - 127) within the E4M3 range; what is not finite stays so (its code is NaN)
MONO_DEV float scaled_to_e4m3(float v, float inv) {
  const float q = v * inv;
  return abs_bits(v) < 0x7f800000u ? fminf(fmaxf(q, -FP8_MAX), FP8_MAX) : __uint_as_float(0x7fc00000u);
}

template <class V>
__global__ __launch_bounds__(T) void k_append(mono_prompt_append_args a) {
  const int lane = lane_id();
  const int64_t i = (int64_t)blockIdx.x * WV + threadIdx.x / WAVE;
  if (i >= a.tokens) return;
  const int req = a.req[i], pos = a.pos[i];
  if (req < 0 || req >= a.requests || pos < 0 || pos >= a.max_pos || pos / PAGE >= a.pt_stride) return;
  const int page = a.page_table[(int64_t)req * a.pt_stride + pos / PAGE], t = pos % PAGE;
  if (page < 0 || page >= a.n_pages) return;
  const V* kv = static_cast<const V*>(a.kv_a) + i * a.kv_stride;
  const int pair = lane % 32;  // lanes 32.. repeat the pairs and store none
  float x[8], p0, p1, k0, k1;
  load8(kv + 8 * lane, x);
  load2(kv + LATENT + 2 * pair, p0, p1);
  load2(static_cast<const V*>(a.ik) + i * a.ik_stride + 2 * lane, k0, k1);
  float g[8];
  load8(static_cast<const uint16_t*>(a.g_kv) + 8 * lane, g);
  const double c = a.rope_cos[(int64_t)pos * (PE / 2) + pair], s = a.rope_sin[(int64_t)pos * (PE / 2) + pair];

  double ss = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += (double)x[j] * (double)x[j];
  const double rk = 1.0 / sqrt(wave_sum_d(ss) * (1.0 / LATENT) + EPS);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = to_bf16((double)x[j] * rk * (double)g[j]);
    m = max(m, abs_bits(x[j]));
  }
  const float r0 = to_bf16((double)p0 * c - (double)p1 * s), r1 = to_bf16((double)p0 * s + (double)p1 * c);
  m = wave_umax(max(m, max(abs_bits(r0), abs_bits(r1))));
  const uint32_t e = a.kv_scale ? proj::code_ceil(fmaxf(__uint_as_float(min(m, 0x7f7fffffu)), 1e-4f) / FP8_MAX) : 127u;
  const float inv = proj::pow2_of(254u - e);
  const int64_t slot = (int64_t)page * PAGE + t;
  uint8_t* row = static_cast<uint8_t*>(a.kv) + slot * (LATENT + PE);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = scaled_to_e4m3(x[j], inv);
  *reinterpret_cast<u32x2*>(row + 8 * lane) = u32x2{fp8x4_pack(x[0], x[1], x[2], x[3]), fp8x4_pack(x[4], x[5], x[6], x[7])};
  const uint32_t two = fp8x2_pack(scaled_to_e4m3(r0, inv), scaled_to_e4m3(r1, inv));
  const uint32_t next = dpp_u<DPP_XOR1>(two);
  if (lane < PE / 2 && lane % 2 == 0) *reinterpret_cast<uint32_t*>(row + LATENT + 2 * lane) = two | next << 16;
  if (lane == 0 && a.kv_scale) a.kv_scale[slot] = proj::pow2_of(e);

  // the index key
  const double mean = wave_sum_d((double)k0 + (double)k1) * (1.0 / INDEX);
  const double d0 = (double)k0 - mean, d1 = (double)k1 - mean;
  const double rs = 1.0 / sqrt(wave_sum_d(d0 * d0 + d1 * d1) * (1.0 / INDEX) + EPS);
  const f32x2 gi = *reinterpret_cast<const f32x2*>(a.g_ik + 2 * lane), bi = *reinterpret_cast<const f32x2*>(a.b_ik + 2 * lane);
  double y0 = d0 * rs * (double)gi[0] + (double)bi[0], y1 = d1 * rs * (double)gi[1] + (double)bi[1];
  if (lane < PE / 2) {
    const double z0 = y0 * c - y1 * s, z1 = y0 * s + y1 * c;
    y0 = z0;
    y1 = z1;
  }
  // Hadamard by butterflies: stride 1 within the lane, then the lanes' own bits
  const double f0 = to_bf16(y0), f1 = to_bf16(y1);
  y0 = f0 + f1;
  y1 = f0 - f1;
#pragma unroll
  for (int b = 1; b < WAVE; b <<= 1) {
    const double q0 = __shfl_xor(y0, b, WAVE), q1 = __shfl_xor(y1, b, WAVE);
    y0 = lane & b ? q0 - y0 : y0 + q0;
    y1 = lane & b ? q1 - y1 : y1 + q1;
  }
  const double root = 0.08838834764831844055;  // 128^-1/2
  const float h0 = to_bf16(y0 * root), h1 = to_bf16(y1 * root);
  const uint32_t hm = row_umax16(max(abs_bits(h0), abs_bits(h1)));
  const bool finite = hm < 0x7f800000u;
  const uint32_t e8 = finite ? proj::code_ceil(proj::mul_rn(fmaxf(__uint_as_float(hm), 6.0f * 0x1p-126f), 1.0f / 6.0f)) : 255u;
  const float ei = proj::pow2_of(254u - min(e8, 254u));
  // FP4 has no NaN: a block that is not finite gets the scale format's NaN
  const uint32_t byte = finite ? proj::e2m1_code(h0 * ei) | proj::e2m1_code(h1 * ei) << 4 : 0u;
  uint32_t w = byte | dpp_u<DPP_XOR1>(byte) << 8;  // right in even lanes
  w |= dpp_u<DPP_XOR2>(w) << 16;                   // right in each fourth lane
  const int64_t at = ((int64_t)page * 4 + lane / 16) * PAGE;
  if (lane % 4 == 0) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.ikv) + (at + t) * 16 + lane % 16) = w;
  if (lane % 16 == 0) static_cast<uint8_t*>(a.iks)[at + t % 16 * 4 + t / 16] = (uint8_t)e8;
}

}  // namespace

hipError_t append(const mono_prompt_append_args& a, hipStream_t st) {
  const uint32_t grid = (uint32_t)((a.tokens + WV - 1) / WV);
  if (a.f32)
    k_append<float><<<grid, T, 0, st>>>(a);
  else
    k_append<uint16_t><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
