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
#include "prompt_index.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 256;
constexpr double EPS = 1e-6;

// 1 / sqrt(a), a > 0: the hardware's estimate (some 24 bits) and two Newton steps
MONO_DEV double rsqrt_d(double a) {
  double y = __builtin_amdgcn_rsq(a);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(0.5 * y, fma(-a * y, y, 1.0), y);
  return y;
}

// v / 2^(e - 127) within the E4M3 range; what is not finite stays so (its code is NaN)
MONO_DEV float scaled_to_e4m3(float v, float inv) {
  const float q = v * inv;
  return abs_bits(v) < 0x7f800000u ? fminf(fmaxf(q, -FP8_MAX), FP8_MAX) : __uint_as_float(0x7fc00000u);
}

template <class V>
__global__ __launch_bounds__(T) void k_append(mono_prompt_append_args a, const int32_t* slot_pos) {
  const int sub = threadIdx.x % 16;
  const int64_t i = (int64_t)blockIdx.x * (T / 16) + threadIdx.x / 16;
  // a lane group without a token to write computes the last token's and stores nothing
  const int64_t n = i < a.tokens ? i : a.tokens - 1;
  int req = a.req[n], pos = a.pos[n], at_pos = slot_pos ? slot_pos[n] : pos;
  bool live = i < a.tokens && req >= 0 && req < a.requests && pos >= 0 && pos < a.max_pos && at_pos >= 0 && at_pos / PAGE < a.pt_stride;
  req = live ? req : 0;
  pos = live ? pos : 0;
  at_pos = live ? at_pos : 0;
  const int page = a.page_table[(int64_t)req * a.pt_stride + at_pos / PAGE], t = at_pos % PAGE;
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
  uint32_t e8;
  const uint32_t codes = index_codes(y, sub, e8);
  if (!live) return;
  const int64_t at = ((int64_t)page * 4 + sub / 4) * PAGE;
  *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.ikv) + (at + t) * 16 + 4 * (sub % 4)) = codes;
  if (sub % 4 == 0) static_cast<uint8_t*>(a.iks)[at + t % 16 * 4 + t / 16] = (uint8_t)e8;
}

}  // namespace

hipError_t append(const mono_prompt_append_args& a, const int32_t* slot_pos, hipStream_t st) {
  const uint32_t grid = (uint32_t)((a.tokens + T / 16 - 1) / (T / 16));
  if (a.f32)
    k_append<float><<<grid, T, 0, st>>>(a, slot_pos);
  else
    k_append<uint16_t><<<grid, T, 0, st>>>(a, slot_pos);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
