// The index queries of a prompt's tokens: what the front launch makes of a decode step's.
//
//   y = bf16(x) of a head's 128 dims, dims [0, 64) rotated, bf16, Hadamard / sqrt(128), bf16,
//   E2M1 with a power-of-two scale for each 32 dims
//
// 16 lanes take a head of a token, four a wave, and form everything between two roundings in
// f64, as the appended keys are: a code does not hang on the order of a sum.
#include "prompt_index.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 256;

template <class V>
__global__ __launch_bounds__(T) void k_query(mono_prompt_query_args a) {
  const int sub = threadIdx.x % 16;
  const int64_t v = (int64_t)blockIdx.x * (T / 16) + threadIdx.x / 16, n = v / INDEX_HEADS;  // (a token's heads fill whole workgroups)
  const int h = v % INDEX_HEADS;
  int pos = a.pos[n];
  const bool live = pos >= 0 && pos < a.max_pos;
  pos = live ? pos : 0;
  float k[8];
  load8(static_cast<const V*>(a.x) + n * a.x_stride + h * INDEX + 8 * sub, k);
  const bool turns = sub < PE / 8;
  float c4[4], s4[4];
  load4(a.rope_cos + (int64_t)pos * (PE / 2) + 4 * (sub % 8), c4);
  load4(a.rope_sin + (int64_t)pos * (PE / 2) + 4 * (sub % 8), s4);
  double y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double c = turns ? c4[i] : 1.0f, s = turns ? s4[i] : 0.0f, y0 = bf16_round(k[2 * i]), y1 = bf16_round(k[2 * i + 1]);
    y[2 * i] = to_bf16(y0 * c - y1 * s);
    y[2 * i + 1] = to_bf16(y0 * s + y1 * c);
  }
  uint32_t e8;
  const uint32_t codes = index_codes(y, sub, e8);
  static_cast<uint32_t*>(a.iq)[v * (INDEX / 8) + sub] = live ? codes : 0u;
  if (sub % 4 == 0) static_cast<uint8_t*>(a.iqs)[v * (INDEX / 32) + sub / 4] = live ? (uint8_t)e8 : 0;
}

}  // namespace

hipError_t index_query(const mono_prompt_query_args& a, hipStream_t st) {
  const uint32_t grid = (uint32_t)(a.tokens * INDEX_HEADS / (T / 16));
  if (a.f32)
    k_query<float><<<grid, T, 0, st>>>(a);
  else
    k_query<uint16_t><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
