// The index queries of a prompt's tokens: what the front launch makes of a decode step's.
//
//   y = bf16(x) of a head's 128 dims, dims [0, 64) rotated, bf16, Hadamard / sqrt(128), bf16,
//   E2M1 with a power-of-two scale for each 32 dims
//
// Everything between two roundings is formed in f64, as the appended keys are: a code does not hang
// on the order of a sum. That makes it a matter of vector instructions as much as of bytes (21 KB a
// token). Four lanes take a head, so five of the transform's seven steps stay in a lane and the other
// two are permutations inside a quad (16 lanes a head: 54 instructions a value instead of 26); and a
// lane holds 16 dims of either half, so every lane has as much to turn. A workgroup is a token:
// its position is one scalar.
//
// 8192 tokens, bf16: 45 us, 3.8 TB/s (16 lanes a head: 69 us); a large copy moves 4.9.
#include "prompt_index.h"

namespace mono {
namespace prompt {
namespace {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int T = INDEX_HEADS * 4, HALF = INDEX / 2, N = HALF / 4;  // N: a lane's dims of either half
static_assert(HALF == PE, "the first half turns");

// Of N dims: the values, rounded to bf16 and exact in f64.
MONO_DEV void load_dims(const uint16_t* p, double* y) {
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    float v[8];
    load8(p + i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i + j] = v[j];
  }
}
MONO_DEV void load_dims(const float* p, double* y) {
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    float v[8];
    load8(p + i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i + j] = bf16_round(v[j]);
  }
}

template <class V>
__global__ __launch_bounds__(T) void k_query(mono_prompt_query_args a) {
  const int64_t n = blockIdx.x;
  const int h = threadIdx.x / 4, sub = threadIdx.x % 4;
  int pos = a.pos[n];
  const bool live = pos >= 0 && pos < a.max_pos;
  pos = live ? pos : 0;
  const V* x = static_cast<const V*>(a.x) + n * a.x_stride + h * INDEX + N * sub;
  double y[2 * N];
  load_dims(x, y);
  load_dims(x + HALF, y + N);
  const int64_t turn = (int64_t)pos * (PE / 2) + N / 2 * sub;
  float c[N / 2], s[N / 2];
  load8(a.rope_cos + turn, c);
  load8(a.rope_sin + turn, s);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const double y0 = y[2 * i], y1 = y[2 * i + 1];
    y[2 * i] = to_bf16(y0 * c[i] - y1 * s[i]);
    y[2 * i + 1] = to_bf16(y0 * s[i] + y1 * c[i]);
  }
#pragma unroll
  for (int x = 1; x < 2 * N; x *= 2)
#pragma unroll
    for (int i = 0; i < 2 * N; ++i)
      if (!(i & x)) {
        const double u = y[i], v = y[i + x];
        y[i] = u + v;
        y[i + x] = u - v;
      }
  lanes_butterfly<1>(y, sub);
  lanes_butterfly<2>(y, sub);
  const int64_t v = n * INDEX_HEADS + h;
  uint32_t e8s = 0;
#pragma unroll
  for (int half = 0; half < 2; ++half) {  // two lanes' dims of a half: a block
    uint32_t k[N / 2];
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const double* p = y + N * half + 2 * i;
      k[i] = pack_bf16(p[0] * 0.08838834764831844055, p[1] * 0.08838834764831844055);  // 128^-1/2
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, k[i] & 0x7fff7fffu));
    }
    uint32_t hm = (uint32_t)max(m[0], m[1]) << 16;
    hm = max(hm, dpp_u<DPP_XOR1>(hm));
    const uint32_t e8 = block_code(hm);
    const float scale = proj::pow2_of(e8);
    u32x2 codes;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint32_t u = 0;
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, as_bf16x2(k[4 * w]), scale, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, as_bf16x2(k[4 * w + 1]), scale, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, as_bf16x2(k[4 * w + 2]), scale, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, as_bf16x2(k[4 * w + 3]), scale, 3);
      codes[w] = live && e8 < 255 ? no_negative_zero(u) : 0u;
    }
    *reinterpret_cast<u32x2*>(static_cast<uint32_t*>(a.iq) + v * (INDEX / 8) + (HALF * half + N * sub) / 8) = codes;
    const uint32_t other = dpp_u<DPP_XOR2>(e8);
    e8s |= (e8 | other << 8) << (16 * half);
  }
  if (sub == 0) static_cast<uint32_t*>(a.iqs)[v] = live ? e8s : 0u;
}

}  // namespace

hipError_t index_query(const mono_prompt_query_args& a, hipStream_t st) {
  const uint32_t grid = (uint32_t)a.tokens;
  if (a.f32)
    k_query<float><<<grid, T, 0, st>>>(a);
  else
    k_query<uint16_t><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
