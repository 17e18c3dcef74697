// Rows of a prompt on their way into and out of the FP8 products: rounding to E4M3 with a
// scale for each 128 columns, sorting the tokens by expert, and the weighted sum back. All
// are bound by the bytes they move (8192 rows of 4096 rounded in 20.5 us, 4.9 TB/s; the sum of
// 8192 tokens x 9 places of 7168 in 296 us, 4.6 TB/s).
#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 1024;     // threads of the row kernels
constexpr int WV = T / WAVE;

// 16 lanes round one block of 128 columns, 8 a lane. `block` counts the blocks of all
// rows, a row's after another.
template <class V>
MONO_DEV void quant_block(const V* x, int64_t stride, uint32_t n_blocks, int kb, const Rows& out, uint32_t block, int sub) {
  const bool in = block < n_blocks;  // whole 16-lane groups: the reduction stays among live values
  const uint32_t b = in ? block : n_blocks - 1;
  const uint32_t row = b / (uint32_t)kb, c = b % (uint32_t)kb;
  float v[8];
  load8(x + (int64_t)row * stride + c * BLK + 8 * sub, v);
  float scale;
  const u32x2 q = quant8(v, scale);
  if (!in) return;
  *reinterpret_cast<u32x2*>(out.q + (size_t)b * BLK + 8 * sub) = q;
  if (sub == 0) out.s[(size_t)c * out.ld + row] = scale;
}

template <class V>
__global__ __launch_bounds__(T) void k_quant_rows(const V* x, int64_t stride, uint32_t n_blocks, int kb, Rows out) {
  quant_block(x, stride, n_blocks, kb, out, blockIdx.x * (T / 16) + threadIdx.x / 16, threadIdx.x % 16);
}

// Blocks [0, experts) sort, the others round rows: neither needs the other.
//
// Sort block e counts the picks of expert e and those of the experts before it, so it knows
// its first place, and writes its picks there, in an order that is its threads' own (a
// place's position among its expert's decides nothing: a row's sums are its own). Its tiles
// go where the counts alone say, too: the experts before e have b places in at most
// min(b, b / bm + e) tiles, so that is where its own begin, and what it has no tile for up
// to the next expert's is left empty (count 0). (65536 picks of 256 experts beside the
// rounding of 8192 rows of 7168: 57 us, of which the rounding alone needs 36; with a
// histogram of every expert in each block 138.)
MONO_DEV int tiles_before(int places, int e, int bm) { return min(places, places / bm + e); }

// Every pick and its index, in an order that is the thread's own and the same each time:
// four neighbours at a time where the ids are aligned for it.
template <class F>
MONO_DEV void for_picks(const int* ids, int picks, F f) {
  const int whole = (uintptr_t)ids % 16 == 0 ? picks / 4 : 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < whole; i += T) {
    const i32x4 v = reinterpret_cast<const i32x4*>(ids)[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) f(4 * i + j, v[j]);
  }
  for (int i = 4 * whole + threadIdx.x; i < picks; i += T) f(i, ids[i]);
}

__global__ __launch_bounds__(T) void k_sort_quant(const uint16_t* x, int64_t stride, uint32_t n_blocks, int kb, Rows out,
                                                  const int* ids, int tokens, int k, int experts, int shared, int bm,
                                                  Sorted S) {
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
  if (e >= experts) {
    quant_block(x, stride, n_blocks, kb, out, (blockIdx.x - experts) * (T / 16) + tid / 16, tid % 16);
    return;
  }
  __shared__ int part[WV][2];
  const int picks = tokens * k, sh_tiles = shared ? (tokens + bm - 1) / bm : 0;
  int mine = 0, less = 0;
  for_picks(ids, picks, [&](int i, int id) {
    mine += id == e ? 1 : 0;
    less += id >= 0 && id < e ? 1 : 0;
    if (e == 0 && (id < 0 || id >= experts)) S.place[i] = -1;
  });
  const int incl = wave_incl_scan(mine), all_less = wave_sum_i(less);
  if (lane == WAVE - 1) part[wave][0] = incl, part[wave][1] = all_less;
  __syncthreads();
  int first = 0, count = 0, at = incl - mine;
#pragma unroll
  for (int w = 0; w < WV; ++w) {
    at += w < wave ? part[w][0] : 0;
    count += part[w][0];
    first += part[w][1];
  }
  const int t0 = tiles_before(first, e, bm);
  const int t1 = e == experts - 1 ? tiles_before(picks, experts, bm) : tiles_before(first + count, e + 1, bm);
  for (int j = tid; j < t1 - t0; j += T)
    S.tiles[sh_tiles + t0 + j] = Tile{e, first + j * bm, max(0, min(bm, count - j * bm)), 0};
  if (shared) {
    for (int t = e * T + tid; t < tokens; t += experts * T) S.token[picks + t] = t;
    for (int j = e * T + tid; j < sh_tiles; j += experts * T)
      S.tiles[j] = Tile{experts, picks + j * bm, min(bm, tokens - j * bm), 0};
  }
  if (count == 0) return;
  at += first;
  for_picks(ids, picks, [&](int i, int id) {
    if (id == e) {
      S.place[i] = at;
      S.token[at++] = i / k;
    }
  });
}

MONO_DEV void load_part(const Parts& p, int64_t place, int c, float (&v)[8]) {
  const u32x4 u = ld_u32x4(p.v + place * p.ld + c);
  const float s = p.s[place * (p.ld / PART) + c / PART];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = u[i];
    v[2 * i] = half_to_f32(w) * s;
    v[2 * i + 1] = half_to_f32(w >> 16) * s;
  }
}

// out[t] = residual[t] + shared part + sum_j weight[t, j] part[place of pick j], in the
// picks' own order (f32 sums, one rounding to bf16). A thread sums 8 columns.
__global__ __launch_bounds__(128) void k_back(Experts a) {
  const int t = blockIdx.x, c = (blockIdx.y * 128 + threadIdx.x) * 8;
  if (c >= a.hidden) return;
  constexpr int U = 8;  // picks loaded together
  float y[8], v[U][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = 0.f;
  u32x4 r = {0u, 0u, 0u, 0u};  // (on its way before the places are waited for)
  if (a.residual) r = ld_u32x4(static_cast<const uint16_t*>(a.residual) + (int64_t)t * a.residual_stride + c);
  if (a.shared) load_part(a.part, a.picks + t, c, y);
  for (int j0 = 0; j0 < a.picks_each; j0 += U) {
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = (int64_t)t * a.picks_each + min(j0 + u, a.picks_each - 1);
      const int p = j0 + u < a.picks_each ? a.sorted.place[j] : -1;
      load_part(a.part, max(p, 0), c, v[u]);  // no place: any place's, not added
      w[u] = p < 0 ? 0.f : a.weights[j];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = p < 0 ? 0.f : v[u][i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fmaf(w[u], v[u][i], y[i]);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = r[i];
      y[2 * i] += bf16_lo(u);
      y[2 * i + 1] += bf16_hi(u);
    }
  }
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_stride + c) =
      u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
}

// The sums of a product whose K was shared out, in the shares' order. A thread adds 4 outputs.
template <bool F32>
__global__ __launch_bounds__(256) void k_join(const float* part, int splits, int64_t rows, int n, void* out, int64_t out_ld) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, each = n / 4;
  if (i >= rows * each) return;
  const int64_t row = i / each, c = 4 * (i % each);
  f32x4 y = *reinterpret_cast<const f32x4*>(part + row * n + c);
  for (int s = 1; s < splits; ++s) y += *reinterpret_cast<const f32x4*>(part + (s * rows + row) * n + c);
  if (F32)
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + row * out_ld + c) = y;
  else
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + row * out_ld + c) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
}

}  // namespace

hipError_t join_product(const Product& a, hipStream_t st) {
  const uint32_t grid = (uint32_t)((a.rows * (a.n / 4) + 255) / 256);
  if (a.f32)
    k_join<true><<<grid, 256, 0, st>>>(a.part, a.plan.splits, a.rows, a.n, a.out, a.out_stride);
  else
    k_join<false><<<grid, 256, 0, st>>>(a.part, a.plan.splits, a.rows, a.n, a.out, a.out_stride);
  return hipGetLastError();
}

hipError_t quant_rows(const void* x, bool f32, int64_t stride, int64_t rows, int k, const Rows& out, hipStream_t st) {
  const int kb = k / BLK;
  const int64_t most = ROUND_BLOCKS / kb;
  for (int64_t r = 0; r < rows; r += most) {
    const uint32_t n = (uint32_t)((rows - r < most ? rows - r : most) * kb), grid = (n + T / 16 - 1) / (T / 16);
    const Rows to{out.q + (size_t)r * k, out.s + r, out.ld};
    if (f32)
      k_quant_rows<<<grid, T, 0, st>>>(static_cast<const float*>(x) + r * stride, stride, n, kb, to);
    else
      k_quant_rows<<<grid, T, 0, st>>>(static_cast<const uint16_t*>(x) + r * stride, stride, n, kb, to);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

hipError_t sort_quant(const void* x, int64_t stride, int64_t tokens, int k, const Rows& out, const int* ids, int picks_each,
                      int experts, bool shared, int bm, const Sorted& sorted, hipStream_t st) {
  const int kb = k / BLK;
  const int64_t most = ROUND_BLOCKS / kb, here = tokens < most ? tokens : most;
  const uint32_t n = (uint32_t)(here * kb), grid = experts + (n + T / 16 - 1) / (T / 16);
  const uint16_t* rows = static_cast<const uint16_t*>(x);
  k_sort_quant<<<grid, T, 0, st>>>(rows, stride, n, kb, out, ids, (int)tokens, picks_each, experts, shared, bm, sorted);
  if (hipError_t e = hipGetLastError()) return e;
  return quant_rows(rows + here * stride, false, stride, tokens - here, k, Rows{out.q + (size_t)here * k, out.s + here, out.ld}, st);
}

hipError_t experts_back(const Experts& a, hipStream_t st) {
  k_back<<<dim3((uint32_t)a.tokens, (a.hidden / 8 + 127) / 128), 128, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
