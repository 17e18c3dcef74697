// Rows of a prompt on their way into and out of the FP8 products: rounding to E4M3 with a
// scale for each 128 columns, sorting the tokens by expert, and the weighted sum back.
#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 512;      // threads of the row kernels
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
// Sort block e counts every expert's picks in LDS (integer atomics: the order does not
// show), so it knows where its own places and tiles begin without another launch, then
// lists its picks in the tokens' order: each wave takes one contiguous share, counts
// its matches, and writes them behind those of the waves before it.
__global__ __launch_bounds__(T) void k_sort_quant(const uint16_t* x, int64_t stride, uint32_t n_blocks, int kb, Rows out,
                                                  const int* ids, int tokens, int k, int experts, int shared, int bm,
                                                  Sorted S) {
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
  if (e >= experts) {
    quant_block(x, stride, n_blocks, kb, out, (blockIdx.x - experts) * (T / 16) + tid / 16, tid % 16);
    return;
  }
  __shared__ int hist[MAX_EXPERTS];
  __shared__ int part[WV][3], found[WV];
  const int picks = tokens * k, sh_tiles = shared ? (tokens + bm - 1) / bm : 0;
  for (int i = tid; i < experts; i += T) hist[i] = 0;
  __syncthreads();
  for (int i = tid; i < picks; i += T) {
    const int id = ids[i];
    if (id >= 0 && id < experts) atomicAdd(&hist[id], 1);
    else if (e == 0) S.place[i] = -1;
  }
  __syncthreads();
  // places and tiles of the experts before this one, and (for the list's length) all tiles
  int before = 0, tiles = 0, all = 0;
  for (int j = tid; j < experts; j += T) {
    const int t = (hist[j] + bm - 1) / bm;
    all += t;
    if (j < e) before += hist[j], tiles += t;
  }
  before = wave_sum_i(before), tiles = wave_sum_i(tiles), all = wave_sum_i(all);
  if (lane == 0) part[wave][0] = before, part[wave][1] = tiles, part[wave][2] = all;
  __syncthreads();
  before = 0, tiles = sh_tiles, all = sh_tiles;
#pragma unroll
  for (int w = 0; w < WV; ++w) before += part[w][0], tiles += part[w][1], all += part[w][2];
  const int count = hist[e];
  for (int j = tid; j < (count + bm - 1) / bm; j += T) S.tiles[tiles + j] = Tile{e, before + j * bm, min(bm, count - j * bm), 0};
  if (e == 0 && tid == 0) *S.n_tiles = all;
  if (shared) {
    for (int t = e * T + tid; t < tokens; t += experts * T) S.token[picks + t] = t;
    for (int j = e * T + tid; j < sh_tiles; j += experts * T)
      S.tiles[j] = Tile{experts, picks + j * bm, min(bm, tokens - j * bm), 0};
  }
  if (count == 0) return;
  const int share = ((picks + WV - 1) / WV + WAVE - 1) / WAVE * WAVE;  // whole waves of picks
  const int i0 = min(picks, wave * share), i1 = min(picks, i0 + share);
  int mine = 0;
  for (int i = i0; i < i1; i += WAVE) mine += __popcll(__ballot(i + lane < i1 && ids[min(i + lane, i1 - 1)] == e));
  if (lane == 0) found[wave] = mine;
  __syncthreads();
  int at = before;
#pragma unroll
  for (int w = 0; w < WV; ++w) at += w < wave ? found[w] : 0;
  for (int i = i0; i < i1; i += WAVE) {
    const bool hit = i + lane < i1 && ids[min(i + lane, i1 - 1)] == e;
    const uint64_t bal = __ballot(hit);
    if (hit) {
      const int p = at + __popcll(bal & ((1ull << lane) - 1ull));
      S.place[i + lane] = p;
      S.token[p] = (i + lane) / k;
    }
    at += __popcll(bal);
  }
}

// out[t] = residual[t] + shared part + sum_j weight[t, j] part[place of pick j], in the
// picks' own order (f32 sums, one rounding to bf16). A thread sums 8 columns.
__global__ __launch_bounds__(128) void k_back(Experts a) {
  const int t = blockIdx.x, c = (blockIdx.y * 128 + threadIdx.x) * 8;
  if (c >= a.hidden) return;
  float y[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = 0.f;
  if (a.shared) load8(a.part + (size_t)(a.picks + t) * a.hidden + c, y);
  for (int j = 0; j < a.picks_each; ++j) {
    const int p = a.sorted.place[(size_t)t * a.picks_each + j];
    if (p < 0) continue;
    const float w = a.weights[(size_t)t * a.picks_each + j];
    load8(a.part + (size_t)p * a.hidden + c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = fmaf(w, v[i], y[i]);
  }
  if (a.residual) {
    load8(static_cast<const uint16_t*>(a.residual) + (int64_t)t * a.residual_stride + c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] += v[i];
  }
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + (int64_t)t * a.out_stride + c) =
      u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
}

}  // namespace

hipError_t quant_rows(const void* x, bool f32, int64_t stride, int64_t rows, int k, const Rows& out, hipStream_t st) {
  const uint32_t n = (uint32_t)(rows * (k / BLK)), grid = (n + T / 16 - 1) / (T / 16);
  if (f32)
    k_quant_rows<<<grid, T, 0, st>>>(static_cast<const float*>(x), stride, n, k / BLK, out);
  else
    k_quant_rows<<<grid, T, 0, st>>>(static_cast<const uint16_t*>(x), stride, n, k / BLK, out);
  return hipGetLastError();
}

hipError_t sort_quant(const void* x, int64_t stride, int64_t tokens, int k, const Rows& out, const int* ids, int picks_each,
                      int experts, bool shared, int bm, const Sorted& sorted, hipStream_t st) {
  const uint32_t n = (uint32_t)(tokens * (k / BLK)), grid = experts + (n + T / 16 - 1) / (T / 16);
  k_sort_quant<<<grid, T, 0, st>>>(static_cast<const uint16_t*>(x), stride, n, k / BLK, out, ids, (int)tokens, picks_each,
                                   experts, shared, bm, sorted);
  return hipGetLastError();
}

hipError_t experts_back(const Experts& a, hipStream_t st) {
  k_back<<<dim3((uint32_t)a.tokens, (a.hidden / 8 + 127) / 128), 128, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
