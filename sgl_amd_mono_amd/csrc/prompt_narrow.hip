// FP8 block products over tiles of at most 64 rows: y[m, n] = sum over blocks b of 128
// columns of sx[m, b] sw[n / 128, b] (xq[m, b] . wq[n, b]).
//
// A workgroup holds 16 (or 16 gate and 16 up) weight rows and up to 64 rows of x; its 8
// waves take the blocks of K in turn, each multiplies E4M3 codes on the scaled MFMA (unit
// scales) and adds the f32 partial times sx sw to its sums, and the waves' sums meet in
// LDS in wave order. The weights are the MFMA's A operand: a lane then holds 4 consecutive
// outputs of one row, and one sx.
#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 512, WV = T / WAVE, BM = 64;

struct Narrow {
  const uint8_t* xq;
  const float* xs;
  int xs_ld;
  const uint8_t* w;
  const float* s;
  int n, kb;           // weight rows of one matrix, blocks of K
  int64_t rows;        // dense: rows of x
  void* out;
  int64_t out_ld;
  const Tile* tiles;   // experts: the tile list and its length
  const int* token;
  int half;            // up: gate rows (the up rows follow)
};

enum Mode { DENSE_BF16, DENSE_F32, UP };

MONO_DEV i32x8 ld_pair(const uint8_t* p, size_t far) {
  const i32x4 a = *reinterpret_cast<const i32x4*>(p), b = *reinterpret_cast<const i32x4*>(p + far);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The wave's share of K (blocks wave, wave + 8, ..) of NT x MT tiles of 16 x 16.
template <bool F32, int NT, int MT>
MONO_DEV void accumulate(const uint8_t* const (&wp)[NT], const float* const (&sp)[NT], const uint8_t* const (&xp)[MT],
                         const float* const (&xsp)[MT], int xs_ld, int kb, int wave, f32x4 (&acc)[NT][MT]) {
  constexpr int U = MT == 4 ? 2 : 4;
  for (int b0 = wave; b0 < kb; b0 += WV * U) {
    i32x8 wv[U][NT], xv[U][MT];
    float sw[U][NT], sx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + WV * u < kb ? b0 + WV * u : b0;  // past the end: the first again, scaled by zero
      const float on = b0 + WV * u < kb ? 1.f : 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        wv[u][i] = ld_pair(wp[i] + (size_t)b * 2048, 1024);
        sw[u][i] = sp[i][b] * on;
      }
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        xv[u][j] = ld_pair(xp[j] + (size_t)b * BLK, 64);
        sx[u][j] = xsp[j][(size_t)b * xs_ld];
      }
    }
    #pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const f32x4 p = mfma_block<F32>(wv[u][i], xv[u][j]);
          const float c = sw[u][i] * sx[u][j];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(p[r], c, acc[i][j][r]);
        }
  }
}

template <int MODE, int NT, int MT>
MONO_DEV void narrow_tile(const Narrow& a, f32x4* red, const uint8_t* w, const float* s, int n0, int64_t first, int count) {
  const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
  const uint8_t *wp[NT], *xp[MT];
  const float *sp[NT], *xsp[MT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int n = n0 + i * a.half;
    wp[i] = w + (size_t)n * a.kb * BLK + 16 * lane;
    sp[i] = s + (size_t)(n / BLK) * a.kb;
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t m = first + min(16 * j + lane % 16, count - 1);  // rows past the tile: its last again, not stored
    const int64_t row = MODE == UP ? a.token[m] : m;
    xp[j] = a.xq + (size_t)row * a.kb * BLK + 16 * (lane / 16);
    xsp[j] = a.xs + row;
  }
  f32x4 acc[NT][MT] = {};
  accumulate<MODE == DENSE_F32, NT, MT>(wp, sp, xp, xsp, a.xs_ld, a.kb, wave, acc);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[((wave * NT + i) * MT + j) * WAVE + lane] = acc[i][j];
  __syncthreads();
  if (tid >= MT * WAVE) return;  // wave j stores m-tile j
  f32x4 y[NT] = {};
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int v = 0; v < WV; ++v) y[i] += red[((v * NT + i) * MT + wave) * WAVE + lane];
  const int m = 16 * wave + lane % 16;
  if (m >= count) return;
  const size_t at = (size_t)(first + m) * a.out_ld + n0 + 4 * (lane / 16);
  if (MODE == UP) {
#pragma unroll
    for (int r = 0; r < 4; ++r) y[0][r] = y[0][r] / (1.0f + expf(-y[0][r])) * y[NT - 1][r];
  }
  if (MODE == DENSE_BF16)
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at) = u32x2{pack_bf16x2(y[0][0], y[0][1]), pack_bf16x2(y[0][2], y[0][3])};
  else
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = y[0];
}

template <int MODE>
__global__ __launch_bounds__(T) void k_narrow(Narrow a) {
  constexpr int NT = MODE == UP ? 2 : 1;
  __shared__ f32x4 red[WV * NT * 4 * WAVE];
  const int n0 = blockIdx.x * 16;
  int64_t first = (int64_t)blockIdx.y * BM;
  int count = MODE == UP ? 0 : (int)min((int64_t)BM, a.rows - first);
  const uint8_t* w = a.w;
  const float* s = a.s;
  if (MODE == UP) {
    const Tile t = a.tiles[blockIdx.y];
    first = t.first;
    count = t.count;
    if (count == 0) return;
    w += (size_t)t.expert * a.n * a.kb * BLK;
    s += (size_t)t.expert * ((a.n + BLK - 1) / BLK) * a.kb;
  }
  if (count <= 16)
    narrow_tile<MODE, NT, 1>(a, red, w, s, n0, first, count);
  else if (count <= 32)
    narrow_tile<MODE, NT, 2>(a, red, w, s, n0, first, count);
  else
    narrow_tile<MODE, NT, 4>(a, red, w, s, n0, first, count);
}

// The experts' down products: K is the mids' few blocks, so the waves share out the weight
// rows (64 each) and not K, and each ends with whole sums.
constexpr int DT = 256, DN = 256, DW = DN / (DT / WAVE) / 16;
static_assert(16 * DW == PART, "a wave's weight rows are a block of Parts");

template <int MT>
MONO_DEV void down_tile(const Experts& a, const Tile& t, int n0, uint8_t* buf) {
  constexpr int U = MT == 1 ? 4 : MT == 2 ? 2 : 1;
  const int lane = threadIdx.x % WAVE, kb = a.inter / BLK;
  const uint8_t* w = a.w2 + ((size_t)t.expert * a.hidden + n0) * a.inter;
  const float* s = a.s2 + ((size_t)t.expert * (a.hidden / BLK) + n0 / BLK) * kb;
  const uint8_t* xp[MT];
  const float* xsp[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = t.first + min(16 * j + lane % 16, t.count - 1);
    xp[j] = a.mid_q.q + (size_t)m * a.inter + 16 * (lane / 16);
    xsp[j] = a.mid_q.s + m;
  }
  f32x4 acc[MT][DW] = {};
  for (int b0 = 0; b0 < kb; b0 += U) {
    i32x8 wv[U][DW], xv[U][MT];
    float c[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = min(b0 + u, kb - 1);
      const float sw = b0 + u < kb ? s[b] : 0.f;  // past the end: the last block again, scaled by zero
#pragma unroll
      for (int i = 0; i < DW; ++i) wv[u][i] = ld_pair(w + (size_t)i * 16 * a.inter + (size_t)b * 2048 + 16 * lane, 1024);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        xv[u][j] = ld_pair(xp[j] + (size_t)b * BLK, 64);
        c[u][j] = xsp[j][(size_t)b * a.mid_q.ld] * sw;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < DW; ++i) {
          const f32x4 p = mfma_block<false>(wv[u][i], xv[u][j]);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(p[r], c[u][j], acc[j][i][r]);
        }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    store_part(buf, a.part, t.first + 16 * j, t.count - 16 * j, n0, acc[j]);
  }
}

__global__ __launch_bounds__(DT) void k_down(Experts a) {
  __shared__ uint8_t bufs[DT / WAVE][2048];
  uint8_t* buf = bufs[threadIdx.x / WAVE];
  const Tile t = a.sorted.tiles[blockIdx.y];
  const int n0 = blockIdx.x * DN + threadIdx.x / WAVE * PART;
  if (t.count == 0 || n0 >= a.hidden) return;
  if (t.count <= 16)
    down_tile<1>(a, t, n0, buf);
  else if (t.count <= 32)
    down_tile<2>(a, t, n0, buf);
  else
    down_tile<4>(a, t, n0, buf);
}

}  // namespace

hipError_t product(const Rows& x, int64_t rows, const void* w, const float* s, int n, int k, void* out, bool f32,
                   int64_t out_stride, hipStream_t st) {
  Narrow a{x.q, x.s, x.ld, static_cast<const uint8_t*>(w), s, n, k / BLK, rows, out, out_stride, nullptr, nullptr, 0};
  const dim3 grid(n / 16, (uint32_t)((rows + BM - 1) / BM));
  if (f32)
    k_narrow<DENSE_F32><<<grid, T, 0, st>>>(a);
  else
    k_narrow<DENSE_BF16><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t experts_up(const Experts& e, hipStream_t st) {
  Narrow a{e.x.q, e.x.s, e.x.ld, e.w13, e.s13, 2 * e.inter, e.hidden / BLK, 0, e.mid, e.inter,
           e.sorted.tiles, e.sorted.token, e.inter};
  k_narrow<UP><<<dim3(e.inter / 16, e.tiles), T, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t experts_down(const Experts& e, hipStream_t st) {
  k_down<<<dim3((e.hidden + DN - 1) / DN, e.tiles), DT, 0, st>>>(e);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
