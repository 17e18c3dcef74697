// FP8 block products over tiles of at most 64 rows: y[m, n] = sum over blocks b of 128
// columns of sx[m, b] sw[n / 128, b] (xq[m, b] . wq[n, b]).
//
// The weights' bytes bound these: every one is read once for a few rows. A workgroup holds
// 16 (or 16 gate and 16 up) weight rows and up to 64 rows of x; its 8 waves (4 for the
// experts' up products) take the blocks of K in turn, so that together they read 16 KB runs
// of each 16 weight rows, each multiplies E4M3 codes on the MFMA and adds the f32 partial
// times sx sw to its sums, and the waves' sums meet in LDS in wave order. The weights are the
// MFMA's A operand: a lane then holds 4 consecutive outputs of one row, and one sx. The rows
// come from L2 straight into registers: against the weights they are few.
//
// Measured (256 experts of 7168 x 512, 8 picks a token): up products of 61 tokens 196 us, 6.1
// TB/s of the 162 experts that they pick, where a kernel that only reads has 6.4 (8 waves, of
// which a CU's registers hold one workgroup, 213); their down products 104 us, 5.7 TB/s (496
// us with K shared out among the waves, which leaves each wave half a block of its own). One
// token's up products take 15 us, 4.5 TB/s (8 waves 17.5: its 288 workgroups were one round
// over the CUs and an eighth of another); in all 34 us a call for 37, 8 tokens 122 for 128,
// 128 tokens 398 for 425. Tiles of 16 rows alone need half the registers, and four workgroups
// a CU were slower from 3 tokens on (8 tokens 127). Mids wider than LDS holds, rounded by a
// launch of their own (5 us): down products of 64 tokens by 65 experts of 7168 x 1024 95 us,
// of 7168 x 2048 189 us, 5 TB/s both; the up products 160 and 320 us, 6 TB/s.
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
  float* part;         // dense, K shared out: f32 [splits, rows, n] instead of out
  int splits;
};

enum Mode { DENSE_BF16, DENSE_F32, UP };

MONO_DEV i32x8 ld_pair(const uint8_t* p, size_t far) {
  const i32x4 a = *reinterpret_cast<const i32x4*>(p), b = *reinterpret_cast<const i32x4*>(p + far);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// The wave's share of K (blocks kb0 + wave, + WV, .. below kb) of NT x MT tiles of 16 x 16.
template <bool F32, int WV, int NT, int MT>
MONO_DEV void accumulate(const uint8_t* const (&wp)[NT], const float* const (&sp)[NT], const uint8_t* const (&xp)[MT],
                         const float* const (&xsp)[MT], int xs_ld, int kb0, int kb, int wave, f32x4 (&acc)[NT][MT]) {
  constexpr int U = MT == 4 ? 2 : NT == 2 ? 3 : 4;
  for (int b0 = kb0 + wave; b0 < kb; b0 += WV * U) {
    i32x8 wv[U][NT], xv[U][MT];
    float sw[U][NT], sx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = b0 + WV * u < kb;
      const int b = in ? b0 + WV * u : b0;  // past the end: the first again, its scale zero (whatever its own is)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        wv[u][i] = ld_pair(wp[i] + (size_t)b * 2048, 1024);
        sw[u][i] = in ? sp[i][b] : 0.f;
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

// A few rows (at most 16, and FEW_BYTES of codes): every workgroup rounds all of them into
// LDS itself while its weights are on their way, which saves the launch that rounds them
// for all (1 x 2112 x 7168: 5.5 us for 2.3 + 5.2, and 8.7 us a call for 11.5).
template <bool F32>
__global__ __launch_bounds__(T) void k_few(const uint16_t* x, int64_t stride, int rows, const uint8_t* w, const float* s,
                                           int kb, void* out, int64_t out_ld) {
  constexpr int U = 8;
  __shared__ __align__(16) uint8_t xq[FEW_BYTES + 16 * 16];  // rows K + 16 bytes apart: 16 rows' pieces meet few banks
  __shared__ float xs[FEW_BYTES / BLK];
  __shared__ f32x4 red[WV][WAVE];
  const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE, n0 = blockIdx.x * 16, ld = kb * BLK + 16;
  const uint8_t* wp = w + (size_t)n0 * kb * BLK + 16 * lane;
  const float* sp = s + (size_t)(n0 / BLK) * kb;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int b0 = wave; b0 < kb + wave; b0 += WV * U) {  // (a wave without blocks takes the first round, for its barrier)
    i32x8 wv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) wv[u] = ld_pair(wp + (size_t)min(b0 + WV * u, kb - 1) * 2048, 1024);
    if (b0 == wave) {
      for (int b = tid / 16; b < rows * kb; b += T / 16) {
        const int row = b / kb, c = b % kb;
        float v[8], scale;
        load8(x + (int64_t)row * stride + c * BLK + 8 * (tid % 16), v);
        const u32x2 q = quant8(v, scale);
        *reinterpret_cast<u32x2*>(xq + row * ld + c * BLK + 8 * (tid % 16)) = q;
        if (tid % 16 == 0) xs[b] = scale;
      }
      __syncthreads();
    }
    const int row = min(lane % 16, rows - 1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + WV * u;
      if (b >= kb) break;
      const i32x8 xv = ld_pair(xq + row * ld + b * BLK + 16 * (lane / 16), 64);
      const f32x4 p = mfma_block<F32>(wv[u], xv);
      const float c = sp[b] * xs[row * kb + b];
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = fmaf(p[r], c, acc[r]);
    }
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave || lane % 16 >= rows) return;
  f32x4 y = red[0][lane];
#pragma unroll
  for (int v = 1; v < WV; ++v) y += red[v][lane];
  const size_t at = (size_t)(lane % 16) * out_ld + n0 + 4 * (lane / 16);
  if (F32)
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + at) = y;
  else
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + at) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
}

template <int MODE, int WV, int NT, int MT>
MONO_DEV void narrow_tile(const Narrow& a, f32x4* red, const uint8_t* w, const float* s, int n0, int64_t first, int count,
                          int kb0, int kb1) {
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
  accumulate<MODE != DENSE_BF16, WV, NT, MT>(wp, sp, xp, xsp, a.xs_ld, kb0, kb1, wave, acc);
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
  if (MODE == UP) {  // (the hardware's exponential and reciprocal: 1e-6 off for gates down to -16)
#pragma unroll
    for (int r = 0; r < 4; ++r) y[0][r] = silu(y[0][r]) * y[NT - 1][r];
  }
  if (MODE != UP && a.splits > 1)
    *reinterpret_cast<f32x4*>(a.part + ((size_t)blockIdx.z * a.rows + first + m) * a.n + n0 + 4 * (lane / 16)) = y[0];
  else if (MODE == DENSE_BF16)
    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at) = u32x2{pack_bf16x2(y[0][0], y[0][1]), pack_bf16x2(y[0][2], y[0][3])};
  else
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = y[0];
}

template <int MODE, int WV>
__global__ __launch_bounds__(WV * WAVE, 2) void k_narrow(Narrow a) {
  constexpr int NT = MODE == UP ? 2 : 1;
  __shared__ f32x4 red[WV * NT * 4 * WAVE];
  const int n0 = blockIdx.x * 16;
  int64_t first = (int64_t)blockIdx.y * BM;
  int count = MODE == UP ? 0 : (int)min((int64_t)BM, a.rows - first);
  const uint8_t* w = a.w;
  const float* s = a.s;
  const int kb0 = MODE == UP ? 0 : (int)blockIdx.z * a.kb / a.splits, kb1 = MODE == UP ? a.kb : ((int)blockIdx.z + 1) * a.kb / a.splits;
  if (MODE == UP) {
    const Tile t = a.tiles[blockIdx.y];
    first = t.first;
    count = t.count;
    if (count == 0) return;
    w += (size_t)t.expert * a.n * a.kb * BLK;
    s += (size_t)t.expert * ((a.n + BLK - 1) / BLK) * a.kb;
  }
  if (count <= 16)
    narrow_tile<MODE, WV, NT, 1>(a, red, w, s, n0, first, count, kb0, kb1);
  else if (count <= 32)
    narrow_tile<MODE, WV, NT, 2>(a, red, w, s, n0, first, count, kb0, kb1);
  else
    narrow_tile<MODE, WV, NT, 4>(a, red, w, s, n0, first, count, kb0, kb1);
}

// The experts' down products: K is the mids' few blocks, so the waves share out the weight
// rows (64 each) and not K, and each ends with whole sums.
constexpr int DT = 256, DN = 256, DW = DN / (DT / WAVE) / 16;
static_assert(16 * DW == PART, "a wave's weight rows are a block of Parts");

// (DM * BLK mids a row fit in LDS: the workgroup rounds its tile's mids itself, while its
// first weights are on their way; wider mids have been rounded by a launch of their own.)
constexpr int DM = 4, DLD = DM * BLK + 16;
struct Mids {
  __align__(16) uint8_t q[BM][DLD];
  float s[BM][DM];
};

template <int MT, bool HERE>
MONO_DEV void down_tile(const Experts& a, const Tile& t, int n0, uint8_t* buf, Mids& mids) {
  constexpr int U = HERE ? (MT == 1 ? DM : 2) : MT == 1 ? 4 : MT == 2 ? 2 : 1;
  const int lane = threadIdx.x % WAVE, kb = a.inter / BLK;
  const bool idle = n0 >= a.hidden;  // (the last workgroup's waves past the matrix: they help round)
  n0 = min(n0, a.hidden - PART);
  const uint8_t* w = a.w2 + ((size_t)t.expert * a.hidden + n0) * a.inter;
  const float* s = a.s2 + ((size_t)t.expert * (a.hidden / BLK) + n0 / BLK) * kb;
  const uint8_t* xp[MT];
  const float* xsp[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = t.first + min(16 * j + lane % 16, t.count - 1);
    xp[j] = HERE ? mids.q[m - t.first] + 16 * (lane / 16) : a.mid_q.q + (size_t)m * a.inter + 16 * (lane / 16);
    xsp[j] = HERE ? mids.s[m - t.first] : a.mid_q.s + m;
  }
  f32x4 acc[MT][DW] = {};
  for (int b0 = 0; b0 < kb; b0 += U) {
    i32x8 wv[U][DW];
    float sw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = min(b0 + u, kb - 1);
      sw[u] = b0 + u < kb ? s[b] : 0.f;  // past the end: the last block again, scaled by zero
#pragma unroll
      for (int i = 0; i < DW; ++i) wv[u][i] = ld_pair(w + (size_t)i * 16 * a.inter + (size_t)b * 2048 + 16 * lane, 1024);
    }
    if (HERE && b0 == 0) {
      for (int b = threadIdx.x / 16; b < t.count * kb; b += DT / 16) {
        const int row = b / kb, c = b % kb, sub = threadIdx.x % 16;
        float v[8], scale;
        load8(a.mid + (size_t)(t.first + row) * a.inter + c * BLK + 8 * sub, v);
        const u32x2 q = quant8(v, scale);
        *reinterpret_cast<u32x2*>(&mids.q[row][c * BLK + 8 * sub]) = q;
        if (sub == 0) mids.s[row][c] = scale;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int b = min(b0 + u, kb - 1);
        const i32x8 xv = ld_pair(xp[j] + (size_t)b * BLK, 64);
        const float c = xsp[j][HERE ? (size_t)b : (size_t)b * a.mid_q.ld] * sw[u];
#pragma unroll
        for (int i = 0; i < DW; ++i) {
          const f32x4 p = mfma_block<false>(wv[u][i], xv);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(p[r], c, acc[j][i][r]);
        }
      }
  }
  if (idle) return;
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    store_part(buf, a.part, t.first + 16 * j, t.count - 16 * j, n0, acc[j]);
  }
}

template <bool HERE>
__global__ __launch_bounds__(DT) void k_down(Experts a) {
  __shared__ uint8_t bufs[DT / WAVE][2048];
  __shared__ Mids mids;
  const Tile t = a.sorted.tiles[blockIdx.y];
  if (t.count == 0) return;
  uint8_t* buf = bufs[threadIdx.x / WAVE];
  const int n0 = blockIdx.x * DN + threadIdx.x / WAVE * PART;
  if (t.count <= 16)
    down_tile<1, HERE>(a, t, n0, buf, mids);
  else if (t.count <= 32)
    down_tile<2, HERE>(a, t, n0, buf, mids);
  else
    down_tile<4, HERE>(a, t, n0, buf, mids);
}

}  // namespace

hipError_t few_product(const Product& a, hipStream_t st) {
  const uint16_t* x = static_cast<const uint16_t*>(a.x);
  if (a.f32)
    k_few<true><<<a.n / 16, T, 0, st>>>(x, a.x_stride, (int)a.rows, a.w, a.s, a.k / BLK, a.out, a.out_stride);
  else
    k_few<false><<<a.n / 16, T, 0, st>>>(x, a.x_stride, (int)a.rows, a.w, a.s, a.k / BLK, a.out, a.out_stride);
  return hipGetLastError();
}

hipError_t narrow_product(const Product& p, hipStream_t st) {
  Narrow a{p.q.q, p.q.s, p.q.ld, p.w, p.s, p.n, p.k / BLK, p.rows, p.out, p.out_stride, nullptr, nullptr, 0, p.part, p.plan.splits};
  const dim3 grid(p.n / 16, (uint32_t)((p.rows + BM - 1) / BM), p.plan.splits);
  if (p.f32)
    k_narrow<DENSE_F32, WV><<<grid, T, 0, st>>>(a);
  else
    k_narrow<DENSE_BF16, WV><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t experts_up(const Experts& e, hipStream_t st) {
  Narrow a{e.x.q, e.x.s, e.x.ld, e.w13, e.s13, 2 * e.inter, e.hidden / BLK, 0, e.mid, e.inter,
           e.sorted.tiles, e.sorted.token, e.inter};
  k_narrow<UP, 4><<<dim3(e.inter / 16, e.tiles), 4 * WAVE, 0, st>>>(a);
  return hipGetLastError();
}

hipError_t experts_down(const Experts& e, hipStream_t st) {
  const dim3 grid((e.hidden + DN - 1) / DN, e.tiles);
  if (e.inter <= DM * BLK) {
    k_down<true><<<grid, DT, 0, st>>>(e);
    return hipGetLastError();
  }
  const int64_t places = e.picks + (e.shared ? e.tokens : 0);
  if (hipError_t r = quant_rows(e.mid, true, e.inter, places, e.inter, e.mid_q, st)) return r;
  k_down<false><<<grid, DT, 0, st>>>(e);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
