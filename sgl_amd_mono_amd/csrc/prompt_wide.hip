// FP8 block products over wide tiles: 256 weight rows by 128 (or 64) rows of x a workgroup,
// two workgroups a CU.
//
//   y[m, n] = sum over blocks b of 128 columns of sx[m, b] sw[n / 128, b] (xq[m, b] . wq[n, b])
//
// Four waves hold 64 weight rows x 128 rows of x each: 4 x 8 tiles of 16 x 16, 128
// accumulators a lane. The weights lie in memory as the MFMA wants them, so a wave loads
// its own straight into registers, a block of K ahead; the rows of x are shared by the
// waves and come through LDS by DMA (global_load_lds), also a block ahead. With waves side
// by side along the weight rows, LDS feeds 16 KB a wave and block of K (1024 cycles of
// MFMA), half of what it can, and the weights pass no LDS at all.
//
// Each block's partial is scaled in f32: 4 FMAs an MFMA, half the vector unit's time under
// the matrix unit's. Issued right behind their MFMA they wait for it (two waves a SIMD, all
// in registers: 4.2 PFLOP/s one MFMA later, 4.9 two later).
//
// Measured: 8192 x 7168 x 4096 209 us, 2.3 PFLOP/s (a library product of the same codes
// with one scale a tensor: 195 us); 1500 x 2112 x 7168 34 us; the up products of 8192 tokens
// x 9 experts of 7168 x 512 739 us, 1.5 PFLOP/s, the down products 519, 1.0. Mids wider than LDS
// holds whole (1500 tokens x 9 of 65 experts): 7168 x 1024 up 353, down 206 us, 7168 x 2048
// up 616, down 345, 1.0 to 1.3 PFLOP/s. f32 outputs, whose codes every wave widens: 1500 x 2112
// x 7168 68 us, 8192 x 2112 x 7168 330, 0.7 PFLOP/s. The MFMAs run for 57 % of the
// cycles of the first (45 % of the up products'), at a clock that the work's power holds at
// 1.9 (1.6) GHz. With every load a cache hit the first takes 208 us: what is left is the
// vector memory path's 48 KB a tile and block, the barrier a block and the last round of
// workgroups. Steps that brought it there, us: 64 x 64 a wave through narrow tiles 1932; this
// split 340; MFMA ahead of the scaling, fragments a step ahead 245; loads spread among the
// MFMAs and LDS pieces without bank conflicts 227; the fragment's reads behind an MFMA 214.
// Tried and left: eight waves over 256 x 256 behind one barrier 251 (a third less from L2, and
// no second workgroup to fill its waits); tiles of 256 x 256 in four waves of 452 registers 320
// (the sums then lie where the vector unit cannot add to them); half tiles for the last round
// 229.
#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int BN = 256, TN = 64, NT = TN / 16, WN = BN / TN, T = WN * WAVE;

struct Wide {
  const uint8_t* xq;
  const float* xs;
  int xs_ld;
  const uint8_t* w;
  const float* s;
  int n, kb;           // weight rows of a matrix, blocks of K
  int64_t rows;        // dense: rows of x
  void* out;
  int64_t out_ld;
  const Tile* tiles;   // experts: the tile list, the token of each place
  const int* token;
  int half;            // up: gate rows (the up rows follow)
  float* mid_s;        // up: the mids' scales [inter / 128, mid_ld]
  int mid_ld;
  Parts part;          // down
  int tiles_m, tiles_n;
  float* split;        // dense, K shared out: f32 [splits, rows, n] instead of out
  int splits;
  int groups;          // resident down: workgroups that share out a tile's weight columns
};

enum Mode { DENSE_BF16, DENSE_F32, UP, DOWN };
static_assert(TN == PART, "a wave's weight rows are a block of Parts");

template <int MT>
struct Stage {
  uint8_t x[16 * MT * BLK];
  float s[MT == 4 ? WN : 1][16 * MT];  // (64 rows: a copy a wave, so that every wave issues the same loads)
};

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;
MONO_DEV void dma16(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((gvoid*)g, (lvoid*)l, 16, 0, 0);
}
MONO_DEV void dma4(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((gvoid*)g, (lvoid*)l, 4, 0, 0);
}

template <int MODE, int MT>
struct WideTile {
  static constexpr int XD = MT / 4;  // groups of 16 rows of x that a wave brings
  const Wide& a;
  const int lane, wave;
  int kb0 = 0, kbs;       // the tile's blocks of K: the first, how many
  const uint8_t* wp[NT];  // the weight tiles (uniform)
  const float* sw[2];     // weight scales in LDS by block of K: of weight tiles 0, 1 and 2, 3
  const uint8_t* xp[XD];  // the lane's rows of x for the DMA
  const float* xsp;       // the lane's row of the scales for the DMA
  f32x4 acc[NT][MT] = {};

  MONO_DEV WideTile(const Wide& a_) : a(a_), lane(threadIdx.x % WAVE), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / WAVE)), kbs(a_.kb) {}

  struct Ahead {
    i32x8 w[NT];
  };

  // The loads of block kb in the order they go out: part 0 the rows' DMA and the scales, part
  // 1 + i weight tile i.
  MONO_DEV void issue(int kb, Stage<MT>& st, Ahead& n, int part) {
    kb += kb0;
    if (part == 0) {
#pragma unroll
      for (int h = 0; h < XD; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) dma16(xp[h] + (size_t)kb * BLK + 64 * q, &st.x[(XD * wave + h) * 2048 + 1024 * q]);
      if (MT == 4)
        dma4(xsp + (size_t)kb * a.xs_ld, st.s[wave]);
      else if (wave < MT / 4)
        dma4(xsp + (size_t)kb * a.xs_ld, &st.s[0][wave * WAVE]);
    } else if (part <= NT) {
      const uint8_t* at = wp[part - 1] + (size_t)kb * 2048;
      const i32x4 lo = *reinterpret_cast<const i32x4*>(at + 16 * (uint32_t)lane);
      const i32x4 hi = *reinterpret_cast<const i32x4*>(at + 16 * (uint32_t)lane + 1024);
      n.w[part - 1] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  MONO_DEV void issue(int kb, Stage<MT>& st, Ahead& n) {
#pragma unroll
    for (int part = 0; part <= NT; ++part) issue(kb, st, n, part);
  }

  // One block's MFMAs, with `ahead(part)` (the loads of a later block) spread among them.
  // FIRST: the sums begin with this block's. (The weight scales come from LDS like the rows':
  // a scalar load among the LDS reads would make each wait for a fragment one for all of
  // them, since the two return in no common order.)
  template <bool FIRST = false, class F>
  MONO_DEV void compute(const Stage<MT>& st, const Ahead& n, int kb, F ahead) {
    const int r = lane % 16, g = lane / 16;
    const uint8_t* x = st.x + r * 64 + ((g ^ (r >> 1 & 3)) * 16);
    const float* xs = st.s[MT == 4 ? wave : 0] + r;
    i32x8 xv[2];  // a fragment ahead: its LDS latency lies under the MFMAs of the one before
    float sx[2];
    const auto load = [&](int j) {
      const i32x4 lo = *reinterpret_cast<const i32x4*>(x + j * 2048), hi = *reinterpret_cast<const i32x4*>(x + j * 2048 + 1024);
      xv[j % 2] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      sx[j % 2] = xs[16 * j];
    };
    load(0);
    const float ws[2] = {sw[0][kb], sw[1][kb]};
    // each MFMA's partial is scaled while the LAG after it run: neither waits for the other
    constexpr int LAG = MT == 4 ? 2 : 1;  // (128 rows have no registers for two: they spill)
    f32x4 p[LAG + 1];
    float c[2][2];
#pragma unroll
    for (int t = 0; t < MT * NT + LAG; ++t) {
      const int i = t % NT, j = t / NT, v = t - LAG;
      if (t < MT * NT) {
        // (behind the fragment's first MFMA, whose wait for LDS then finds nothing younger to wait for)
        if (i == 1 && j + 1 < MT) load(j + 1);
        p[t % (LAG + 1)] = mfma_block<MODE == DENSE_F32>(n.w[i], xv[j % 2]);
        if (i == 0) c[j % 2][0] = sx[j % 2] * ws[0], c[j % 2][1] = sx[j % 2] * ws[1];
        __builtin_amdgcn_sched_barrier(0);
      }
      if (v >= 0) {
        f32x4& to = acc[v % NT][v / NT];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float f = c[v / NT % 2][v % NT / 2];
          to[e] = FIRST ? p[v % (LAG + 1)][e] * f : fmaf(p[v % (LAG + 1)][e], f, to[e]);
        }
        // the sums stay here: moved behind the next barrier, they would hold 64 more registers
        asm volatile("" : "+v"(to));
      }
      if (t % 2 == 0 && t / 2 <= NT) ahead(t / 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  MONO_DEV void compute(const Stage<MT>& st, const Ahead& n, int kb) {
    compute(st, n, kb, [](int) {});
  }

  // The wave's loads but the last `LEFT` have come, and every wave's: a stage is whole.
  template <int LEFT>
  MONO_DEV void arrive() {
    __builtin_amdgcn_s_waitcnt((LEFT & 15) | 7 << 4 | (LEFT >> 4) << 14);  // (and lgkmcnt 0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // 128 rows: one block of K ahead. Past the end the last block comes again and is not used.
  MONO_DEV void run(Stage<MT>& s0, Stage<MT>& s1) {
    Ahead a0, a1;
    issue(0, s0, a0);
    int kb = 0;
    for (; kb + 1 < kbs; kb += 2) {
      arrive<0>();
      compute(s0, a0, kb, [&](int part) { issue(kb + 1, s1, a1, part); });
      arrive<0>();
      compute(s1, a1, kb + 1, [&](int part) { issue(min(kb + 2, kbs - 1), s0, a0, part); });
    }
    arrive<0>();
    if (kb < kbs) compute(s0, a0, kb);
  }

  // 64 rows: half the MFMA time a block to hide the same latency under, so two blocks ahead
  // (1500 x 2112 x 7168: one ahead 97 us, two 52; three no better than two).
  MONO_DEV void run(Stage<MT>& s0, Stage<MT>& s1, Stage<MT>& s2) {
    constexpr int EACH = 2 * XD + 1 + 2 * NT;  // a stage's loads, the same for every wave
    const int last = kbs - 1;
    Ahead a0, a1, a2;
    issue(0, s0, a0);
    __builtin_amdgcn_sched_barrier(0);  // (arrive counts loads: none of these goes out before the stage above)
    issue(min(1, last), s1, a1);
    int kb = 0;
    for (; kb + 2 < kbs; kb += 3) {
      arrive<EACH>();
      compute(s0, a0, kb, [&](int part) { issue(min(kb + 2, last), s2, a2, part); });
      arrive<EACH>();
      compute(s1, a1, kb + 1, [&](int part) { issue(min(kb + 3, last), s0, a0, part); });
      arrive<EACH>();
      compute(s2, a2, kb + 2, [&](int part) { issue(min(kb + 4, last), s1, a1, part); });
    }
    arrive<0>();
    if (kb < kbs) compute(s0, a0, kb);
    if (kb + 1 < kbs) compute(s1, a1, kb + 1);
  }
};

// Where a tile lies: its weight columns and scales, its rows of x.
struct Place {
  const uint8_t* w;
  const float* s;
  int64_t first;
  int count, tn, split;
};

template <int MODE, int MT, class... Stages>
MONO_DEV void tile(const Wide& a, const Place& at, float (*sw)[MAX_DIM / BLK], uint32_t (*top)[128], uint8_t* buf, Stages&... stages) {
  constexpr int BM = 16 * MT;
  const int64_t first = at.first;
  const int count = at.count, tn = at.tn;
  WideTile<MODE, MT> W(a);
  const int lane = W.lane, wn = W.wave;
  if (MODE != UP && MODE != DOWN && MT == 4) {
    W.kb0 = at.split * a.kb / a.splits;
    W.kbs = (at.split + 1) * a.kb / a.splits - W.kb0;
  }
  // the wave's weight tiles: 64 neighbouring rows, or (up) 32 gate rows and their up rows
  int row[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    row[i] = MODE == UP ? tn * (BN / 2) + wn * (TN / 2) + 16 * (i % 2) + (i / 2) * a.half : tn * BN + wn * TN + 16 * i;
    const int n = min(row[i], a.n - 16);  // past the matrix: its last rows again, not stored
    W.wp[i] = at.w + (size_t)n * a.kb * BLK;
  }
  // the tile's two rows of weight scales (gate and up; else of its two 128 weight rows)
  for (int i = threadIdx.x; i < 2 * W.kbs; i += T) {
    const int h = i >= W.kbs, kb = i - h * W.kbs;
    const int n = MODE == UP ? tn * (BN / 2) + h * a.half : min(tn * BN + h * BLK, a.n - 1);
    sw[h][kb] = at.s[(size_t)(n / BLK) * a.kb + W.kb0 + kb];
  }
  W.sw[0] = sw[MODE == UP ? 0 : wn / 2];
  W.sw[1] = sw[MODE == UP ? 1 : wn / 2];
#pragma unroll
  for (int h = 0; h < W.XD; ++h) {
    const int r = lane / 4;  // 16 rows x 64 bytes a DMA; the 16-byte pieces are swapped by row so that a
                             // fragment's reads (16 rows, one piece) meet every bank once
    const int64_t m = first + min((W.XD * W.wave + h) * 16 + r, count - 1);
    W.xp[h] = a.xq + (size_t)(MODE == UP ? a.token[m] : m) * a.kb * BLK + (((lane % 4) ^ (r >> 1 & 3)) * 16);
  }
  {
    const int64_t m = first + min((W.wave * WAVE + lane) % BM, count - 1);
    W.xsp = a.xs + (MODE == UP ? a.token[m] : m);
  }
  W.run(stages...);

  const int g = lane / 16;
  if (MODE == UP) {
    // mids, their block's scale over the four waves' 128 of them, codes
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          W.acc[i][j][e] = silu(W.acc[i][j][e]) * W.acc[i + 2][j][e];
          m = max(m, abs_bits(W.acc[i][j][e]));
        }
      m = groups_umax(m);
      if (g == 0) top[wn][16 * j + lane] = m;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int m = 16 * j + lane % 16;
      uint32_t t = top[0][m];
#pragma unroll
      for (int v = 1; v < WN; ++v) t = max(t, top[v][m]);
      const BlockScale bs = block_scale(t);
      if (m >= count) continue;
      uint8_t* q = static_cast<uint8_t*>(a.out) + (size_t)(first + m) * a.out_ld;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint32_t*>(q + row[i] + 4 * g) =
            fp8x4_pack(to_code_range(W.acc[i][j][0], bs), to_code_range(W.acc[i][j][1], bs),
                       to_code_range(W.acc[i][j][2], bs), to_code_range(W.acc[i][j][3], bs));
      if (wn == 0 && g == 0) a.mid_s[(size_t)tn * a.mid_ld + first + m] = bs.scale;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const f32x4 y[NT] = {W.acc[0][j], W.acc[1][j], W.acc[2][j], W.acc[3][j]};
    if (MODE == DOWN) {
      if (row[0] < a.n) store_part(buf, a.part, first + 16 * j, count - 16 * j, row[0], y);
    } else if (MT == 4 && a.splits > 1) {
      if (16 * j + lane % 16 < count)
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (row[i] < a.n)
            *reinterpret_cast<f32x4*>(a.split + ((size_t)at.split * a.rows + first + 16 * j + lane % 16) * a.n + row[i] + 4 * g) = y[i];
    } else if (MODE == DENSE_BF16) {
      u32x2 h[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) h[i] = u32x2{pack_bf16x2(y[i][0], y[i][1]), pack_bf16x2(y[i][2], y[i][3])};
      store_rows(buf, h, [&](int r, int c, u32x4 v) {
        if (16 * j + r < count && row[0] + c < a.n)
          *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.out) + (first + 16 * j + r) * a.out_ld + row[0] + c) = v;
      });
    } else if (16 * j + lane % 16 < count) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (row[i] < a.n)
          *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + (first + 16 * j + lane % 16) * a.out_ld + row[i] + 4 * g) = y[i];
    }
  }
}

// The experts' down products where K is short (a few blocks of mids): the tile's rows stay in
// LDS whole and each wave goes through its weight columns, 64 at a time, without a barrier;
// the next weights are on their way at every moment, also while sums are stored.
// 256 columns a turn, at most so many turns a workgroup (8192 tokens x 7168 columns: 2 turns 528
// us, 4 496, 7 501, 14 554; 1500 tokens 225, 231, 247, 281).
constexpr int TURNS = 4;

template <int KB, int MT>
MONO_DEV void resident_tile(const Wide& a, const Place& at, int group, float* sw, uint8_t* buf, Stage<MT> (&st)[KB]) {
  WideTile<DOWN, MT> W(a);
  const int lane = W.lane, r = lane / 4, last = a.kb - 1;
  using Ahead = typename WideTile<DOWN, MT>::Ahead;
#pragma unroll
  for (int h = 0; h < W.XD; ++h)
    W.xp[h] = a.xq + (size_t)(at.first + min((W.XD * W.wave + h) * 16 + r, at.count - 1)) * a.kb * BLK +
              (((lane % 4) ^ (r >> 1 & 3)) * 16);
  W.xsp = a.xs + at.first + min((W.wave * WAVE + lane) % (16 * MT), at.count - 1);
  // the scales of the columns to come, [a turn's two 128 columns][KB]; past K's end zero
  const int step = a.groups * BN;
  for (int i = threadIdx.x; i < (a.n + step - 1) / step * 2 * KB; i += T) {
    const int c = group * BN + i / (2 * KB) * step + i / KB % 2 * BLK, kb = i % KB;
    sw[i] = c < a.n && kb <= last ? at.s[(size_t)(c / BLK) * a.kb + kb] : 0.f;
  }
  Ahead n[2];
  // block kb of the 64 columns from col on; past K's end (an odd number of blocks) the last one
  const auto weights = [&](int col, int kb, Ahead& to, int part) {
    const int c = min(col, a.n - PART), b = min(kb, last);
    if (part && part <= NT) {
      const uint8_t* p = at.w + (size_t)(c + 16 * (part - 1)) * a.kb * BLK + (size_t)b * 2048;
      const i32x4 lo = *reinterpret_cast<const i32x4*>(p + 16 * (uint32_t)lane);
      const i32x4 hi = *reinterpret_cast<const i32x4*>(p + 16 * (uint32_t)lane + 1024);
      to.w[part - 1] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  int col = group * BN + W.wave * TN;
  W.sw[0] = W.sw[1] = sw + W.wave / 2 * KB;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) W.issue(min(kb, last), st[kb], n[0], 0);
#pragma unroll
  for (int part = 1; part <= NT; ++part) weights(col, 0, n[0], part);
  W.template arrive<0>();
  for (; col < a.n; col += step) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const auto ahead = [&](int part) {
        weights(kb + 1 < KB ? col : col + step, kb + 1 < KB ? kb + 1 : 0, n[(kb + 1) % 2], part);
      };
      if (kb == 0)
        W.template compute<true>(st[kb], n[kb % 2], kb, ahead);
      else
        W.compute(st[kb], n[kb % 2], kb, ahead);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const f32x4 y[NT] = {W.acc[0][j], W.acc[1][j], W.acc[2][j], W.acc[3][j]};
      store_part(buf, a.part, at.first + 16 * j, at.count - 16 * j, col, y);
    }
    W.sw[0] = W.sw[1] = W.sw[0] + 2 * KB;
  }
}

template <int KB>
__global__ __launch_bounds__(T, 2) void k_down_resident(Wide a) {
  static_assert(KB % 2 == 0, "the weights' two register sets alternate");
  __shared__ Stage<8> st[KB];
  __shared__ float sw[TURNS * 2 * KB];
  __shared__ uint8_t bufs[WN][2048];
  const int per = gridDim.x / 8, b = (blockIdx.x % 8) * per + blockIdx.x / 8, tm = b / a.groups;
  if (tm >= a.tiles_m) return;
  const Tile t = a.tiles[tm];
  if (t.count == 0) return;
  const Place at{a.w + (size_t)t.expert * a.n * a.kb * BLK, a.s + (size_t)t.expert * (a.n / BLK) * a.kb, t.first, t.count, 0, 0};
  uint8_t* buf = bufs[threadIdx.x / WAVE];
  if (t.count <= 64)
    resident_tile<KB, 4>(a, at, b % a.groups, sw, buf, reinterpret_cast<Stage<4>(&)[KB]>(st));
  else
    resident_tile<KB, 8>(a, at, b % a.groups, sw, buf, st);
}

template <int MODE, int MT>
__global__ __launch_bounds__(T, MODE == DENSE_F32 ? 1 : 2) void k_wide(Wide a) {
  // (objects of their own: the compiler then knows that a stage's reads need not wait for
  // another's DMA)
  __shared__ Stage<4> l0, l1, l2;
  __shared__ Stage<8> h0, h1;
  __shared__ float sw[2][MAX_DIM / BLK];
  __shared__ uint32_t top[MODE == UP ? WN : 1][128];
  __shared__ uint8_t bufs[MODE == UP || MODE == DENSE_F32 ? 1 : WN][2048];
  uint8_t* buf = bufs[MODE == UP || MODE == DENSE_F32 ? 0 : threadIdx.x / WAVE];
  // a block's XCD is its index modulo 8: each XCD takes neighbouring tiles, whose rows and
  // weights its L2 then holds once for all
  const int per = gridDim.x / 8;
  int b = (blockIdx.x % 8) * per + blockIdx.x / 8;
  Place at{a.w, a.s, 0, 0, 0, 0};
  if (MODE == UP || MODE == DOWN) {
    const int tm = b / a.tiles_n;
    if (tm >= a.tiles_m) return;
    const Tile t = a.tiles[tm];
    if (t.count == 0) return;
    at.tn = b % a.tiles_n;
    at.first = t.first;
    at.count = t.count;
    at.w += (size_t)t.expert * a.n * a.kb * BLK;
    at.s += (size_t)t.expert * ((a.n + BLK - 1) / BLK) * a.kb;
  } else {
    constexpr int GM = 8;  // row tiles side by side
    const int tiles = a.tiles_m * a.tiles_n;
    at.split = b / tiles;
    if (at.split >= a.splits) return;
    b -= at.split * tiles;
    const int group = b / (GM * a.tiles_n), in = b % (GM * a.tiles_n), high = min(GM, a.tiles_m - group * GM);
    at.tn = in / high;
    at.first = (int64_t)(group * GM + in % high) * (16 * MT);
    at.count = (int)min((int64_t)(16 * MT), a.rows - at.first);
  }
  if constexpr (MT == 4)
    tile<MODE, 4>(a, at, sw, top, buf, l0, l1, l2);
  else if ((MODE == UP || MODE == DOWN) && at.count <= 64)
    tile<MODE, 4>(a, at, sw, top, buf, l0, l1, l2);
  else
    tile<MODE, 8>(a, at, sw, top, buf, h0, h1);
}

template <int MODE, int MT>
hipError_t launch(const Wide& a, int splits, hipStream_t st) {
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n * splits;
  k_wide<MODE, MT><<<(uint32_t)((tiles + 7) / 8 * 8), T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t wide_product(const Product& p, hipStream_t st) {
  Wide a{p.q.q, p.q.s, p.q.ld, p.w, p.s, p.n, p.k / BLK, p.rows, p.out, p.out_stride};
  const bool low = p.f32 || p.plan.bm == 64;
  a.tiles_n = (p.n + BN - 1) / BN;
  a.tiles_m = (int)((p.rows + (low ? 63 : 127)) / (low ? 64 : 128));
  a.split = p.part;
  a.splits = p.plan.splits;
  if (p.f32) return launch<DENSE_F32, 4>(a, a.splits, st);
  return low ? launch<DENSE_BF16, 4>(a, a.splits, st) : launch<DENSE_BF16, 8>(a, 1, st);
}

hipError_t wide_experts_up(const Experts& e, hipStream_t st) {
  Wide a{e.x.q, e.x.s, e.x.ld, e.w13, e.s13, 2 * e.inter, e.hidden / BLK, 0, e.mid_q.q, e.inter,
         e.sorted.tiles, e.sorted.token, e.inter, e.mid_q.s, e.mid_q.ld};
  a.tiles_m = e.tiles;
  a.tiles_n = e.inter / BLK;
  return launch<UP, 8>(a, 1, st);
}

hipError_t wide_experts_down(const Experts& e, hipStream_t st) {
  Wide a{e.mid_q.q, e.mid_q.s, e.mid_q.ld, e.w2, e.s2, e.hidden, e.inter / BLK, 0, nullptr, 0,
         e.sorted.tiles, e.sorted.token};
  a.part = e.part;
  a.tiles_m = e.tiles;
  a.tiles_n = (e.hidden + BN - 1) / BN;
  if (a.kb > 4) return launch<DOWN, 8>(a, 1, st);
  a.groups = (a.tiles_n + TURNS - 1) / TURNS;
  const uint32_t grid = (uint32_t)(((int64_t)a.tiles_m * a.groups + 7) / 8 * 8);
  if (a.kb > 2)
    k_down_resident<4><<<grid, T, 0, st>>>(a);
  else
    k_down_resident<2><<<grid, T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
