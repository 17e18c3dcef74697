// Host-side declarations of the prompt-width operators (internal to the library): FP8
// block products, paged cache appends and routed experts over up to MAX_ROWS rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mono.h"

namespace mono {
namespace prompt {

constexpr int BLK = 128;             // a scale's block of rows' and weights' columns
constexpr int MAX_EXPERTS = 1024;    // routed experts (a sort block each)
constexpr int MAX_DIM = 1 << 16;     // columns and outputs of a product
constexpr int64_t MAX_ROWS = 1 << 20;  // rows a call; picks of all rows of an experts call
constexpr int64_t MAX_ELEMENTS = (1ll << 35) - 1;  // of the rows of a product or an experts call

constexpr int LATENT = 512, PE = 64, INDEX = 128, PAGE = 64;

// Rows rounded to E4M3: codes [rows, k] and scales [k / 128, ld] (a block's scales of
// consecutive rows lie together: a product's lanes hold one row each).
struct Rows {
  uint8_t* q;
  float* s;
  int ld;
};

// One tile of expert work: `count` sorted places from `first` on, of expert `expert`.
struct Tile {
  int expert, first, count, pad;
};

// The tokens sorted by expert. Place p < picks holds a routed pick, place picks + t
// token t's row of the shared expert.
struct Sorted {
  int* token;  // [picks + tokens] token of each place
  int* place;  // [picks] place of each pick (token * k + j), -1: routed nowhere
  Tile* tiles; // [all_tiles], some of them empty (count 0)
};

// The tile list's length: the shared expert's tiles, then room for every routed expert's
// whole tiles and a partial one of each (and never more than one for each pick).
inline int64_t all_tiles(int64_t tokens, int64_t picks, int experts, int bm, bool shared) {
  const int64_t routed = picks / bm + experts;
  return (shared ? (tokens + bm - 1) / bm : 0) + (picks < routed ? picks : routed);
}

// The experts' outputs before their weighted sum, [places, ld]: f16 values and, for each 64
// columns of a place, the power of two that they are multiplied by, which puts the largest
// of them into [2^14, 2^15). 16 bits halve the bytes of the largest tensor of a call; a value is
// 2^-11 of itself off at most, an eighth of the output's own rounding to bf16 (2^-8); below 2^-29
// of its block's largest value, 2^-39 of that.
constexpr int PART = 64;
struct Parts {
  uint16_t* v;
  float* s;
  int ld;
};

// Blocks that one launch rounds at most: 16 threads each in workgroups of 1024, and one such
// workgroup more for each expert that sorts beside them. A launch's threads are counted in 32
// bits; more rows take another launch.
constexpr int64_t ROUND_BLOCKS = 1 << 27;
static_assert(ROUND_BLOCKS * 16 + MAX_EXPERTS * 1024 < 1ll << 32, "a rounding launch's threads");
static_assert(ROUND_BLOCKS >= MAX_DIM / BLK, "a launch rounds at least a row");

hipError_t quant_rows(const void* x, bool f32, int64_t stride, int64_t rows, int k, const Rows& out, hipStream_t st);
hipError_t sort_quant(const void* x, int64_t stride, int64_t tokens, int k, const Rows& out, const int* ids, int picks_each,
                      int experts, bool shared, int bm, const Sorted& sorted, hipStream_t st);
// How a product runs, by its sizes alone.
//
// FEW     at most 16 rows of FEW_BYTES codes: every workgroup rounds them for itself
// NARROW  up to WIDE_ROWS rows (f32: NARROW_TILES_F32 workgroups): workgroups of 16 weight rows
//         and up to 64 rows, 8 waves along K
// WIDE    more: tiles of 256 weight rows x 64 or 128 rows, waves along the weight rows
//
// (narrow / wide, us a call in a graph, rows x 2112 x 7168: 17 rows 11.0 / 13.3, 24 12.3 / 13.5,
// 33 19.0 / 14.2, 65 24.9 / 16.0; x 7168 x 4096: 17 11.4 / 13.2, 33 16.9 / 14.4. In f32, whose
// wide tiles widen their codes in every wave: rows x 576 x 7168: 129 rows 16.6 / 19.6, 257
// 23.1 / 21.1; x 2112: 45 18.6 / 19.1, 65 22.2 / 20.4; x 128: 1024 23.9 / 24.5.)
//
// `splits` > 1: K is shared out over that many workgroups, whose f32 sums a second launch
// adds in order. Where the tiles alone leave CUs without work, and each share keeps at
// least 8 blocks of K.
constexpr int FEW_BYTES = 32768;
constexpr int WIDE_ROWS = 32, NARROW_TILES_F32 = 128;
struct ProductPlan {
  enum Kind { FEW, NARROW, WIDE } kind;
  int splits;
  int bm;  // rows of a tile
};
inline ProductPlan product_plan(int64_t rows, int n, int k, bool f32) {
  if (rows <= 16 && rows * k <= FEW_BYTES) return {ProductPlan::FEW, 1, 16};
  const int kb = k / BLK;
  constexpr int64_t FULL = 256;  // workgroups that leave no CU without one
  int64_t tiles;
  ProductPlan p;
  const int64_t narrow = n / 16 * ((rows + 63) / 64);
  if (f32 ? narrow <= NARROW_TILES_F32 : rows <= WIDE_ROWS) {
    p = {ProductPlan::NARROW, 1, 64};
    tiles = narrow;
  } else {
    const int64_t wide = (n + 255) / 256;
    p = {ProductPlan::WIDE, 1, (rows + 127) / 128 * wide < 256 ? 64 : 128};
    tiles = (rows + p.bm - 1) / p.bm * wide;
  }
  const int64_t s = FULL / tiles < kb / 8 ? FULL / tiles : kb / 8;
  if (p.bm == 64 && s > 1) p.splits = (int)s;
  return p;
}

// A product's launch. part: f32 [splits, rows, n] where splits > 1.
struct Product {
  const void* x;
  int64_t x_stride;
  Rows q;  // the rows' codes (not FEW)
  int64_t rows;
  const uint8_t* w;
  const float* s;
  int n, k;
  void* out;
  int64_t out_stride;
  bool f32;
  float* part;
  ProductPlan plan;
};
hipError_t few_product(const Product& a, hipStream_t st);
hipError_t narrow_product(const Product& a, hipStream_t st);
hipError_t wide_product(const Product& a, hipStream_t st);
hipError_t join_product(const Product& a, hipStream_t st);

struct Experts {
  Rows x, mid_q;
  Sorted sorted;
  float* mid;  // f32 [places, inter]
  Parts part;
  const uint8_t *w13, *w2;
  const float *s13, *s2, *weights;
  const void* residual;
  int64_t residual_stride;
  void* out;
  int64_t out_stride;
  int64_t tokens, picks;
  int picks_each, experts, hidden, inter, bm, tiles;
  bool shared, wide;
};
hipError_t experts_up(const Experts& a, hipStream_t st);
hipError_t experts_down(const Experts& a, hipStream_t st);
hipError_t wide_experts_up(const Experts& a, hipStream_t st);
hipError_t wide_experts_down(const Experts& a, hipStream_t st);
hipError_t experts_back(const Experts& a, hipStream_t st);

hipError_t append(const mono_prompt_append_args& a, hipStream_t st);

}  // namespace prompt
}  // namespace mono
