// Host-side declarations of the prompt-width operators (internal to the library): FP8
// block products, paged cache appends and routed experts over up to MAX_ROWS rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "mono.h"

namespace mono {
namespace prompt {

constexpr int BLK = 128;             // a scale's block of rows' and weights' columns
constexpr int MAX_EXPERTS = 1024;    // routed experts (a sort block each)
constexpr int MAX_DIM = 1 << 16;     // columns and outputs of a product
constexpr int64_t MAX_ROWS = 1 << 20;  // rows a call; picks of all rows of an experts call
constexpr int64_t MAX_ELEMENTS = (1ll << 35) - 1;  // of the rows of a product or an experts call

constexpr int LATENT = 512, PE = 64, INDEX = 128, INDEX_HEADS = 64, PAGE = 64;
constexpr int MAX_COLUMNS = 8192;  // pages that a call scores or selects from: 524288 keys
constexpr int MAX_HEADS = 128;

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

hipError_t append(const mono_prompt_append_args& a, const int32_t* slot_pos, hipStream_t st);
hipError_t index_query(const mono_prompt_query_args& a, hipStream_t st);
hipError_t page_scores(const mono_prompt_scores_args& a, hipStream_t st);
hipError_t select_pages(const mono_prompt_select_args& a, hipStream_t st);

// MLA attention over cache pages: of each token's list of pages (attention), or of all of its
// request's (tree: `starts` is given, and tokens are nodes).
struct Paged {
  const void* q;  // bf16 [tokens, heads, 576]
  int64_t tokens;
  int heads;
  const int32_t *req, *pos, *pages;
  int picks;
  const int32_t *starts, *prefix;
  const int64_t* mask;
  const int32_t* page_table;
  int requests, pt_stride, n_pages;
  const void* kv;
  const float* kv_scale;
  float scale_log2;  // the softmax scale x log2(e)
  void* out;         // bf16 [tokens, heads, 512]
  // how it is shared out: heads a workgroup, workgroups a token's heads, workgroups a token's
  // pages (not planned trees), and all of them
  int head_rows, head_tiles, splits;
  int64_t work;
  // trees of few nodes, planned on the device: workgroups, and what each node's chunks are
  int tasks;
  struct NodePlan* plan;  // [tokens]
  int64_t parts;
  float *part, *part_m, *part_l;  // pages shared out: f32 [parts, heads, 512] and [.., heads] twice
};
struct NodePlan {
  int chunks, part;  // its chunks of pages (0: a node of no request), the first one's part
};

// How the pages are shared out. Only where the tokens' heads alone would leave CUs without
// work: two workgroups a CU (FULL), a page each at least. A tree's pages are known on the device
// only; with up to PLANNED nodes' tiles of heads, of up to PLAN_REQUESTS requests, its workgroups plan
// there, FULL of them or FULL more than tiles, so that long nodes have two or more. Planned and not:
// 4000 keys, 64 nodes 44 and 101 us, 256 nodes 98 and 114, 256 of ragged requests 49 and 97; 8 nodes of 30000
// keys beside 480 shorter ones 139 and 616. The plan and a join that finds little cost what it
// costs: 500 keys, 64 nodes 24.4 and 23.5, 512 nodes 37 and 34, 1000 nodes 64 and 59.
//
// 32 heads a workgroup read a page once for two tiles of 16. But where the slots are not full, tiles by
// themselves end sooner: of tokens, where a page a tile is FULL tasks at most (1 token, 32 pages 10.9 us
// and 12.3; 8 tokens, 512 such tasks, 20.8 and 22.3; 2000 tokens 516 and 314). Of trees the host knows no
// lengths, and the width of their tables says nothing of them (nor is a node's rounding to hang on it): up
// to TREE_TILES tiles go by themselves. Alone and in pairs, us at 1000, 4000, 16000, 32000 and 64000 keys,
// 32 heads: 1 node 11.5 13.4 18.7 21.7 25.8 and 13.1 14.7 25.6 26.7 28.3; 8 nodes 15.9 20.0 30.3 41.0 62.8 and
// 16.5 23.8 33.6 40.8 56.0; 16 nodes 17.0 24.8 41.2 63.2 and 22.0 27.9 40.5 55.6.
constexpr int FULL = 512, PLANNED = 1024, PLAN_REQUESTS = 256, TREE_TILES = 16;
inline void paged_plan(Paged& a, int pages) {
  const int64_t tiles = a.tokens * ((a.heads + 15) / 16);
  a.head_rows = a.heads <= 16 || (a.starts ? tiles <= TREE_TILES : tiles * pages <= FULL) ? 16 : 32;
  a.head_tiles = (a.heads + a.head_rows - 1) / a.head_rows;
  const int64_t whole = a.tokens * a.head_tiles;
  a.splits = 1;
  a.work = whole;
  if (a.starts) {
    if (whole <= PLANNED && pages > 1 && a.requests > 0 && a.requests <= PLAN_REQUESTS) {
      const int64_t spare = whole <= FULL / 2 ? FULL - whole : FULL;  // tasks beside one a node's tile
      a.tasks = a.work = whole + spare;
      // nodes of two chunks or more: with as many nodes as spare tasks they have most parts
      a.parts = std::min<int64_t>((spare + std::min(spare, whole)) / a.head_tiles, a.tokens * (pages + 1ll));
    }
    return;
  }
  const int64_t fit = FULL / whole;
  a.splits = (int)std::max<int64_t>(std::min<int64_t>(fit, pages), 1);
  a.work = whole * a.splits;
  if (a.splits > 1) a.parts = a.tokens * a.splits;
}
hipError_t paged_attention(const Paged& a, hipStream_t st);
hipError_t join_attention(const Paged& a, hipStream_t st);

}  // namespace prompt
}  // namespace mono
