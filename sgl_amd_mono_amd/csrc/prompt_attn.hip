// MLA attention over pages of the latent cache: of the pages that each token selected
// (attention), and of a whole prefix with the drafted tokens that a mask leaves (tree).
//
//   s[h, j] = scale kvs[j] (q[h] . c[j]),  576 dims;  out[h] = sum_j softmax_j(s) kvs[j] c[j, :512]
//
// A workgroup takes a token and up to 32 of its heads, and walks through pages of 64 keys with
// a running maximum and sum. A page is one piece of 36 KB, brought to LDS as it lies by DMA
// (global_load_lds), the next one while this one is worked on, and read from there twice: as
// rows for q . c and transposed (ds_read_b64_tr_b8) for p . v.
//
//   q . c   wave w: keys 16 w .. + 15 against every head, in E4M3 as the cache has them
//   p . v   wave w: dims 128 w .. + 127 over all 64 keys, widened to bf16 in registers, exactly;
//           the probabilities meet in LDS
//
// q is split into two E4M3 pieces of four significant bits, which hold bf16's eight: q . c is then
// two FP8 products of twice bf16's rate and the keys are not widened. Two things are less exact so.
// Elements below 2^-14 of their head's largest (2^-10 in the last 64 dims, whose pieces share an
// instruction and so a scale) lose bits: they are off by 2^-21.8 (2^-17.8) of the largest at most. And
// the FP8 instruction does not sum in full f32: it lines its products up with the largest and cuts what
// is below, up to 2^-16 of a logit's terms' magnitudes (seen of unlike elements; of random ones two logits'
// difference is off by 2^-18 of both at most, 2^-20.5 in the root of squares). Outputs in bf16 do not show
// it: against 64 bits they are off by 0.00211, 0.00169 and 0.00201 of their norm (777 tokens, 5 nodes, 129
// nodes) here and with q in bf16 against widened keys; with q 64 times as large, logits of 110, by 0.00069,
// 0.00051 and 0.00069 here and 0.00067, 0.00050 and 0.00068 there. That form takes longer: 4096 tokens 648 us
// for 604, 777 tokens 49 for 43, 129 nodes 38.7 for 33.7, 1024 nodes 592 for 550 (side by side on one card).
//
// Probabilities times their key's scale are rounded to bf16, off by 2^-8 of each at most and at random,
// beside the output's own 2^-8, which alone is 0.0017 of the norm; their sum adds up the f32 values. (Two
// E4M3 pieces of them were tried: small ones lose bits against the largest, which outputs that hang on many
// keys show.)
//
// The maximum that the sums refer to stays as it is until a probability passes 2^4 (a ratio of
// sums does not depend on it, and bf16 and f32 hold 2^4 as well as 1): the waves' maxima then meet
// and the sums are scaled, which happens on a token's first page and rarely after it.
//
// Two workgroups a CU (80 KB of LDS, 256 registers a lane), a page of 32 heads in 1.15 us a CU:
// 4096 tokens of 32 heads over 2048 keys 584 to 632 us by the card, 910 to 985 TFLOP/s; a large bf16 product
// reaches 1180 to 1200. Matrix instructions (44 % of the cycles) and vector issue (50 %: the widening, the
// probabilities, addresses), at a clock that power holds at 1.75 to 1.9 GHz, are what bounds it.
// Heads of up to 16 take one tile of 16 (2000 tokens 224 us, in a half-empty pair of them 304), up
// to 32 two side by side (2000 tokens 314 us, as two workgroups 516, which read the pages twice).
#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 256, WAVES = 4, ROW = LATENT + PE, PAGE_BYTES = PAGE * ROW;
constexpr int BLOCKS = ROW / 64, BLOCK_BYTES = PAGE * 64;  // a page's rows in blocks of 64 dims
constexpr int HEADS = 32;
// NONE: no maximum yet, the lowest there can be (and finite: what is taken from it is a number)
constexpr float NEG_INF = -__builtin_inff(), NONE = -__FLT_MAX__, EXP2_SLACK = 16.0f;

// A page and its keys' scales.
struct Stage {
  alignas(16) uint8_t kv[PAGE_BYTES];
  float scale[PAGE];
};
constexpr int P_PITCH = PAGE + 8;  // (8 heads' 16 bytes fall on distinct banks)
struct Lds {
  Stage stage[2];  // (at the start the second holds q's pieces, at the end both the outputs' rows)
  alignas(16) uint16_t p[HEADS][P_PITCH];
  float top[WAVES][HEADS];  // the waves' maxima, at the end their sums
  float by[HEADS];          // what a head's sums are scaled by
  uint32_t q_scale[HEADS];
  int over[WAVES];
  int slot[WAVE];       // a run of 64 pages of the list: where each lies in the pool
  uint64_t seen[WAVE];  // and which of its keys are seen
};

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lvoid;
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// DMA of 16 (4) bytes a lane, from base + the lane's offset to `to` + 16 (4) lane. The builtin
// does the same, but the compiler then waits for it before the first read of any LDS; written
// out, it writes no register that the compiler knows of, and is waited for where a page is used.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is named so that nothing of the compiler's own comes between)
MONO_DEV void dma16(const uint8_t* base, uint32_t offset, void* to, bool go) {
  asm volatile(
      "s_cmp_eq_u32 %3, 0\n\t"
      "s_cbranch_scc1 .Lno_dma%=\n\t"
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2\n"
      ".Lno_dma%=:" ::"s"((uint32_t)(uintptr_t)(lvoid*)to), "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(go ? 1 : 0)) : "memory", "m0", "scc");
}
MONO_DEV void dma4(const float* base, uint32_t offset, void* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"((uint32_t)(uintptr_t)(lvoid*)to), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop

// 16 lanes read 8 rows x 16 bytes of LDS transposed: lane l gives the address of bytes
// 8 (l % 2) .. of row l / 2 and gets byte l of each of the 8 rows.
MONO_DEV u32x2 lds_transposed(const uint8_t* p) { return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)p)); }

// E4M3 x E4M3; the second operand's lanes have scales, byte B of `scale`
template <int B>
MONO_DEV f32x4 mfma_16(const i32x8& a, const i32x8& b, const f32x4& c, int scale) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 127, B, scale);
}
// The values' MFMAs, dims x keys against keys x heads in bf16, as wide as there are tiles of heads.
// Of C[S x S] += A[S x K] B[K x S] lane l has row / column l % S, k 8 (l / S) .. + 7, and of C rows
// 8 (i / 4) + 4 (l / S) + i % 4 of column l % S.
MONO_DEV f32x16 values_mfma(const bf16x8& a, const bf16x8& b, const f32x16& c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
MONO_DEV f32x4 values_mfma(const bf16x8& a, const bf16x8& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <int MT>
struct Values {
  static constexpr int S = 16 * MT, K = 512 / S, R = S * S / WAVE;  // R: registers of C
  static constexpr int TILES = LATENT / WAVES / S;                 // of dims, a wave
  typedef float C __attribute__((ext_vector_type(R)));
};
MONO_DEV bf16x8 widen8(const u32x2& w) {
  bf16x8 v;
  widen4(w[0], v, 0);
  widen4(w[1], v, 4);
  return v;
}
MONO_DEV i32x8 join(const u32x4& lo, const u32x4& hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// Four values of at most 448 x `unit` (a power of two) as two E4M3 pieces each: the nearest
// multiple of `unit`, and what is left in multiples of `fine`.
MONO_DEV void two_pieces(const float (&v)[4], float unit, float fine, uint32_t& hi, uint32_t& lo) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  i16x2 h = {0, 0}, l = {0, 0};
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, v[0], v[1], unit, false);
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, v[2], v[3], unit, true);
  hi = __builtin_bit_cast(uint32_t, h);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, unit, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, unit, true);
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, v[0] - a[0], v[1] - a[1], fine, false);
  l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, v[2] - b[0], v[3] - b[1], fine, true);
  lo = __builtin_bit_cast(uint32_t, l);
}

// A page in LDS: block by block of 64 dims, in each the keys' 64 bytes as four units of 16,
// swapped by the key's number so that neither the 16 keys' reads of one unit nor a transposed
// read of 8 keys' two halves meets a bank twice. (A DMA turn is then 16 keys' 64 bytes of one
// block: a lane's place in it is the same for every block and wave.)
MONO_DEV uint32_t unit_of(uint32_t key, uint32_t u) { return u ^ (key >> 1 & 3); }

// Barriers that leave the next page's DMA in flight (a __syncthreads would wait for it).
// (The waits are builtins, which the compiler's own count of loads takes part in.)
template <bool LOADS>
MONO_DEV void meet_of() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(LOADS ? 0x0070 : 0xc07f);  // lgkmcnt(0), and vmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
MONO_DEV void meet() { meet_of<false>(); }
MONO_DEV void meet_after_loads() { meet_of<true>(); }

// this lane's index from an opaque copy: addresses are formed where they are used and not held
// in registers across the loop
MONO_DEV uint32_t lane_now(uint32_t lane) {
  asm volatile("" : "+v"(lane));
  __builtin_assume(lane < WAVE);
  return lane;
}

MONO_DEV uint32_t pack2(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}

// the larger / the sum over the four lane groups l, l ^ 16, l ^ 32, l ^ 48
MONO_DEV float groups_max(float v) {
  u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
MONO_DEV float groups_sum(float v) {
  u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// What a workgroup reads: pages [lo, hi) of a token's list (attention) or of its request's
// (tree), and which keys of each are seen.
struct Reads {
  const int32_t* table;  // the request's row of the page table
  const int32_t* list;   // attention: the token's pages
  int lo, hi;
  int64_t end;           // keys at positions below it are seen
  uint64_t draft;        // tree: bit j: the key at position end + j is seen too
};

// bit j: key j of page `page` is seen
MONO_DEV uint64_t seen_of(const Reads& rd, int page, bool tree) {
  const int64_t n = rd.end - (int64_t)page * PAGE;
  uint64_t m = n >= PAGE ? ~0ull : n > 0 ? (1ull << n) - 1 : 0;
  if (tree && n < PAGE && n > -PAGE) m |= n >= 0 ? rd.draft << n : rd.draft >> -n;
  return m;
}

// A workgroup's task: a token (node), heads 16 MT ht .., chunk `chunk` of `chunks` of its pages, whose
// parts are rows of part `part` (chunks > 1).
struct Task {
  int64_t t;
  int ht, chunk, chunks;
  int64_t part;
  bool any;  // it has pages
};

MONO_DEV void node_reads(const Paged& a, int64_t t, int req, Reads& rd) {
  rd.table = a.page_table + (int64_t)req * a.pt_stride;
  rd.end = max(a.prefix[req], 0);
  rd.draft = (uint64_t)a.mask[t];
}

// A request's nodes and pages (the last one or two hold the draft's keys, the last one perhaps none and
// then, perhaps, behind the table: how pages are shared out hangs on the prefix alone and not on how wide
// the table is. MOST_PAGES: more than the card's memory holds).
constexpr int MOST_PAGES = 1 << 23;
struct Request {
  int64_t first;
  int n, pages;
};
MONO_DEV Request request_of(const Paged& a, int r) {
  const int at = min(r, a.requests - 1);
  const int from = a.starts[at], to = a.starts[at + 1], prefix = a.prefix[at];
  Request q;
  q.first = min((int64_t)max(from, 0), a.tokens);
  q.n = r < a.requests ? (int)max(min((int64_t)to, a.tokens) - q.first, (int64_t)0) : 0;
  q.pages = q.n ? (int)min((int64_t)min(a.pt_stride, MOST_PAGES), ((int64_t)max(prefix, 0) + PAGE - 1) / PAGE) + 1 : 0;
  return q;
}
// Lane l: requests l, 64 + l, .. of up to PLAN_REQUESTS.
constexpr int REQUEST_SETS = PLAN_REQUESTS / WAVE;
struct Requests {
  Request of[REQUEST_SETS];
};
template <class F>
MONO_DEV void each_set(const Paged& a, F f) {
#pragma unroll
  for (int i = 0; i < REQUEST_SETS; ++i)
    if (i == 0 || WAVE * i < a.requests) f(i);
}

// Planned trees: each node's pages in chunks of so many, a request's nodes side by side over
// the same chunk: the fewest pages a chunk that make at most `most` tasks, between their share of
// all pages and that of all pages beside a short chunk a node. `tasks` comes to be how many there are.
//
// Two workgroups a CU, but one where that has FEW_PAGES pages at most: fewer parts to write and
// join are then worth more (20000 keys, 512 and 256 tasks: 1 node 21.9 and 19.0 us, 4 nodes 26.8 and 26.7,
// 8 nodes 32.5 and 36.1, 16 nodes 44.0 and 49.6; 4000 keys, 8 nodes 23.7 and 20.0, 16 nodes 30.6 and 27.3).
// And whole nodes where chunks save
// at most JOIN_PAGES pages (9 pages a node, 128 nodes: in twos 34 us, whole 28.5; 64 nodes, in threes 25,
// whole 27). More nodes than one round's half are whole but for those longer than a workgroup's share.
constexpr int FEW_PAGES = 8, JOIN_PAGES = 4;
MONO_DEV int chunk_pages(const Paged& a, const Requests& r, int64_t& tasks) {
  int64_t total = 0;
  uint32_t longest = 0;
  each_set(a, [&](int i) {
    const int64_t pages = (int64_t)r.of[i].n * r.of[i].pages;
    total += wave_sum_i((int)(pages & 0xffff)) + ((int64_t)wave_sum_i((int)(pages >> 16)) << 16);
    longest = max(longest, wave_umax((uint32_t)r.of[i].pages));
  });
  total *= a.head_tiles;
  const auto share = [](int64_t n, int by) { return (int)max((n + by - 1) / by, (int64_t)1); };
  const auto made = [&](int each) {
    int n = 0;
    each_set(a, [&](int i) { n += wave_sum_i(r.of[i].n * ((r.of[i].pages + each - 1) / each)); });
    return n * a.head_tiles;
  };
  const int least = (int)a.tokens * a.head_tiles;
  const int most = total <= FULL / 2 * FEW_PAGES && least <= FULL / 4 ? FULL / 2 : (int)a.work;
  int lo = share(total, min(most, FULL)), hi = max(share(total, most - least), lo);
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (made(mid) <= most) hi = mid;
    else lo = mid + 1;
  }
  if ((int)longest <= hi + JOIN_PAGES) hi = max((int)longest, 1);
  tasks = min((int64_t)made(hi), a.work);  // (more only by starts that do not ascend)
  return hi;
}

// Task `id` of them; false behind the last.
MONO_DEV bool planned_task(const Paged& a, const Requests& r, int each, int id, Task& k, Reads& rd) {
  k.ht = id % a.head_tiles;
  id /= a.head_tiles;
  int part = 0;
  bool found = false;
  each_set(a, [&](int i) {
    const Request q = r.of[i];
    const int chunks = (q.pages + each - 1) / each, tasks = q.n * chunks, parts = chunks > 1 ? tasks : 0;
    const int upto = wave_incl_scan(tasks), parts_upto = wave_incl_scan(parts);
    const uint64_t here = __ballot(upto > id);
    if (here && !found) {
      found = true;
      const int l = __builtin_ctzll(here);
      const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int nodes = of(q.n), at = id - (of(upto) - of(tasks)), node = at % nodes;
      k.chunk = at / nodes;
      k.chunks = of(chunks);
      k.part = part + of(parts_upto) - of(parts) + node * k.chunks + k.chunk;
      k.t = (int64_t)of((int)q.first) + node;
      node_reads(a, k.t, WAVE * i + l, rd);
      rd.lo = k.chunk * each;
      rd.hi = min(rd.lo + each, of(q.pages));
      k.any = true;
    }
    id -= __builtin_amdgcn_readlane(upto, WAVE - 1);
    part += __builtin_amdgcn_readlane(parts_upto, WAVE - 1);
  });
  return found && (k.chunks == 1 || k.part < a.parts);  // (more parts only by starts that do not ascend)
}

template <bool TREE>
MONO_DEV void task_of(const Paged& a, int lane, int64_t id, Task& k, Reads& rd) {
  k.ht = (int)(id % a.head_tiles);
  const int64_t rest = id / a.head_tiles;
  k.t = rest / a.splits, k.chunk = (int)(rest % a.splits), k.chunks = a.splits;
  k.part = rest;
  k.any = false;
  int pages;
  if (TREE) {
    // the request whose nodes hold t: as many starts as are at most t
    int at = 0;
    for (int r0 = 0; r0 <= a.requests; r0 += WAVE) at += __popcll(__ballot(r0 + lane <= a.requests && a.starts[min(r0 + lane, a.requests)] <= k.t));
    if (at < 1 || at > a.requests) return;
    node_reads(a, k.t, at - 1, rd);
    const int drafted = rd.draft ? 64 - __builtin_clzll(rd.draft) : 0;
    pages = (int)min((int64_t)a.pt_stride, (rd.end + drafted + PAGE - 1) / PAGE);
  } else {
    const int req = a.req[k.t], pos = a.pos[k.t];
    if (req < 0 || req >= a.requests || pos < 0) return;
    rd.table = a.page_table + (int64_t)req * a.pt_stride;
    rd.list = a.pages + k.t * a.picks;
    rd.end = (int64_t)pos + 1;
    rd.draft = 0;
    pages = a.picks;
  }
  rd.lo = (int)((int64_t)pages * k.chunk / k.chunks);
  rd.hi = (int)((int64_t)pages * (k.chunk + 1) / k.chunks);
  k.any = rd.lo < rd.hi;
}

template <int MT, bool TREE>
MONO_DEV void attend(const Paged& a, Lds& L, int lane, int wave, const Task& task, const Reads& rd) {
  // (one tile of heads leaves registers to hold addresses in: 2000 tokens 237 -> 224 us)
  const auto here = [&]() { return MT == 1 ? (uint32_t)lane : lane_now(lane); };
  const int64_t t = task.t;
  const int h0 = task.ht * 16 * MT;
  const bool any = task.any;
  using V = Values<MT>;
  typename V::C o[V::TILES];  // of lane l: dims 128 wave + S t + 8 (i / 4) + 4 (l / S) + i % 4 of head l % S
  float m_ref[MT], l_run[MT];
#pragma unroll
  for (int c = 0; c < MT; ++c) m_ref[c] = NONE, l_run[c] = 0.f;
#pragma unroll
  for (int b = 0; b < V::TILES; ++b)
#pragma unroll
    for (int i = 0; i < V::R; ++i) o[b][i] = 0.f;
  if (any) {
    int buf = 0;
    uint64_t live = 0;  // pages left of a run of 64 of the list
    // page i's way to LDS: this wave's 16 keys, a block of dims at a time, and the scales
    const auto place_of = [&](int i) { return (int64_t)__builtin_amdgcn_readfirstlane(L.slot[i]) * PAGE; };
    const auto lane_place = [&]() {
      const uint32_t ln = here();
      return ln / 4 * ROW + 16 * unit_of(ln / 4, ln % 4);
    };
    const auto bring = [&](int64_t first, uint32_t at, Stage& to, int b, bool go) {
      dma16(static_cast<const uint8_t*>(a.kv) + (first + 16 * wave) * ROW + 64 * b, at, &to.kv[b * BLOCK_BYTES + wave * 1024], go);
    };
    const auto bring_scales = [&](int64_t first, Stage& to) {
      if (wave == 0 && a.kv_scale) dma4(a.kv_scale + first, 4 * here(), to.scale);
    };
    const auto run_from = [&](int at) {  // the run that begins at page `at` of the list, and its first page on its way
      int page = -1, slot = -1;
      if (at + lane < rd.hi) page = TREE ? at + lane : rd.list[at + lane];
      uint64_t seen = 0;
      if (page >= 0 && page < a.pt_stride) {
        slot = rd.table[page];
        if (slot >= 0 && slot < a.n_pages) seen = seen_of(rd, page, TREE);
      }
      live = __ballot(seen != 0);
      meet();  // (the run before has been read)
      if (wave == 0) L.slot[lane] = slot, L.seen[lane] = seen;
      meet();
      if (live) {
        const int64_t first = place_of(__builtin_ctzll(live));
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) bring(first, lane_place(), L.stage[buf], b, true);
        bring_scales(first, L.stage[buf]);
      }
    };
    int at = rd.lo;
    run_from(at);
    // q's heads as two pieces (behind the first page, which more steps led to): wave w's eight
    // heads, 8 lanes each, through LDS to all the waves
    if (wave < 2 * MT) {
      const uint32_t ln = here(), head = 8 * wave + ln / 8;
      const uint16_t* row = static_cast<const uint16_t*>(a.q) + (t * a.heads + min(h0 + (int)head, a.heads - 1)) * ROW + 8 * (ln % 8);
      u32x4 v[BLOCKS];
      uint32_t most = 0;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        v[b] = ld_u32x4(row + 64 * b);
#pragma unroll
        for (int i = 0; i < 4; ++i) most = max(most, max(v[b][i] & 0x7fffu, v[b][i] >> 16 & 0x7fffu));
      }
      most = max(most, dpp_u<DPP_XOR1>(most));
      most = max(most, dpp_u<DPP_XOR2>(most));
      most = max(most, dpp_u<DPP_HALF_MIRROR>(most));
      // the power of two that puts the largest into (224, 448]
      const uint32_t e = max((most >> 7) + ((most & 0x7fu) > 0x60u ? 1u : 0u), 16u);
      const bool finite = most < 0x7f80u;
      const float unit = __uint_as_float((finite ? e - 8u : 127u) << 23), fine = unit * 0.0625f;
      // (q that is not finite: scales that are NaN, and so are its outputs)
      if (ln % 8 == 0) L.q_scale[head] = finite ? (e - 8u) | (e - 12u) << 8 : 0xffffu;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        u32x2 piece[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x[4] = {bf16_lo(v[b][2 * h]), bf16_hi(v[b][2 * h]), bf16_lo(v[b][2 * h + 1]), bf16_hi(v[b][2 * h + 1])};
          uint32_t hi, lo;
          two_pieces(x, unit, b < BLOCKS - 1 ? fine : unit, hi, lo);
          piece[0][h] = hi, piece[1][h] = lo;
        }
        uint8_t* to = &L.stage[1].kv[head * ROW + 64 * b + 16 * unit_of(head, ln % 8 / 2) + 8 * (ln % 2)];
        *reinterpret_cast<u32x2*>(to) = piece[0];
        *reinterpret_cast<u32x2*>(to + 16 * MT * ROW) = piece[1];
      }
    }
    static_assert(2 * HEADS * ROW <= PAGE_BYTES, "q's pieces fit a page's place");
    meet();
    // lane (g, r): of head 16 c + r units g of the blocks of 64 dims, two blocks an MFMA; of the last
    // block both pieces in one
    i32x8 q[MT][BLOCKS];  // pieces of blocks 0 and 1, 2 and 3, ..; then the last
    int q_scale = 0;
    {
      const uint32_t ln = here(), r = ln % 16, g = ln / 16;
#pragma unroll
      for (int c = 0; c < MT; ++c) {
        const uint8_t* row = &L.stage[1].kv[(16 * c + r) * ROW + 16 * unit_of(r, g)];
        const auto unit = [&](int piece, int b) { return *reinterpret_cast<const u32x4*>(row + piece * 16 * MT * ROW + 64 * b); };
#pragma unroll
        for (int k = 0; k < BLOCKS / 2; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) q[c][2 * k + h] = join(unit(h, 2 * k), unit(h, 2 * k + 1));
        q[c][BLOCKS - 1] = join(unit(0, BLOCKS - 1), unit(1, BLOCKS - 1));
        q_scale |= (int)(L.q_scale[16 * c + r] << 16 * c);
      }
    }
    // The lane's places that every page uses, held across pages: in a page's DMA, its keys for q . c and
    // as values (the unit's swap apart), and in the probabilities as they are written and read. No more
    // registers are left with two tiles of heads (32 trees of 32 nodes 597 -> 572 us).
    uint32_t dma_place, key_place, value_place, value_swap, to_place, from_place;
    {
      const uint32_t ln = here(), group = ln / V::S, row = ln % 16 / 2;
      dma_place = lane_place();
      key_place = (16 * wave + ln % 16) * 64 + 16 * unit_of(ln % 16, ln / 16);
      // (lane l reads bytes of key 8 group + l % 16 / 2 and gets one dim of the eight keys)
      value_place = 2 * wave * BLOCK_BYTES + (8 * group + row) * 64 + 8 * (ln % 2);
      value_swap = 16 * unit_of(row, ln / 16 % MT);
      to_place = ln % 16 * P_PITCH + 16 * wave + ln / 16 * 4;
      from_place = ln % V::S * P_PITCH + 8 * group;
      asm volatile("" : "+v"(dma_place), "+v"(key_place), "+v"(value_place), "+v"(value_swap), "+v"(to_place), "+v"(from_place));
    }
    for (;;) {
      // of the page that comes first, which keys are seen; where the one after it lies
      uint64_t mask = 0;
      int64_t ahead = 0;
      const auto seen_at = [&](uint64_t m) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)m) |
               (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(m >> 32)) << 32;
      };
      if (live) {
        const uint64_t rest = live & (live - 1);
        mask = seen_at(L.seen[__builtin_ctzll(live)]);
        ahead = place_of(__builtin_ctzll(rest ? rest : live));
      }
      while (live) {  // a page, while the next one of the run comes
        Stage &st = L.stage[buf], &next = L.stage[buf ^ 1];
        live &= live - 1;
        meet_after_loads();  // the page has come, and every wave is done with the one before
        const bool partial = mask != ~0ull, more = live != 0;
        if (partial) {  // what is not seen may hold anything, a NaN too: zeros instead
          const uint32_t ln = here();
          if (!(mask >> (16 * wave + ln / 4) & 1)) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) *reinterpret_cast<u32x4*>(&st.kv[b * BLOCK_BYTES + 1024 * wave + 16 * ln]) = u32x4{0u, 0u, 0u, 0u};
            if (ln % 4 == 0) st.scale[16 * wave + ln / 4] = 0.f;
          }
          meet();
        }
        if (more) bring_scales(ahead, next);
        f32x4 s[MT];
#pragma unroll
        for (int c = 0; c < MT; ++c) s[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        {
          const uint8_t* key = &st.kv[key_place];
          const auto unit = [&](int b) { return *reinterpret_cast<const u32x4*>(key + BLOCK_BYTES * b); };
          i32x8 coming = join(unit(0), unit(1));  // (the next step's keys, read while this one's MFMAs run)
#pragma unroll
          for (int k = 0; k < BLOCKS / 2 + 1; ++k) {
            const i32x8 keys = coming;
            if (k < BLOCKS / 2) {
              const u32x4 lo = unit(2 * k + 2), hi = k + 1 < BLOCKS / 2 ? unit(2 * k + 3) : lo;
              coming = join(lo, hi);
              __builtin_amdgcn_sched_barrier(0);
            }
            if (k < BLOCKS / 2) {
#pragma unroll
              for (int c = 0; c < MT; ++c) s[c] = c ? mfma_16<2>(keys, q[c][2 * k], s[c], q_scale) : mfma_16<0>(keys, q[c][2 * k], s[c], q_scale);
              bring(ahead, dma_place, next, 2 * k, more);  // (nine DMAs at once hold the wave up for 1000 cycles)
#pragma unroll
              for (int c = 0; c < MT; ++c) s[c] = c ? mfma_16<3>(keys, q[c][2 * k + 1], s[c], q_scale) : mfma_16<1>(keys, q[c][2 * k + 1], s[c], q_scale);
              bring(ahead, dma_place, next, 2 * k + 1, more);
            } else {
#pragma unroll
              for (int c = 0; c < MT; ++c) s[c] = c ? mfma_16<2>(keys, q[c][2 * k], s[c], q_scale) : mfma_16<0>(keys, q[c][2 * k], s[c], q_scale);
              bring(ahead, dma_place, next, 2 * k, more);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) asm volatile("" : "+v"(s[c]));  // (formed here, not where they are used)
        // lane (g, r): keys 16 wave + 4 g + j of head 16 c + r
        const uint32_t first_key = 16 * wave + here() / 16 * 4;
        f32x4 ks = {1.f, 1.f, 1.f, 1.f}, by;
        if (a.kv_scale) ks = *reinterpret_cast<const f32x4*>(&st.scale[first_key]);
#pragma unroll
        for (int j = 0; j < 4; ++j) by[j] = ks[j] * a.scale_log2;
        if (partial) {  // (a logit of minus infinity, whatever the scale's sign)
          const uint32_t mine = (uint32_t)(mask >> first_key);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            by[j] = mine >> j & 1 ? by[j] : 1.f;
#pragma unroll
            for (int c = 0; c < MT; ++c) s[c][j] = mine >> j & 1 ? s[c][j] : NEG_INF;
          }
        }
        float ps[MT];
        // (a logit is rounded before the maximum is taken from it, as the maximum was: at 2^31 one FMA for both
        // leaves half a step of the product, 2^7, and the largest key's own power overflows)
        const auto weigh = [&]() {  // the probabilities to LDS, and whether one of the workgroup's is over EXP2_SLACK
          uint16_t* to = &L.p[0][to_place];
          float top = 0.f;
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __builtin_amdgcn_exp2f(__fsub_rn(__fmul_rn(s[c][j], by[j]), m_ref[c]));
            ps[c] = (y[0] + y[1]) + (y[2] + y[3]);
            top = fmaxf(fmaxf(top, fmaxf(y[0], y[1])), fmaxf(y[2], y[3]));
            *reinterpret_cast<u32x2*>(to + c * 16 * P_PITCH) = u32x2{pack2(y[0] * ks[0], y[1] * ks[1]), pack2(y[2] * ks[2], y[3] * ks[3])};
            __builtin_amdgcn_sched_barrier(0);
          }
          const bool over = __any(top > EXP2_SLACK);
          if (lane == 0) L.over[wave] = over;
          meet();
          return __builtin_amdgcn_readfirstlane(L.over[0] | L.over[1] | L.over[2] | L.over[3]);
        };
        if (weigh()) {
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float m = NONE;
#pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, __fmul_rn(s[c][j], by[j]));
            m = groups_max(m);
            if (here() < 16) L.top[wave][16 * c + here()] = m;
          }
          meet();
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float m = m_ref[c];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, L.top[w][16 * c + here() % 16]);
            const float by = __builtin_amdgcn_exp2f(m_ref[c] - m);
            m_ref[c] = m;
            l_run[c] *= by;
            if (wave == 0 && here() < 16) L.by[16 * c + here()] = by;
          }
          weigh();
          const float by = L.by[here() % V::S];
#pragma unroll
          for (int b = 0; b < V::TILES; ++b)
#pragma unroll
            for (int i = 0; i < V::R; ++i) o[b][i] *= by;
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) l_run[c] += ps[c];

        // the values, transposed and widened: S dims x K keys against K keys x S heads
        {
          const uint16_t* pr = &L.p[0][from_place];
          const uint8_t* keys = &st.kv[value_place];
          constexpr int N = PAGE / V::K * V::TILES, VAHEAD = 4;  // (tile i % TILES of keys K (i / TILES) ..)
          u32x2 w[VAHEAD];
          bf16x8 pk[2];
          const auto read = [&](int i) {
            const int unit = i % V::TILES * MT;  // of 16 dims, four a block
            w[i % VAHEAD] = lds_transposed(keys + unit / 4 * BLOCK_BYTES + (value_swap ^ unit % 4 * 16) + i / V::TILES * V::K * 64);
          };
          const auto read_p = [&](int k) { pk[k % 2] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(pr + V::K * k)); };
          read_p(0);
#pragma unroll
          for (int i = 0; i < VAHEAD; ++i) read(i);
          const uint64_t rest = live & (live - 1);
          const int next_i = more ? __builtin_ctzll(live) : 0, after_i = __builtin_ctzll(rest ? rest : more ? live : 1);
          const uint64_t next_seen = L.seen[next_i];
          const int after_slot = L.slot[after_i];
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (i % V::TILES == 0 && i + V::TILES < N) read_p(i / V::TILES + 1);
            const bf16x8 v = widen8(w[i % VAHEAD]);
            if (i + VAHEAD < N) read(i + VAHEAD);
            o[i % V::TILES] = values_mfma(v, pk[i / V::TILES % 2], o[i % V::TILES]);
            __builtin_amdgcn_sched_barrier(0);
          }
          mask = seen_at(next_seen);
          ahead = (int64_t)__builtin_amdgcn_readfirstlane(after_slot) * PAGE;
        }
        buf ^= 1;
      }
      at += WAVE;
      if (at >= rd.hi) break;
      run_from(at);
    }
  }

  // the heads' sums: over the lane groups, then the waves
  const int tid = wave * WAVE + (int)here(), ln = tid % WAVE, heads = min(16 * MT, a.heads - h0);
  __syncthreads();  // (the last page's readers)
#pragma unroll
  for (int c = 0; c < MT; ++c) {
    const float l = groups_sum(l_run[c]);
    if (ln < 16) L.top[wave][16 * c + ln] = l;
    if (wave == 0 && ln < 16) L.by[16 * c + ln] = m_ref[c];
  }
  __syncthreads();
  const auto sum_of = [&](int head) { return (L.top[0][head] + L.top[1][head]) + (L.top[2][head] + L.top[3][head]); };
  // the outputs through LDS, so that rows go out whole
  const int head = ln % V::S, dim0 = 128 * wave + 4 * (ln / V::S);
  if (task.chunks > 1) {
    const int64_t first = task.part * a.heads + h0;  // this chunk's rows of the parts
    if (tid < heads) {
      const float l = sum_of(tid);
      a.part_m[first + tid] = l == 0.f ? NEG_INF : L.by[tid];
      a.part_l[first + tid] = l;
    }
    if (!any) return;
    float* stage = reinterpret_cast<float*>(&L.stage);
    constexpr int PITCH = LATENT + 4;
    static_assert(HEADS * PITCH * 4 <= sizeof L.stage, "the parts fit the pages' places");
#pragma unroll
    for (int b = 0; b < V::TILES; ++b)
#pragma unroll
      for (int i = 0; i < V::R / 4; ++i)
        *reinterpret_cast<f32x4*>(stage + head * PITCH + dim0 + V::S * b + 8 * i) = f32x4{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]};
    __syncthreads();
    float* part = a.part + first * LATENT;
    for (int u = tid; u < heads * (LATENT / 4); u += T)
      *reinterpret_cast<f32x4*>(part + 4 * u) = *reinterpret_cast<const f32x4*>(stage + u / (LATENT / 4) * PITCH + u % (LATENT / 4) * 4);
    return;
  }
  uint16_t* stage = reinterpret_cast<uint16_t*>(&L.stage);
  constexpr int PITCH = LATENT + 8;
  const float l = sum_of(head), inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int b = 0; b < V::TILES; ++b)
#pragma unroll
    for (int i = 0; i < V::R / 4; ++i)
      *reinterpret_cast<u32x2*>(stage + head * PITCH + dim0 + V::S * b + 8 * i) =
          u32x2{pack2(o[b][4 * i] * inv, o[b][4 * i + 1] * inv), pack2(o[b][4 * i + 2] * inv, o[b][4 * i + 3] * inv)};
  __syncthreads();
  uint16_t* out = static_cast<uint16_t*>(a.out) + (t * a.heads + h0) * LATENT;
  for (int u = tid; u < heads * (LATENT / 8); u += T)
    *reinterpret_cast<u32x4*>(out + 8 * u) = *reinterpret_cast<const u32x4*>(stage + u / (LATENT / 8) * PITCH + u % (LATENT / 8) * 8);
}

// Which task workgroup b takes; it runs on XCD b mod 8. Neighbouring tasks read many of the same
// pages, which one L2 then holds, so an XCD takes BLOCK of them in a row; and all XCDs go through
// the tokens together and from the last one down, since a prompt's later tokens have more pages:
// the short tasks are left for the end (600 tokens from position 0: an eighth of the tokens for each
// XCD 52 us, single tokens 40, fours 39.5, fours from the last 29, sixty-fours from the last 41; 4096
// tokens of 5 requests 410, 310, 303, 298, 307).
constexpr int BLOCK = 4;
MONO_DEV int64_t task_id(uint32_t b, int64_t tasks) {
  const uint32_t i = b / 8;
  return tasks - 1 - ((int64_t)(i / BLOCK * 8 + b % 8) * BLOCK + i % BLOCK);
}

template <int MT, bool TREE, bool PLANNED>
__global__ __launch_bounds__(T, 2) void k_pages(Paged a) {
  __shared__ Lds L;
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  int64_t tasks = a.work;
  int pages = 0;
  Requests requests;
  if (PLANNED) {
    for (int64_t t = (int64_t)blockIdx.x * T + threadIdx.x; t < a.tokens; t += (int64_t)gridDim.x * T)
      if (t < a.starts[0] || t >= a.starts[a.requests]) a.plan[t] = NodePlan{0, 0};  // nodes of no request
    each_set(a, [&](int i) { requests.of[i] = request_of(a, WAVE * i + lane); });
    pages = chunk_pages(a, requests, tasks);
  }
  const int64_t id = task_id(blockIdx.x, tasks);
  if (id < 0) return;
  Task task;
  Reads rd;
  if (!PLANNED)
    task_of<TREE>(a, lane, id, task, rd);
  else {
    if (!planned_task(a, requests, pages, (int)id, task, rd)) return;
    if (threadIdx.x == 0 && task.ht == 0 && task.chunk == 0) a.plan[task.t] = NodePlan{task.chunks, (int)task.part};
  }
  attend<MT, TREE>(a, L, lane, wave, task, rd);
}

// A head's parts as one, each scaled to the largest of their maxima, in the parts' order. Wave w of
// W takes every W-th part, eight of them in flight; the waves' sums meet in LDS. A workgroup takes
// 512 / S dims of a head, or H heads, a wave each.
constexpr int MAX_SPLITS = FULL + 1, JOIN_AHEAD = 8;  // (a node alone beside FULL more tasks)
template <int W, int S, int H>
__global__ __launch_bounds__(W * H * WAVE) void k_join(Paged a) {
  static_assert(W == 1 || H == 1, "waves share a head or have one each");
  constexpr int N = LATENT / S, V = N / WAVE;  // dims: of the workgroup, of a lane
  typedef float Vec __attribute__((ext_vector_type(V < 4 ? V : 4)));
  constexpr int VECS = V < 4 ? 1 : V / 4, EACH = V / VECS;
  __shared__ float weights[H][MAX_SPLITS + JOIN_AHEAD * W];
  __shared__ alignas(16) float sums[W * H][N];
  const int lane = threadIdx.x % WAVE, wv = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), wave = wv % W, tid = WAVE * wave + lane;
  float* by = weights[wv / W];
  const auto meet_waves = [&]() {
    if (W > 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  const int64_t row = (int64_t)(blockIdx.x / S) * H + wv / W, t = row / a.heads;
  const int slice = blockIdx.x % S, h = (int)(row % a.heads);
  if (t >= a.tokens) return;
  int splits = a.splits;
  int64_t part = t * a.splits;
  if (a.plan) {
    const NodePlan p = a.plan[t];
    splits = p.chunks, part = p.part;
    if (splits == 1) return;  // it was written whole
    if (splits < 0 || splits > MAX_SPLITS || part < 0 || part + splits > a.parts) splits = 0;  // (starts that do not ascend)
  }
  const int64_t step = a.heads, first = part * step + h;
  float m = NEG_INF, l = 0.f;
  for (int s = lane; s < splits; s += WAVE) m = fmaxf(m, a.part_m[first + s * step]);
  m = wave_max(m);
  for (int s = lane; s < splits; s += WAVE) {
    const float ps = a.part_l[first + s * step], w = __builtin_amdgcn_exp2f(a.part_m[first + s * step] - m);
    l += ps == 0.f ? 0.f : ps * w;
    if (wave == 0) by[s] = ps == 0.f ? -1.f : w;  // -1: it saw nothing and wrote nothing
  }
  if (wave == 0)
    for (int i = lane; i < JOIN_AHEAD * W; i += WAVE) by[splits + i] = -1.f;
  l = wave_sum(l);
  meet_waves();
  float o[V] = {};
  for (int s0 = wave; s0 < splits; s0 += JOIN_AHEAD * W) {
    Vec v[JOIN_AHEAD][VECS];
#pragma unroll
    for (int i = 0; i < JOIN_AHEAD; ++i) {
      const float* row = a.part + (first + min(s0 + i * W, splits - 1) * step) * LATENT + N * slice + EACH * lane;
#pragma unroll
      for (int j = 0; j < VECS; ++j) v[i][j] = *reinterpret_cast<const Vec*>(row + N / VECS * j);
    }
#pragma unroll
    for (int i = 0; i < JOIN_AHEAD; ++i) {
      const float w = by[s0 + i * W];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = w == -1.f ? o[j] : fmaf(v[i][j / EACH][j % EACH], w, o[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sums[wv][N / VECS * (j / EACH) + EACH * lane + j % EACH] = o[j];
  meet_waves();
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint32_t* out = static_cast<uint32_t*>(a.out) + (t * a.heads + h) * (LATENT / 2) + N / 2 * slice;
  for (int u = tid; u < N / 2; u += W * WAVE) {
    float r[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) r[0] += sums[wv - wave + w][2 * u], r[1] += sums[wv - wave + w][2 * u + 1];
    out[u] = pack2(r[0] * inv, r[1] * inv);
  }
}

}  // namespace

hipError_t paged_attention(const Paged& a, hipStream_t st) {
  const auto launch = [&](auto kernel) {
    kernel<<<(uint32_t)((a.work + 8 * BLOCK - 1) / (8 * BLOCK) * (8 * BLOCK)), T, 0, st>>>(a);
    return hipGetLastError();
  };
  if (!a.starts) return launch(a.head_rows == 16 ? k_pages<1, false, false> : k_pages<2, false, false>);
  if (a.plan) return launch(a.head_rows == 16 ? k_pages<1, true, true> : k_pages<2, true, true>);
  return launch(a.head_rows == 16 ? k_pages<1, true, false> : k_pages<2, true, false>);
}

hipError_t join_attention(const Paged& a, hipStream_t st) {
  const int64_t heads = a.tokens * a.heads;
  // Few heads have many parts each, and too few workgroups: four waves each and four workgroups
  // (attention and join: 1 node of 32 heads, 20000 keys 19.0 us, one wave 26.9; 4 nodes 26.7 and 30.8).
  // From 512 heads on one wave does (16 nodes, 1000 keys 23.1 and 23.9, 64 nodes 32.3 and 42.0). Of
  // thousands of heads most were written whole: four a workgroup (1000 nodes, 500 keys 64 us and 68, but
  // 16 nodes 24.9 and 22.3).
  if (heads <= 256)
    k_join<4, 4, 1><<<(uint32_t)(4 * heads), 4 * WAVE, 0, st>>>(a);
  else if (heads <= 2048)
    k_join<1, 1, 1><<<(uint32_t)heads, WAVE, 0, st>>>(a);
  else
    k_join<1, 1, 4><<<(uint32_t)((heads + 3) / 4), 4 * WAVE, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
