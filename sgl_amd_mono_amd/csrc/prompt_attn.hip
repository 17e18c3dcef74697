// MLA attention over pages of the latent cache: of the pages that each token selected
// (attention), and of a whole prefix with the drafted tokens that a mask leaves (tree).
//
//   s[h, j] = scale kvs[j] (q[h] . c[j]),  576 dims;  out[h] = sum_j softmax_j(s) kvs[j] c[j, :512]
//
// A workgroup takes a token and up to 32 of its heads, and walks through pages of 64 keys with
// a running maximum and sum. A page is one piece of 36 KB, brought to LDS as it lies by DMA
// (global_load_lds), the next one while this one is worked on, and read from there twice: as
// rows for q . c and transposed (ds_read_b64_tr_b8) for p . v, widened to bf16 in registers
// each time, exactly.
//
//   q . c   wave w: keys 16 w .. + 15 against every head, whose q stays in registers
//   p . v   wave w: dims 128 w .. + 127 over all 64 keys; the probabilities meet in LDS
//
// The maximum that the sums refer to stays as it is until a logit passes it by 2^8 (a ratio of
// sums does not depend on it, bf16 and f32 hold 2^8 as well as 1): the waves' maxima then meet
// and the sums are scaled, which happens on a token's first page and rarely after it.
//
// Probabilities are rounded to bf16 for the matrix unit, 2^-9 of each at random beside the
// output's own 2^-9; their sum adds up the f32 values.
#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int T = 256, WAVES = 4, ROW = LATENT + PE, PAGE_BYTES = PAGE * ROW;
constexpr int BLOCKS = ROW / 64, BLOCK_BYTES = PAGE * 64;  // a page's rows in blocks of 64 dims
constexpr int DT = LATENT / WAVES / 16;                   // tiles of 16 dims a wave
constexpr int AHEAD = 2;                                  // blocks read before they are used
// NONE: no maximum yet, so low that any logit passes it (and finite: what is taken from it is a number)
constexpr float NEG_INF = -__builtin_inff(), NONE = -1e38f, SLACK = 8.0f;

// A page and its keys' scales.
struct Stage {
  alignas(16) uint8_t kv[PAGE_BYTES];
  float scale[PAGE];
};
template <int MT>
struct Lds {
  Stage stage[2];
  alignas(16) uint16_t p[16 * MT][PAGE + 8];
  float top[WAVES][16 * MT], sum[WAVES][16 * MT];
  int over[WAVES];
  int slot[WAVE];       // a run of 64 pages of the list: where each lies in the pool
  uint64_t seen[WAVE];  // and which of its keys are seen
};

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

MONO_DEV bf16x8 widen8(uint32_t lo, uint32_t hi) {
  bf16x8 v;
  widen4(lo, v, 0);
  widen4(hi, v, 4);
  return v;
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

// What a workgroup reads: a token's pages [lo, hi) of its list (attention) or of its request's
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

template <bool TREE>
MONO_DEV bool reads_of(const Paged& a, int64_t t, int split, Reads& rd) {
  int pages;
  if (TREE) {
    // the request whose nodes hold t: as many starts as are at most t
    const int lane = threadIdx.x % WAVE;
    int req = -1, at = 0;
    for (int r0 = 0; r0 <= a.requests; r0 += WAVE) at += __popcll(__ballot(r0 + lane <= a.requests && a.starts[min(r0 + lane, a.requests)] <= t));
    req = at - 1;
    if (req < 0 || req >= a.requests) return false;
    rd.table = a.page_table + (int64_t)req * a.pt_stride;
    rd.end = max(a.prefix[req], 0);
    rd.draft = (uint64_t)a.mask[t];
    const int drafted = rd.draft ? 64 - __builtin_clzll(rd.draft) : 0;
    pages = (int)min((int64_t)a.pt_stride, (rd.end + drafted + PAGE - 1) / PAGE);
  } else {
    const int req = a.req[t], pos = a.pos[t];
    if (req < 0 || req >= a.requests || pos < 0) return false;
    rd.table = a.page_table + (int64_t)req * a.pt_stride;
    rd.list = a.pages + t * a.picks;
    rd.end = (int64_t)pos + 1;
    rd.draft = 0;
    pages = a.picks;
  }
  rd.lo = (int)((int64_t)pages * split / a.splits);
  rd.hi = (int)((int64_t)pages * (split + 1) / a.splits);
  return rd.lo < rd.hi;
}

template <int MT, bool TREE>
__global__ __launch_bounds__(T, 2) void k_pages(Paged a) {
  __shared__ Lds<MT> L;
  const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  // the XCDs (workgroup b runs on XCD b mod 8) take neighbouring work each: neighbouring tokens
  // read many of the same pages, which one L2 then holds
  const int64_t each = (a.work + 7) / 8, id = blockIdx.x % 8 * each + blockIdx.x / 8;
  if (blockIdx.x / 8 >= each || id >= a.work) return;
  const int ht = (int)(id % a.head_tiles);
  const int64_t rest = id / a.head_tiles;
  // attention: a token's splits side by side; tree: a split's nodes
  const int64_t t = TREE ? rest % a.tokens : rest / a.splits;
  const int split = (int)(TREE ? rest / a.tokens : rest % a.splits), h0 = ht * 16 * MT;
  Reads rd;
  const bool any = reads_of<TREE>(a, t, split, rd);

  f32x4 o[DT][MT];
  float m_ref[MT], l_run[MT];
#pragma unroll
  for (int c = 0; c < MT; ++c) {
    m_ref[c] = NONE, l_run[c] = 0.f;
#pragma unroll
    for (int b = 0; b < DT; ++b) o[b][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (any) {
    int buf = 0;
    uint64_t live = 0;  // pages left of a run of 64 of the list
    // page i's way to LDS: this wave's 16 keys, a block of dims at a time, and the scales
    const auto place_of = [&](int i) { return (int64_t)__builtin_amdgcn_readfirstlane(L.slot[i]) * PAGE; };
    const auto lane_place = [&]() {
      const uint32_t ln = lane_now(lane);
      return ln / 4 * ROW + 16 * unit_of(ln / 4, ln % 4);
    };
    const auto bring = [&](int64_t first, uint32_t at, Stage& to, int b, bool go) {
      dma16(static_cast<const uint8_t*>(a.kv) + (first + 16 * wave) * ROW + 64 * b, at, &to.kv[b * BLOCK_BYTES + wave * 1024], go);
    };
    const auto bring_scales = [&](int64_t first, Stage& to) {
      if (wave == 0 && a.kv_scale) dma4(a.kv_scale + first, 4 * lane_now(lane), to.scale);
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
    bf16x8 q[MT][2 * BLOCKS];  // (behind the first page, which more steps led to)
    {
      const uint32_t ln = lane_now(lane), r = ln % 16, g = ln / 16;
      // q of heads 16 c + r: dims 64 b + 16 g + 8 h .. + 7 (the order in which a lane reads a row's units)
#pragma unroll
      for (int c = 0; c < MT; ++c) {
        const uint16_t* row = static_cast<const uint16_t*>(a.q) + (t * a.heads + min(h0 + 16 * c + (int)r, a.heads - 1)) * ROW + 16 * g;
#pragma unroll
        for (int k = 0; k < 2 * BLOCKS; ++k) q[c][k] = __builtin_bit_cast(bf16x8, ld_u32x4(row + 64 * (k / 2) + 8 * (k % 2)));
      }
    }
    for (;;) {
      while (live) {  // a page, while the next one of the run comes
        Stage &st = L.stage[buf], &next = L.stage[buf ^ 1];
        const int i = __builtin_ctzll(live);
        live &= live - 1;
        meet_after_loads();  // the page has come, and every wave is done with the one before
        const uint64_t seen_here = L.seen[i];
        const uint64_t mask = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)seen_here) |
                              (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(seen_here >> 32)) << 32;
        const bool partial = mask != ~0ull;
        if (partial) {  // what is not seen may hold anything, a NaN too: zeros instead
          const uint32_t ln = lane_now(lane);
          if (!(mask >> (16 * wave + ln / 4) & 1))
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) *reinterpret_cast<u32x4*>(&st.kv[b * BLOCK_BYTES + 1024 * wave + 16 * ln]) = u32x4{0u, 0u, 0u, 0u};
          meet();
        }
        const bool more = live != 0;
        const int64_t ahead = place_of(more ? __builtin_ctzll(live) : i);
        if (more) bring_scales(ahead, next);

        f32x4 s[MT];
#pragma unroll
        for (int c = 0; c < MT; ++c) s[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        {
          const uint32_t ln = lane_now(lane);
          const uint32_t at_lane = lane_place();
          const uint8_t* key = &st.kv[(16 * wave + ln % 16) * 64 + 16 * unit_of(ln % 16, ln / 16)];
          u32x4 w[AHEAD];  // (the order of reads, conversions and MFMAs is held: left alone, each read is waited for at once)
#pragma unroll
          for (int b = 0; b < AHEAD; ++b) w[b] = *reinterpret_cast<const u32x4*>(key + BLOCK_BYTES * b);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) {
            const bf16x8 k0 = widen8(w[b % AHEAD][0], w[b % AHEAD][1]);
#pragma unroll
            for (int c = 0; c < MT; ++c) s[c] = mfma_bf16(k0, q[c][2 * b], s[c]);
            __builtin_amdgcn_sched_barrier(0);
            const bf16x8 k1 = widen8(w[b % AHEAD][2], w[b % AHEAD][3]);
            if (b + AHEAD < BLOCKS) w[b % AHEAD] = *reinterpret_cast<const u32x4*>(key + BLOCK_BYTES * (b + AHEAD));
#pragma unroll
            for (int c = 0; c < MT; ++c) s[c] = mfma_bf16(k1, q[c][2 * b + 1], s[c]);
            bring(ahead, at_lane, next, b, more);  // (nine DMAs at once hold the wave up for 1000 cycles)
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        // lane (g, r): keys 16 wave + 4 g + j of head 16 c + r
        const uint32_t first_key = 16 * wave + lane_now(lane) / 16 * 4;
        f32x4 ks = {1.f, 1.f, 1.f, 1.f}, by;
        if (a.kv_scale) ks = *reinterpret_cast<const f32x4*>(&st.scale[first_key]);
        const uint32_t mine = partial ? (uint32_t)(mask >> first_key) : 15u;
        if (partial)
#pragma unroll
          for (int j = 0; j < 4; ++j) ks[j] = mine >> j & 1 ? ks[j] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) by[j] = ks[j] * a.scale_log2;
        float ps[MT];
        const auto weigh = [&]() {  // the probabilities to LDS, and whether one is over 2^SLACK
          const uint32_t ln = lane_now(lane);
          float top = NEG_INF;
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = fmaf(s[c][j], by[j], -m_ref[c]);
            if (partial)
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = mine >> j & 1 ? y[j] : NEG_INF;
            top = fmaxf(fmaxf(top, fmaxf(y[0], y[1])), fmaxf(y[2], y[3]));
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __builtin_amdgcn_exp2f(y[j]);
            ps[c] = (y[0] + y[1]) + (y[2] + y[3]);
            *reinterpret_cast<u32x2*>(&L.p[16 * c + ln % 16][16 * wave + 4 * (ln / 16)]) =
                u32x2{pack2(y[0] * ks[0], y[1] * ks[1]), pack2(y[2] * ks[2], y[3] * ks[3])};
          }
          return top > SLACK;
        };
        const bool over = __any(weigh());
        if (lane == 0) L.over[wave] = over;
        meet();
        const int any_over = L.over[0] | L.over[1] | L.over[2] | L.over[3];
        // the values, transposed: dims 128 wave + 16 b .. of 32 keys a step; the first reads already here
        constexpr int N = PAGE / 32 * DT, VAHEAD = 4;
        u32x2 vw[VAHEAD];
        const auto value_place = [&]() {
          const uint32_t ln = lane_now(lane);
          return &st.kv[2 * wave * BLOCK_BYTES + (8 * (ln / 16) + ln % 16 / 2) * 64 + 8 * (ln % 2)];
        };
        const auto read = [&](const uint8_t* keys, uint32_t swap, int i) {
          vw[i % VAHEAD] = lds_transposed(keys + i / DT * 2048 + i % DT / 4 * BLOCK_BYTES + 16 * (swap ^ i % 4));
        };
        const auto first_reads = [&]() {
          const uint8_t* keys = value_place();
          const uint32_t swap = unit_of(lane_now(lane) % 16 / 2, 0);
#pragma unroll
          for (int i = 0; i < VAHEAD; ++i) read(keys, swap, i);
        };
        first_reads();
        if (__builtin_amdgcn_readfirstlane(any_over)) {
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float m = NONE;
#pragma unroll
            for (int j = 0; j < 4; ++j) m = fmaxf(m, mine >> j & 1 ? s[c][j] * by[j] : NONE);
            m = groups_max(m);
            if (lane_now(lane) < 16) L.top[wave][16 * c + lane_now(lane)] = m;
          }
          meet();
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float m = m_ref[c];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, L.top[w][16 * c + lane_now(lane) % 16]);
            const float by = __builtin_amdgcn_exp2f(m_ref[c] - m);
            m_ref[c] = m;
            l_run[c] *= by;
#pragma unroll
            for (int b = 0; b < DT; ++b)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[b][c][j] *= by;
          }
          weigh();
          meet();
          first_reads();  // (again: held across this path they would spill)
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) l_run[c] += ps[c];

        {
          const uint8_t* keys = value_place();
          const uint32_t ln = lane_now(lane), swap = unit_of(ln % 16 / 2, 0);
          bf16x8 pk[MT];
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (i % DT == 0) {
#pragma unroll
              for (int c = 0; c < MT; ++c)
                pk[c] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(&L.p[16 * c + ln % 16][32 * (i / DT) + 8 * (ln / 16)]));
            }
            const bf16x8 v = widen8(vw[i % VAHEAD][0], vw[i % VAHEAD][1]);
            if (i + VAHEAD < N) read(keys, swap, i + VAHEAD);
#pragma unroll
            for (int c = 0; c < MT; ++c) o[i % DT][c] = mfma_bf16(v, pk[c], o[i % DT][c]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        buf ^= 1;
      }
      at += WAVE;
      if (at >= rd.hi) break;
      run_from(at);
    }
  }

  const int tid = wave * WAVE + (int)lane_now(lane), g = tid % WAVE / 16, r = tid % 16;
  // the heads' sums: over the lane groups, then the waves
  float l[MT];
  __syncthreads();  // (the last page's readers)
#pragma unroll
  for (int c = 0; c < MT; ++c) {
    l[c] = groups_sum(l_run[c]);
    if (g == 0) L.sum[wave][16 * c + r] = l[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < MT; ++c) {
    l[c] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) l[c] += L.sum[w][16 * c + r];
  }
  const int heads = min(16 * MT, a.heads - h0);
  if (a.splits > 1) {
    const int64_t first = (t * a.splits + split) * a.heads + h0;  // this split's rows of the parts
    if (wave == 0 && g == 0)
#pragma unroll
      for (int c = 0; c < MT; ++c)
        if (16 * c + r < heads) {
          a.part_m[first + 16 * c + r] = l[c] == 0.f ? NEG_INF : m_ref[c];
          a.part_l[first + 16 * c + r] = l[c];
        }
    if (!any) return;
#pragma unroll
    for (int c = 0; c < MT; ++c)
      if (16 * c + r < heads)
#pragma unroll
        for (int b = 0; b < DT; ++b)
          *reinterpret_cast<f32x4*>(a.part + (first + 16 * c + r) * LATENT + 16 * (DT * wave + b) + 4 * g) = o[b][c];
    return;
  }
  // through LDS, so that rows go out whole
  uint16_t* stage = reinterpret_cast<uint16_t*>(L.stage[0].kv);
  constexpr int PITCH = LATENT + 8;
  static_assert(16 * MT * PITCH * 2 <= PAGE_BYTES, "the outputs fit a page's place");
#pragma unroll
  for (int c = 0; c < MT; ++c) {
    const float by = l[c] == 0.f ? 0.f : 1.0f / l[c];
#pragma unroll
    for (int b = 0; b < DT; ++b)
      *reinterpret_cast<u32x2*>(stage + (16 * c + r) * PITCH + 16 * (DT * wave + b) + 4 * g) =
          u32x2{pack_bf16x2(o[b][c][0] * by, o[b][c][1] * by), pack_bf16x2(o[b][c][2] * by, o[b][c][3] * by)};
  }
  __syncthreads();
  uint16_t* out = static_cast<uint16_t*>(a.out) + (t * a.heads + h0) * LATENT;
  for (int u = tid; u < heads * (LATENT / 8); u += T)
    *reinterpret_cast<u32x4*>(out + 8 * u) = *reinterpret_cast<const u32x4*>(stage + u / (LATENT / 8) * PITCH + u % (LATENT / 8) * 8);
}

// A head's parts as one, each scaled to the largest of their maxima. A wave takes every fourth
// part, eight of them in flight; the waves' sums meet in LDS.
constexpr int MAX_SPLITS = 512, JOIN_AHEAD = 8;
__global__ __launch_bounds__(T) void k_join(Paged a) {
  __shared__ float by[MAX_SPLITS + JOIN_AHEAD * WAVES];
  __shared__ alignas(16) float sums[WAVES][LATENT];
  const int tid = threadIdx.x, lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int64_t t = blockIdx.x / a.heads;
  const int h = blockIdx.x % a.heads;
  const int64_t step = a.heads, first = t * a.splits * step + h;
  float m = NEG_INF, l = 0.f;
  for (int s = lane; s < a.splits; s += WAVE) m = fmaxf(m, a.part_m[first + s * step]);
  m = wave_max(m);
  for (int s = lane; s < a.splits; s += WAVE) {
    const float ps = a.part_l[first + s * step], w = __builtin_amdgcn_exp2f(a.part_m[first + s * step] - m);
    l += ps == 0.f ? 0.f : ps * w;
    if (wave == 0) by[s] = ps == 0.f ? -1.f : w;  // -1: it saw nothing and wrote nothing
  }
  if (wave == 0 && lane < JOIN_AHEAD * WAVES) by[a.splits + lane] = -1.f;
  l = wave_sum(l);
  __syncthreads();
  float o[8] = {};
  for (int s0 = wave; s0 < a.splits; s0 += JOIN_AHEAD * WAVES) {
    f32x4 v[JOIN_AHEAD][2];
#pragma unroll
    for (int i = 0; i < JOIN_AHEAD; ++i) {
      const float* row = a.part + (first + min(s0 + i * WAVES, a.splits - 1) * step) * LATENT + 8 * lane;
      v[i][0] = *reinterpret_cast<const f32x4*>(row);
      v[i][1] = *reinterpret_cast<const f32x4*>(row + 4);
    }
#pragma unroll
    for (int i = 0; i < JOIN_AHEAD; ++i) {
      const float w = by[s0 + i * WAVES];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = w == -1.f ? o[j] : fmaf(v[i][j / 4][j % 4], w, o[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) *reinterpret_cast<f32x4*>(&sums[wave][8 * lane + 4 * j]) = f32x4{o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]};
  __syncthreads();
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  float r[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    r[j] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) r[j] += sums[w][2 * tid + j];
  }
  reinterpret_cast<uint32_t*>(a.out)[((t * a.heads + h) * LATENT) / 2 + tid] = pack_bf16x2(r[0] * inv, r[1] * inv);
}

}  // namespace

hipError_t paged_attention(const Paged& a, hipStream_t st) {
  const uint32_t grid = (uint32_t)((a.work + 7) / 8 * 8);
  const bool tree = a.starts != nullptr;
  if (a.head_rows == 16) {
    if (tree) k_pages<1, true><<<grid, T, 0, st>>>(a);
    else k_pages<1, false><<<grid, T, 0, st>>>(a);
  } else {
    if (tree) k_pages<2, true><<<grid, T, 0, st>>>(a);
    else k_pages<2, false><<<grid, T, 0, st>>>(a);
  }
  return hipGetLastError();
}

hipError_t join_attention(const Paged& a, hipStream_t st) {
  k_join<<<(uint32_t)(a.tokens * a.heads), T, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
