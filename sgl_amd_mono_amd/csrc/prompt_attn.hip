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
constexpr int UNITS = ROW / 16, BLOCKS = ROW / 64;  // 16-byte pieces and 64-dim blocks of a row
constexpr int DT = LATENT / WAVES / 16;             // tiles of 16 dims a wave
constexpr int DMAS = PAGE_BYTES / 16 / T;           // 16-byte pieces a thread and page
static_assert(PAGE_BYTES == DMAS * 16 * T, "whole DMA turns");
constexpr float NEG_INF = -__builtin_inff(), SLACK = 8.0f;

template <int MT>
struct Lds {
  alignas(16) uint8_t kv[2][PAGE_BYTES];  // (the outputs' rows at the end)
  uint16_t p[16 * MT][PAGE + 8];
  float top[WAVES][16 * MT], sum[WAVES][16 * MT];
  int over[WAVES];
};

typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

// 16 lanes read 8 rows x 16 bytes of LDS transposed: lane l gives the address of bytes
// 8 (l % 2) .. of row l / 2 and gets byte l of each of the 8 rows.
MONO_DEV u32x2 lds_transposed(const uint8_t* p) { return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)p)); }

MONO_DEV bf16x8 widen8(uint32_t lo, uint32_t hi) {
  bf16x8 v;
  widen4(lo, v, 0);
  widen4(hi, v, 4);
  return v;
}

// Where unit u of row `row` lies in LDS: within its four units swapped by the row's number / 4,
// so that 16 rows' same unit (their rows are 16 banks apart, mod 64) and 8 rows' two units of a
// transposed read meet no bank twice.
MONO_DEV int unit_of(int row, int u) { return u ^ (row >> 2 & 3); }

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
  const int tid = threadIdx.x, lane = tid % WAVE, g = lane / 16, r = lane % 16, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
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
    m_ref[c] = NEG_INF, l_run[c] = 0.f;
#pragma unroll
    for (int b = 0; b < DT; ++b) o[b][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (any) {
    // q of heads 16 c + r: dims 64 b + 16 g + 8 h .. + 7 (the order in which a lane reads a row's units)
    bf16x8 q[MT][2 * BLOCKS];
#pragma unroll
    for (int c = 0; c < MT; ++c) {
      const uint16_t* row = static_cast<const uint16_t*>(a.q) + (t * a.heads + min(h0 + 16 * c + r, a.heads - 1)) * ROW + 16 * g;
#pragma unroll
      for (int k = 0; k < 2 * BLOCKS; ++k) q[c][k] = __builtin_bit_cast(bf16x8, ld_u32x4(row + 64 * (k / 2) + 8 * (k % 2)));
    }
    int buf = 0;
    for (int at = rd.lo; at < rd.hi; at += WAVE) {
      // lane l: page at + l of the list, where it lies and what of it is seen
      int page = -1, slot = -1;
      if (at + lane < rd.hi) page = TREE ? at + lane : rd.list[at + lane];
      uint64_t seen = 0;
      if (page >= 0 && page < a.pt_stride) {
        slot = rd.table[page];
        if (slot >= 0 && slot < a.n_pages) seen = seen_of(rd, page, TREE);
      }
      uint64_t live = __ballot(seen != 0);
      const auto bring = [&](int i, int to, f32x4& scale) {
        const int64_t first = (int64_t)__builtin_amdgcn_readlane(slot, i) * PAGE;
        const uint8_t* from = static_cast<const uint8_t*>(a.kv) + first * ROW;
#pragma unroll
        for (int k = 0; k < DMAS; ++k) {
          const int u = k * T + tid, row = u / UNITS;
          __builtin_amdgcn_global_load_lds((gvoid*)(from + row * ROW + 16 * unit_of(row, u % UNITS)),
                                           (lvoid*)(&L.kv[to][(k * T + wave * WAVE) * 16]), 16, 0, 0);
        }
        scale = a.kv_scale ? *reinterpret_cast<const f32x4*>(a.kv_scale + first + 16 * wave + 4 * g) : f32x4{1.f, 1.f, 1.f, 1.f};
      };
      f32x4 next;
      if (live) bring(__builtin_ctzll(live), buf, next);
      while (live) {
        const int i = __builtin_ctzll(live);
        live &= live - 1;
        const uint64_t mask = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)seen, i) |
                              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(seen >> 32), i) << 32;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // the page has come, and every wave is done with the one before
        f32x4 ks = next;
        if (mask != ~0ull) {  // what is not seen may hold anything, a NaN too: zeros instead
          for (int u = tid; u < PAGE * UNITS; u += T)
            if (!(mask >> (u / UNITS) & 1)) *reinterpret_cast<u32x4*>(&L.kv[buf][16 * u]) = u32x4{0u, 0u, 0u, 0u};
          __syncthreads();
        }
        if (live) bring(__builtin_ctzll(live), buf ^ 1, next);

        f32x4 s[MT];
#pragma unroll
        for (int c = 0; c < MT; ++c) s[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        const uint8_t* kv = L.kv[buf];
        {
          const int row = 16 * wave + r;
          const uint8_t* key = kv + row * ROW + 16 * unit_of(row, g);
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(key + 64 * b);
            const bf16x8 k0 = widen8(w[0], w[1]), k1 = widen8(w[2], w[3]);
#pragma unroll
            for (int c = 0; c < MT; ++c) {
              s[c] = mfma_bf16(k0, q[c][2 * b], s[c]);
              s[c] = mfma_bf16(k1, q[c][2 * b + 1], s[c]);
            }
          }
        }
        // lane (g, r): keys 16 wave + 4 g + j of head 16 c + r, in units of log2
        const uint32_t mine = (uint32_t)(mask >> (16 * wave + 4 * g)) & 15u;
        float p[MT][4], top[MT];
        bool over = false;
#pragma unroll
        for (int c = 0; c < MT; ++c) {
          top[c] = NEG_INF;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[c][j] = mine >> j & 1 ? s[c][j] * (ks[j] * a.scale_log2) : NEG_INF;
            top[c] = fmaxf(top[c], s[c][j]);
          }
          over |= top[c] > m_ref[c] + SLACK;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) ks[j] = mine >> j & 1 ? ks[j] : 0.f;
        const auto store_p = [&]() {
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            const float ref = m_ref[c] == NEG_INF ? 0.f : m_ref[c];
#pragma unroll
            for (int j = 0; j < 4; ++j) p[c][j] = __builtin_amdgcn_exp2f(s[c][j] - ref);
            *reinterpret_cast<u32x2*>(&L.p[16 * c + r][16 * wave + 4 * g]) =
                u32x2{pack_bf16x2(p[c][0] * ks[0], p[c][1] * ks[1]), pack_bf16x2(p[c][2] * ks[2], p[c][3] * ks[3])};
          }
        };
        store_p();
        const bool mine_over = __any(over);
        if (lane == 0) L.over[wave] = mine_over;
        __syncthreads();
        if (L.over[0] | L.over[1] | L.over[2] | L.over[3]) {
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            const float m = groups_max(top[c]);
            if (g == 0) L.top[wave][16 * c + r] = m;
          }
          __syncthreads();
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            float m = m_ref[c];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, L.top[w][16 * c + r]);
            const float by = m_ref[c] == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(m_ref[c] - m);
            m_ref[c] = m;
            l_run[c] *= by;
#pragma unroll
            for (int b = 0; b < DT; ++b)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[b][c][j] *= by;
          }
          store_p();
          __syncthreads();
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) l_run[c] += (p[c][0] + p[c][1]) + (p[c][2] + p[c][3]);

        // dims 128 wave + 16 b .. of the values, transposed, against 32 keys' probabilities a step
#pragma unroll
        for (int k = 0; k < PAGE / 32; ++k) {
          bf16x8 pk[MT];
#pragma unroll
          for (int c = 0; c < MT; ++c) pk[c] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(&L.p[16 * c + r][32 * k + 8 * g]));
          const int row = 32 * k + 8 * g + r / 2;
          const uint8_t* at_row = kv + row * ROW + 8 * (r % 2);
#pragma unroll
          for (int b = 0; b < DT; ++b) {
            const u32x2 w = lds_transposed(at_row + 16 * unit_of(row, DT * wave + b));
            const bf16x8 v = widen8(w[0], w[1]);
#pragma unroll
            for (int c = 0; c < MT; ++c) o[b][c] = mfma_bf16(v, pk[c], o[b][c]);
          }
        }
        buf ^= 1;
      }
    }
  }

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
  uint16_t* stage = reinterpret_cast<uint16_t*>(L.kv[0]);
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

// A head's parts as one: each scaled to the largest of their maxima.
__global__ __launch_bounds__(LATENT / 4) void k_join(Paged a) {
  const int64_t t = blockIdx.x / a.heads;
  const int h = blockIdx.x % a.heads;
  const int64_t step = a.heads, first = t * a.splits * step + h;
  float m = NEG_INF, l = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_m[first + s * step]);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float ps = a.part_l[first + s * step];
    if (ps == 0.f) continue;  // it saw nothing and wrote nothing
    const float by = __builtin_amdgcn_exp2f(a.part_m[first + s * step] - m);
    l = fmaf(ps, by, l);
    const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + (first + s * step) * LATENT + 4 * threadIdx.x);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = fmaf(v[j], by, o[j]);
  }
  const float by = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + (t * a.heads + h) * LATENT + 4 * threadIdx.x) =
      u32x2{pack_bf16x2(o[0] * by, o[1] * by), pack_bf16x2(o[2] * by, o[3] * by)};
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
  k_join<<<(uint32_t)(a.tokens * a.heads), LATENT / 4, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
