// The cheap score of a page: the largest index score of its keys that a token sees.
//
//   out[t, p] = max over keys j of page p at positions <= pos[t] of
//               sum_h iw[t, h] max(0, q[t, h] . k[j])        (64 heads of 128 FP4 dims)
//
// A wave takes a token and a run of pages. The token's query stays in registers as the FP4 MFMA
// wants it, with half its heads' weights, the next page's keys come ahead. A 32 x 32 MFMA's lanes
// hold one key each and 16 heads: the ReLU and the weighted sum are two FMAs a value, and a key's
// heads meet in one swap of halves. They bound the kernel: some 180 vector operations a token and
// page, issuing 97 % of the time, beside 256 cycles of MFMA. 8192 tokens from position 0: 205 to 213 us by the
// card, 2.6 to 2.7 PFLOP/s (a maximum and an FMA a value: 290 us; the products alone would take some 65).
//
// FP4 products and their sum are exact in f32 where a query's and a key's scales lie close; the weighted sum is
// f32 throughout. As x / 2 + |x| / 2 a head's ReLU leaves a rounding of the size of a product that it
// cuts off, 2^-24 of it. A page with a score that is not finite is formed again with the ReLU as a
// maximum: one half may leave f32's range where their sum does not (the test for it: 2 us of 208).
#include <algorithm>

#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int WAVES = 4, HT = INDEX_HEADS / 32, KT = PAGE / 32;
constexpr float NEG_INF = -__builtin_inff();
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Lane l: row (head, key) l % 32 of a tile; of the 128 dims two MFMAs of 64, of those half l / 32.
struct Query {
  u32x4 q[HT][2];
  uint32_t scale;         // byte 2 h + k: the row's scale of head tile h, dims 64 k + 32 (l / 32) ..
  float halves[HT][16];   // half the weights of heads 32 h + 8 (i / 4) + 4 (l / 32) + i % 4
};
struct Keys {
  u32x4 k[KT][2];
  uint32_t scale[2];      // byte 2 t: the scale of key tile t
};

MONO_DEV i32x8 fp4_operand(const u32x4& v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// head tile H against key tile K (the scales' bytes are picked by constants of the instruction)
template <int H, int K>
MONO_DEV f32x16 dots(const Query& q, const Keys& k) {
  f32x16 d = {};
  d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(q.q[H][0]), fp4_operand(k.k[K][0]), d, 4, 4, 2 * H, (int)q.scale,
                                                      2 * K, (int)k.scale[0]);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(q.q[H][1]), fp4_operand(k.k[K][1]), d, 4, 4, 2 * H + 1,
                                                         (int)q.scale, 2 * K, (int)k.scale[1]);
}

// the larger, or a NaN where either is one
struct OpNanMax {
  MONO_DEV float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); }
};

// sum_h w_h max(0, x_h) of a lane's 16 heads as sum_h w_h / 2 (x_h + |x_h|): an FMA takes |x| as it
// is, and a NaN stays one.
MONO_DEV float weighted(const float (&halves)[16], const f32x16& d) {
  float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i % 2] = fmaf(halves[i], d[i], s[i % 2]);
    t[i % 2] = fmaf(halves[i], fabsf(d[i]), t[i % 2]);
  }
  return (s[0] + s[1]) + (t[0] + t[1]);
}

// halves (a lo . a hi, b lo . b hi)
template <class Op>
MONO_DEV float swap_halves(float a, float b, Op op) {
  const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return op(__uint_as_float(v[0]), __uint_as_float(v[1]));
}

// The scores of the page's keys (lane = key) for one token.
MONO_DEV float key_scores(const Query& q, const Keys& k) {
  f32x16 d[2];  // a tile's MFMAs go out before the sums of the one before
  float s[KT];
  d[0] = dots<0, 0>(q, k);
  d[1] = dots<1, 0>(q, k);
  s[0] = weighted(q.halves[0], d[0]);
  d[0] = dots<0, 1>(q, k);
  s[0] += weighted(q.halves[1], d[1]);
  d[1] = dots<1, 1>(q, k);
  s[1] = weighted(q.halves[0], d[0]);
  s[1] += weighted(q.halves[1], d[1]);
  return swap_halves(s[0], s[1], OpAdd());
}

// The same with the ReLU formed before the weight, a maximum and an FMA a value: where a sum of the two
// halves left f32's range, or met an infinity of either sign in it, this one need not (and a NaN
// that is left is one of the definition's). The weights are twice their halves, exactly.
MONO_DEV float cut_off(const float (&halves)[16], const f32x16& d) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = fmaf(2.0f * halves[i], __builtin_elementwise_maximum(d[i], 0.f), s);
  return s;
}
MONO_DEV float key_scores_cut_off(const Query& q, const Keys& k) {
  float s[KT];
  s[0] = cut_off(q.halves[0], dots<0, 0>(q, k));
  s[0] += cut_off(q.halves[1], dots<1, 0>(q, k));
  s[1] = cut_off(q.halves[0], dots<0, 1>(q, k));
  s[1] += cut_off(q.halves[1], dots<1, 1>(q, k));
  return swap_halves(s[0], s[1], OpAdd());
}

__global__ __launch_bounds__(WAVES * WAVE, 4) void k_scores(mono_prompt_scores_args a, int run) {
  const int lane = threadIdx.x % WAVE, half = lane / 32, r = lane % 32;
  // the workgroup's waves take neighbouring tokens over the same pages, which the CU's cache then holds
  // (and the runs of pages lie far apart in the grid: late pages are seen by late tokens only, and
  // workgroups a few apart share an XCD)
  const int64_t t = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  if (t >= a.tokens) return;
  const int p0 = (int)blockIdx.y * run, p1 = min(p0 + run, a.columns);
  const int pos = min(a.pos[t], PAGE * p1 - 1), req = a.req[t];
  // how many keys from page p0 on the token sees, and in how many pages
  const int seen = pos >= 0 && req >= 0 && req < a.requests ? max(pos + 1 - PAGE * p0, 0) : 0, n = (seen + PAGE - 1) / PAGE;
  float best = NEG_INF;  // lane l: the score of page p0 + l
  const int at = p0 + min(lane, max(n - 1, 0));
  const int id = n > 0 && at < a.pt_stride ? a.page_table[(int64_t)req * a.pt_stride + at] : -1;
  uint64_t live = __ballot(lane < n && id >= 0 && id < a.n_pages);
  if (live) {
    const auto load = [&](int p, Keys& k) {
      const int64_t page = __builtin_amdgcn_readlane(id, p);
      const uint8_t* ikv = static_cast<const uint8_t*>(a.ikv) + page * (PAGE * INDEX / 2) + half * (PAGE * 16) + r * 16;
      const uint8_t* iks = static_cast<const uint8_t*>(a.iks) + page * (PAGE * INDEX / 32) + half * PAGE + r % 16 * 4;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < KT; ++i) k.k[i][c] = ld_u32x4(ikv + 2 * c * (PAGE * 16) + 512 * i);
        k.scale[c] = *reinterpret_cast<const uint32_t*>(iks + 2 * c * PAGE) >> (8 * (r / 16));  // byte t / 16 is key t's
      }
    };
    Keys k, next;
    load(__builtin_ctzll(live), next);
    Query q;
    q.scale = 0;
#pragma unroll
    for (int h = 0; h < HT; ++h) {
      const int64_t row = t * INDEX_HEADS + 32 * h + r;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        q.q[h][c] = ld_u32x4(static_cast<const uint8_t*>(a.iq) + row * (INDEX / 2) + 16 * (2 * c + half));
        q.scale |= (uint32_t)static_cast<const uint8_t*>(a.iqs)[row * (INDEX / 32) + 2 * c + half] << 8 * (2 * h + c);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.iw) + t * INDEX_HEADS + 32 * h + 8 * i + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) q.halves[h][4 * i + e] = 0.5f * (e & 1 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]));
      }
    }
    uint64_t again = 0;  // pages with a score that is not finite
    while (live) {
      const int p = __builtin_ctzll(live);
      live &= live - 1;
      k = next;
      load(live ? __builtin_ctzll(live) : p, next);
      const float key = key_scores(q, k);
      const bool mine = lane < seen - PAGE * p;
      if (__any(mine && !__builtin_isfinite(key))) again |= 1ull << p;
      const float top = wave_reduce(mine ? key : NEG_INF, OpNanMax());
      best = lane == p ? top : best;
    }
    while (again) {  // (by itself, so that the loop above holds no more registers: it has none to spare)
      const int p = __builtin_ctzll(again);
      again &= again - 1;
      load(p, k);
      const float key = key_scores_cut_off(q, k);
      const float top = wave_reduce(lane < seen - PAGE * p ? key : NEG_INF, OpNanMax());
      best = lane == p ? top : best;
    }
  }
  if (p0 + lane < p1) a.out[t * a.columns + p0 + lane] = best;
}

}  // namespace

hipError_t page_scores(const mono_prompt_scores_args& a, hipStream_t st) {
  const int64_t groups = (a.tokens + WAVES - 1) / WAVES;
  // pages a workgroup: as many as leave 2048 workgroups, two rounds of them (a run's query is loaded
  // once; 64 tokens of 30000 keys: 2048 workgroups 16.8 us, 4096 24.5, 512 19.7), but 32 at most
  // (8192 tokens: 16 pages a run 235 us, 32 230)
  const int run = (int)std::min<int64_t>(std::max<int64_t>(groups * a.columns / 2048, 1), 32);
  const int64_t runs = (a.columns + run - 1) / run;
  k_scores<<<dim3((uint32_t)groups, (uint32_t)runs), WAVES * WAVE, 0, st>>>(a, run);  // (one dim holds 2^32 threads)
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
