// The cheap score of a page: the largest index score of its keys that a token sees.
//
//   out[t, p] = max over keys j of page p at positions <= pos[t] of
//               sum_h iw[t, h] max(0, q[t, h] . k[j])        (64 heads of 128 FP4 dims)
//
// A wave takes four tokens and a run of pages. The tokens' queries stay in registers as the
// FP4 MFMA wants them (16 registers each), a page's keys come once for all four, the next
// page's ahead. An MFMA's 16 heads x 16 keys take two vector operations a value (the ReLU and
// the weighted sum), twice the MFMA's own time: they bound the kernel.
#include <algorithm>

#include "prompt_common.h"

namespace mono {
namespace prompt {
namespace {

constexpr int WAVES = 4, NT = 4, HT = INDEX_HEADS / 16, KT = PAGE / 16;
constexpr float NEG_INF = -__builtin_inff();

struct Query {
  u32x4 q[HT];
  uint32_t scale;    // byte ht: the lane's row's scale of head tile ht
  uint32_t w[HT][2]; // weights of heads 16 ht + 4 g .. + 3
};
struct Keys {
  u32x4 k[KT];
  uint32_t scale;    // byte kt: the lane's key's scale of key tile kt
};

MONO_DEV i32x8 fp4_operand(const u32x4& v) { return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}; }

// (the scales' bytes are picked by constants of the instruction)
template <int H, int K>
MONO_DEV f32x4 dots(const Query& q, const Keys& k) {
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_operand(q.q[H]), fp4_operand(k.k[K]), z, 4, 4, H, (int)q.scale, K,
                                                          (int)k.scale);
}
template <int K>
MONO_DEV void dots(const Query& q, const Keys& k, f32x4 (&d)[HT]) {
  static_assert(HT == 4, "64 heads");
  d[0] = dots<0, K>(q, k), d[1] = dots<1, K>(q, k), d[2] = dots<2, K>(q, k), d[3] = dots<3, K>(q, k);
}

// the larger, or a NaN where either is one
MONO_DEV float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

MONO_DEV float weighted(const Query& q, const f32x4 (&d)[HT]) {
  float s = 0.f;
#pragma unroll
  for (int h = 0; h < HT; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = i & 1 ? bf16_hi(q.w[h][i / 2]) : bf16_lo(q.w[h][i / 2]);
      s = fmaf(w, nan_max(d[h][i], 0.f), s);
    }
  return s;
}

// 16: rows (a0 + a1, b0 + b1, a2 + a3, b2 + b3) of 16 lanes; 32: halves (a lo + a hi, b lo + b hi)
template <int LANES>
MONO_DEV float swap_sum(float a, float b) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  const auto v = LANES == 16 ? __builtin_amdgcn_permlane16_swap(x, y, false, false) : __builtin_amdgcn_permlane32_swap(x, y, false, false);
  return __uint_as_float(v[0]) + __uint_as_float(v[1]);
}

struct OpNanMax {
  MONO_DEV float operator()(float a, float b) const { return nan_max(a, b); }
};

// The page's score for one token, whose first `seen` keys (lane = key) count.
MONO_DEV float page_score(const Query& q, const Keys& k, int seen, int lane) {
  f32x4 d[2][HT];  // a key tile's MFMAs go out before the sums of the one before
  float s[KT];
  dots<0>(q, k, d[0]);
  dots<1>(q, k, d[1]);
  s[0] = weighted(q, d[0]);
  dots<2>(q, k, d[0]);
  s[1] = weighted(q, d[1]);
  dots<3>(q, k, d[1]);
  s[2] = weighted(q, d[0]);
  s[3] = weighted(q, d[1]);
  // each key's sum over the four lane groups; tile j's ends in lane group j, so lane = key
  const float key = swap_sum<32>(swap_sum<16>(s[0], s[1]), swap_sum<16>(s[2], s[3]));
  return wave_reduce(lane < seen ? key : NEG_INF, OpNanMax());
}

__global__ __launch_bounds__(WAVES * WAVE, 2) void k_scores(mono_prompt_scores_args a, int run, int runs, int64_t tasks) {
  const int lane = threadIdx.x % WAVE, g = lane / 16, r = lane % 16;
  const int64_t task = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  if (task >= tasks) return;
  const int64_t t0 = task / runs * NT;
  const int p0 = (int)(task % runs) * run, p1 = min(p0 + run, a.columns);
  Query q[NT];
  int req[NT], seen[NT];  // the token's request and how many keys from page p0 on it sees
  float best[NT];         // lane l: the score of page p0 + l
  uint32_t left = 0;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t t = min(t0 + j, a.tokens - 1);
    const int pos = min(a.pos[t], (p1 << 6) - 1);
    req[j] = a.req[t];
    seen[j] = t0 + j < a.tokens && pos >= 0 && req[j] >= 0 && req[j] < a.requests ? pos + 1 - (p0 << 6) : 0;
    if (seen[j] > 0) left |= 1u << j;
    best[j] = NEG_INF;
  }
  left = __builtin_amdgcn_readfirstlane(left);
  if (left) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t t = min(t0 + j, a.tokens - 1);
      q[j].scale = 0;
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        const int64_t row = t * INDEX_HEADS + 16 * h + r;
        q[j].q[h] = ld_u32x4(static_cast<const uint8_t*>(a.iq) + row * (INDEX / 2) + 16 * g);
        q[j].scale |= (uint32_t)static_cast<const uint8_t*>(a.iqs)[row * (INDEX / 32) + g] << 8 * h;
        const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.iw) + t * INDEX_HEADS + 16 * h + 4 * g);
        q[j].w[h][0] = w[0], q[j].w[h][1] = w[1];
      }
    }
  }
  while (left) {  // the tokens of one request at a time (mostly all of them)
    const int first = __builtin_ctz(left);
    int rq = 0, most = 0;
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) rq = j == first ? req[j] : rq;
    rq = __builtin_amdgcn_readfirstlane(rq);
#pragma unroll
    for (int j = 0; j < NT; ++j)
      if ((left >> j & 1) && req[j] == rq) {
        mine |= 1u << j;
        most = max(most, seen[j]);
      }
    mine = __builtin_amdgcn_readfirstlane(mine);
    left &= ~mine;
    // the run's pages, lane l page p0 + l; those that hold a key that is seen, one after another
    const int n = (__builtin_amdgcn_readfirstlane(most) + PAGE - 1) / PAGE;  // (at most `run`: seen ends with the run)
    const int at = p0 + min(lane, n - 1);
    const int id = at < a.pt_stride ? a.page_table[(int64_t)rq * a.pt_stride + at] : -1;
    uint64_t live = __ballot(lane < n && id >= 0 && id < a.n_pages);
    const auto load = [&](int p, Keys& k) {
      const int64_t page = __builtin_amdgcn_readlane(id, p);
      const uint8_t* ikv = static_cast<const uint8_t*>(a.ikv) + page * (PAGE * INDEX / 2) + g * (PAGE * 16) + r * 16;
#pragma unroll
      for (int i = 0; i < KT; ++i) k.k[i] = ld_u32x4(ikv + 256 * i);
      k.scale = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.iks) + page * (PAGE * INDEX / 32) + g * PAGE + r * 4);
    };
    Keys k, next;
    if (live) load(__builtin_ctzll(live), next);
    while (live) {
      const int p = __builtin_ctzll(live);
      live &= live - 1;
      k = next;
      load(live ? __builtin_ctzll(live) : p, next);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int here = __builtin_amdgcn_readfirstlane(seen[j]) - (p << 6);
        if ((mine >> j & 1) && here > 0) {
          const float s = page_score(q[j], k, here, lane);
          best[j] = lane == p ? s : best[j];
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
    if (t0 + j < a.tokens && p0 + lane < p1) a.out[(t0 + j) * a.columns + p0 + lane] = best[j];
}

}  // namespace

hipError_t page_scores(const mono_prompt_scores_args& a, hipStream_t st) {
  const int64_t groups = (a.tokens + NT - 1) / NT;
  // pages a wave: as many as leave 8192 waves, two rounds of them (a run's queries are loaded once)
  const int run = (int)std::min<int64_t>(std::max<int64_t>(groups * a.columns / 8192, 1), 16);
  const int runs = (a.columns + run - 1) / run;
  const int64_t tasks = groups * runs;
  k_scores<<<(uint32_t)((tasks + WAVES - 1) / WAVES), WAVES * WAVE, 0, st>>>(a, run, runs, tasks);
  return hipGetLastError();
}

}  // namespace prompt
}  // namespace mono
