// Which pages a token reads: the first and the last few that it sees, and of the others the
// best-scored, exactly, a tie's lowest page first.
//
// A row's scores as whole numbers in the same order; the k-th largest is found by halving the range
// between two bounds of it, and what is at or above it goes out in ascending order of pages. A row
// lies in registers: of one wave, up to 1024 columns, of a workgroup above.
//
// 8192 rows of 512 columns: 11.4 us, 9 rows 4.3 us. Of the former reading and ordering the scores takes
// 4.4, the search 4.8 and writing 2.5 (each timed with what follows left out). A row takes 485 scalar and
// 370 vector instructions: a step of the search is a compare, a ballot's count and a scalar sum for each
// 64 scores, some ten steps (bit by bit from the top eighteen). A CU has 32 rows and issues a scalar
// instruction a cycle, 6.5 us of them. More than 2048 columns take 32 scores a lane, whose masks do not fit
// the scalar registers (383 of them spill): 8192 rows of 2048 columns 44 us, of 4096 159; 4096 rows of 8192
// columns 89.
#include "prompt_common.h"
#include "prompt_search.h"

namespace mono {
namespace prompt {
namespace {

// larger key = larger value; +0 above -0, a NaN by its bits
MONO_DEV uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// What the waves of a row have each, in every one of them. (Two places in turn: one barrier a time.)
template <int W>
struct RowWaves {
  int (*lds)[W];
  int wave, turn;
  template <class Op>
  MONO_DEV uint32_t all(uint32_t v, Op op) {
    if (W == 1) return v;
    int* at = lds[turn];
    turn ^= 1;
    if (threadIdx.x % WAVE == 0) at[wave] = (int)v;
    __syncthreads();
    v = (uint32_t)at[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v = op(v, (uint32_t)at[w]);
    return __builtin_amdgcn_readfirstlane((int)v);
  }
  MONO_DEV int sum(int v) {
    return (int)all((uint32_t)v, [](uint32_t a, uint32_t b) { return a + b; });
  }
  MONO_DEV uint32_t most(uint32_t v) {
    return all(v, [](uint32_t a, uint32_t b) { return max(a, b); });
  }
  // the sum over the waves before this one
  MONO_DEV int before(int v) {
    if (W == 1) return 0;
    int* at = lds[turn];
    turn ^= 1;
    if (threadIdx.x % WAVE == 0) at[wave] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < wave; ++w) v += at[w];
    return v;
  }
};

// W waves a row, N values a lane: value i of lane l of wave w is column (w N + i) 64 + l.
template <int W, int N>
__global__ __launch_bounds__(256) void k_select(mono_prompt_select_args a) {
  __shared__ int lds[2][W];
  const int lane = threadIdx.x % WAVE, wv = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), w = wv % W;
  RowWaves<W> row_waves{lds, w, 0};
  const int64_t t = (int64_t)blockIdx.x * (4 / W) + wv / W;
  if (t >= a.tokens) return;  // (W > 1: of the whole workgroup)
  const int pos = __builtin_amdgcn_readfirstlane(a.pos[t]);
  const int n = pos < 0 ? 0 : min(pos / PAGE + 1, a.columns);  // pages that the token sees
  const int mine = pos < 0 ? -1 : min(pos / PAGE, a.columns - 1);
  const float* row = a.scores + t * a.stride;
  int32_t* out = a.pages + t * a.picks;
  uint32_t key[N];
  uint32_t always = 0;  // bit i: value i is taken whatever its score
  int forced = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (w * N + i) * WAVE + lane;
    const uint32_t k = order_key(row[min(c, a.columns - 1)]);
    const bool f = c < n && (c < a.first || c > mine - a.last);
    always |= f ? 1u << (i % 32) : 0u;
    static_assert(N <= 32, "a bit each");
    forced += __popcll(__ballot(f));
    key[i] = c < n && !f ? k : 0u;  // (only what is open is above 0)
  }
  const auto open = [&](int i) { return (w * N + i) * WAVE + lane < n && !(always >> i & 1); };
  forced = row_waves.sum(forced);
  // picks left for the scores; an open key above `top` is taken, and of those equal to it the
  // first `border`
  const int need = a.picks - forced, rest = n - forced;
  uint32_t top = 0;
  int border = need > 0 ? INT32_MAX : 0;
  if (need == 0) top = 0xffffffffu;
  if (need > 0 && need < rest) {
    const auto count = [&](auto at_least) {
      int m = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) m += __popcll(__ballot(at_least(key[i])));
      return row_waves.sum(m);
    };
    // Bounds of the k-th largest: the largest key above; below, as many keys as there are lanes
    // with one, each lane's largest, are at least the smallest of those.
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) most = max(most, key[i]);
    const uint32_t hi = row_waves.most(wave_umax(most));
    top = row_waves.most(need <= WAVE ? ~wave_umax(~most) : 0u);
    int kept;
    top = largest_kept_by(need, top, hi, kept, [&](uint32_t mid) { return count([&](uint32_t k) { return k >= mid; }); });
    if (kept != need) border = need - count([&](uint32_t k) { return k > top; });
  }
  int ties_before = 0, taken_before = 0;
  if (W > 1) {  // what the waves before this one take
    int eq = 0, gt = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      eq += __popcll(__ballot(open(i) && key[i] == top));
      gt += __popcll(__ballot((always >> i & 1) || (key[i] > top)));
    }
    ties_before = row_waves.before(eq);
    taken_before = row_waves.before(gt);
    taken_before += min(ties_before, border);
  }
  int at = taken_before, ties = ties_before;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool eq = open(i) && key[i] == top;
    const uint64_t eqs = __ballot(eq);
    const bool tie = eq && ties + (int)__popcll(eqs & ((1ull << lane) - 1)) < border;
    const bool take = (always >> i & 1) || (key[i] > top) || tie;
    const uint64_t taken = __ballot(take);
    const int place = at + (int)__popcll(taken & ((1ull << lane) - 1));
    if (take) out[place] = (w * N + i) * WAVE + lane;
    at += __popcll(taken);
    ties += __popcll(eqs);
  }
  if (w == W - 1)
    for (int i = at + lane; i < a.picks; i += WAVE) out[i] = -1;
}

}  // namespace

hipError_t select_pages(const mono_prompt_select_args& a, hipStream_t st) {
  const auto launch = [&](auto kernel, int rows) {
    kernel<<<(uint32_t)((a.tokens + rows - 1) / rows), 256, 0, st>>>(a);
    return hipGetLastError();
  };
  // a wave a row and a workgroup a row: 8192 rows of 512 columns 11.5 and 24.8 us, 9 rows 4.5 and 5.9; of
  // 1000 columns 21 and 40, 9 rows 7.0 and 6.4; of 2048 columns 37 and 41, 9 rows 13.3 and 6.0
  if (a.columns <= 128) return launch(k_select<1, 2>, 4);
  if (a.columns <= 256) return launch(k_select<1, 4>, 4);
  if (a.columns <= 512) return launch(k_select<1, 8>, 4);
  if (a.columns <= 1024) return launch(k_select<1, 16>, 4);
  if (a.columns <= 2048) return launch(k_select<4, 8>, 1);
  return launch(k_select<4, 32>, 1);  // 8192 columns: MAX_COLUMNS
}

}  // namespace prompt
}  // namespace mono
