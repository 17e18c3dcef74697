// The search of a page selection, apart from where the keys lie: plain C++, so that a program on
// the host can run it over any counts.
#pragma once

#include <stdint.h>

namespace mono {
namespace prompt {

// A value in (lo, hi], lo < hi, that halves it: rounded up, and no sum of the two passes 32 bits
// (a NaN's key may be the largest number that there is).
constexpr uint32_t upper_middle(uint32_t lo, uint32_t hi) { return hi - (hi - lo) / 2; }
static_assert(upper_middle(0, 0xffffffffu) == 0x80000000u && upper_middle(0xfffffffeu, 0xffffffffu) == 0xffffffffu && upper_middle(0, 1) == 1,
              "above lo, or the search does not end");

// The largest of [lo, hi] that `need` keys or more are at least, where lo is one such and no value above hi
// is: each step takes half of what is left. It ends early at a value that just `need` keys are at least. `kept`:
// how many keys are at least the result, as far as they were counted (0: they were not).
template <class Count>
constexpr uint32_t largest_kept_by(int need, uint32_t lo, uint32_t hi, int& kept, Count count) {
  kept = 0;
#pragma unroll 1
  while (lo < hi && kept != need) {
    const uint32_t mid = upper_middle(lo, hi);
    const int m = count(mid);
    if (m >= need) lo = mid, kept = m;
    else hi = mid - 1;
  }
  return lo;
}

}  // namespace prompt
}  // namespace mono
