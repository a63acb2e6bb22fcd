// How a launch of the attention over a serving cache cuts its work (attention_cache.hip): the units of an entry
// (head of the cache, row group) have as many rounds each as the entry's positions take, and workgroups
// take stretches of rounds. Nothing of HIP in here, so that the arithmetic is tested on the host.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define CT2X_LINE_FN __host__ __device__ __forceinline__
#else
#define CT2X_LINE_FN inline
#endif

namespace ct2x {

// The line of all rounds and how many workgroups share it: the first `longer` take `each` + 1 rounds.
// (A line has less than 2^31 rounds: longer ones are not made, line_is_too_long.)
struct Line {
  uint32_t total, groups, each, longer;
  CT2X_LINE_FN uint32_t start(uint32_t w) const { return w * each + (w < longer ? w : longer); }
  // the workgroup that holds round x
  CT2X_LINE_FN uint32_t holder(uint32_t x) const {
    const uint32_t ahead = longer * (each + 1);
    return x < ahead ? x / (each + 1) : longer + (x - ahead) / each;
  }
};

// units of at most `rounds` rounds each
CT2X_LINE_FN bool line_is_too_long(int64_t units, int64_t rounds) { return units * rounds >= int64_t{1} << 31; }

// A workgroup's rounds x .. x1 - 1, taken unit by unit. `before`: the round of the line that the present
// entry's unit `first` begins at. A workgroup that has one unit for itself counts from that unit's first round:
// with many row groups and positions an entry's rounds do not fit 32 bits.
struct Stretch {
  uint32_t x, x1, before, first;
  struct Part {
    uint32_t unit, r0, r1;  // of the entry; its rounds r0 .. r1 - 1
  };
  static CT2X_LINE_FN Stretch whole(uint32_t unit, uint32_t rounds) { return Stretch{0, rounds, 0, unit}; }
  // n: rounds of each of the entry's units
  CT2X_LINE_FN Part part(uint32_t n) const {
    const uint32_t unit = (x - before) / n, r0 = x - before - unit * n;
    return Part{first + unit, r0, x1 - x < n - r0 ? r0 + (x1 - x) : n};
  }
  // behind that part; true: the next one is the next entry's
  CT2X_LINE_FN bool pass(const Part& p, uint32_t n, uint32_t units) {
    x += p.r1 - p.r0;
    const bool ends = p.r1 == n && p.unit + 1 == units;
    if (ends) before = x;
    return ends;
  }
};

}  // namespace ct2x
