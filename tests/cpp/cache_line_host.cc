// csrc/cache_line.h on the host: what every workgroup of a launch takes (tests/test_cache_line.py).
#include <vector>

#include "../../ctranslate2_amd/csrc/cache_line.h"

using namespace ct2x;

// A workgroup that has unit `unit` of `units` for itself, n rounds: its parts, as unit, r0, r1.
extern "C" int line_whole(uint32_t unit, uint32_t units, uint32_t n, uint32_t* out, int room) {
  Stretch s = Stretch::whole(unit, n);
  int parts = 0;
  while (s.x < s.x1 && parts < room) {
    const Stretch::Part p = s.part(n);
    out[3 * parts] = p.unit;
    out[3 * parts + 1] = p.r0;
    out[3 * parts++ + 2] = p.r1;
    s.pass(p, n, units);
  }
  return parts;
}

// A line over `entries` of `units` units with rounds[e] rounds each, cut for `groups` workgroups: 0 if every
// round is taken once, in order, each workgroup's share differs by one at most and holder() names who took it.
extern "C" int line_check(int entries, uint32_t units, const uint32_t* rounds, uint32_t groups) {
  Line line{0, groups, 0, 0};
  for (int e = 0; e < entries; ++e) line.total += rounds[e] * units;
  line.each = line.total / groups;
  line.longer = line.total - line.each * groups;
  uint32_t next = 0, unit = 0, r = 0;
  int entry = 0;
  for (uint32_t w = 0; w < groups; ++w) {
    Stretch s{line.start(w), line.start(w + 1), 0, 0};
    if (s.x != next || s.x1 - s.x < line.each || s.x1 - s.x > line.each + 1) return 1;
    int b = 0;
    while (b < entries && s.before + rounds[b] * units <= s.x) s.before += rounds[b++] * units;
    while (s.x < s.x1) {
      const uint32_t n = rounds[b];
      const Stretch::Part p = s.part(n);
      if (b != entry || p.unit != unit || p.r0 != r || p.r1 <= p.r0 || p.r1 > n) return 2;
      for (uint32_t x = s.x; x < s.x + (p.r1 - p.r0); ++x)
        if (line.holder(x) != w) return 3;
      next += p.r1 - p.r0;
      r = p.r1 == n ? 0 : p.r1;
      if (p.r1 == n && ++unit == units) {
        unit = 0;
        ++entry;
      }
      if (s.pass(p, n, units)) ++b;
      if (b != entry) return 4;
    }
  }
  return next == line.total && entry == entries ? 0 : 5;
}

extern "C" int line_too_long(int64_t units, int64_t rounds) { return line_is_too_long(units, rounds); }
