// Host-side check of the block operators' outputs against what they read and write beside them: views with strides, as bytes.
// A kernel writes some rows while others are still read, so memory that two of them share gives results that depend on
// timing; such a call is refused.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <cstdint>

namespace sq {

namespace overlap {
using Wide = __int128;  // strides and counts come from a caller
}

// `run` contiguous bytes at every index of up to three axes; at null or a count of zero: nothing.
struct View {
  overlap::Wide begin, last;  // where the first and the last run start
  int64_t run;
  int64_t count[3], stride[3];  // strides in bytes, not negative
  bool empty;

  View(const void* at, int64_t run, int64_t n0 = 1, int64_t s0 = 0, int64_t n1 = 1, int64_t s1 = 0, int64_t n2 = 1, int64_t s2 = 0)
      : begin(reinterpret_cast<uintptr_t>(at)),
        last(begin + overlap::Wide{s0} * (n0 - 1) + overlap::Wide{s1} * (n1 - 1) + overlap::Wide{s2} * (n2 - 1)),
        run(run), count{n0, n1, n2}, stride{s0, s1, s2}, empty(at == nullptr || run <= 0 || n0 <= 0 || n1 <= 0 || n2 <= 0) {}
};

namespace overlap {

struct Term {
  Wide step, most;  // step * (0 .. most)
};

// Whether a sum of one multiple of each term lies in [low, high]; terms by falling step.  For nested strides each level leaves
// one or two multiples to try; a layout that needs more than `budget` steps counts as reached.
inline bool reaches(const Term* term, int n, Wide low, Wide high, int& budget) {
  if (n == 0) return low <= 0 && high >= 0;
  if (--budget < 0) return true;
  Wide rest = 0;
  for (int i = 1; i < n; ++i) rest += term[i].step * term[i].most;
  const Wide need = low - rest;
  const Wide first = need > 0 ? (need + term[0].step - 1) / term[0].step : 0;
  const Wide last = high < 0 ? -1 : std::min(high / term[0].step, term[0].most);
  for (Wide x = first; x <= last; ++x)
    if (reaches(term + 1, n - 1, low - x * term[0].step, high - x * term[0].step, budget)) return true;
  return false;
}

// the same for terms in any order, equal steps as one
inline bool sum_within(Term* term, int n, Wide low, Wide high) {
  std::sort(term, term + n, [](const Term& a, const Term& b) { return a.step > b.step; });
  int kept = 0;
  for (int i = 0; i < n; ++i) {
    if (term[i].step <= 0 || term[i].most <= 0) continue;
    if (kept > 0 && term[kept - 1].step == term[i].step) term[kept - 1].most += term[i].most;
    else term[kept++] = term[i];
  }
  int budget = 4096;
  return reaches(term, kept, low, high, budget);
}

}  // namespace overlap

// Whether two views share a byte.
inline bool overlaps(const View& a, const View& b) {
  using overlap::Wide;
  if (a.empty || b.empty || a.last + a.run <= b.begin || b.last + b.run <= a.begin) return false;
  // a run of a begins at a.begin + A, one of b at b.last - B, A and B sums of the terms: they share a byte where
  // -a.run < (a.begin + A) - (b.last - B) < b.run
  overlap::Term term[6];
  for (int i = 0; i < 3; ++i) {
    term[i] = {a.stride[i], Wide{a.count[i]} - 1};
    term[3 + i] = {b.stride[i], Wide{b.count[i]} - 1};
  }
  const Wide from = a.begin - b.last;
  return overlap::sum_within(term, 6, -Wide{a.run} + 1 - from, Wide{b.run} - 1 - from);
}

// Whether two indices of a view share a byte.
inline bool overlaps_itself(const View& a) {
  using overlap::Wide;
  if (a.empty) return false;
  Wide inside = a.run;  // axes that contain one another in order, as most do: nothing to look for
  bool nested = true;
  for (int i = 2; i >= 0; --i) {
    if (a.count[i] == 1) continue;
    nested = nested && a.stride[i] >= inside;
    inside += Wide{a.stride[i]} * (a.count[i] - 1);
  }
  if (nested) return false;
  for (int lead = 0; lead < 3; ++lead) {  // indices that differ first on axis `lead`, there by one or more
    const Wide most = Wide{a.count[lead]} - 1;
    if (most <= 0) continue;
    overlap::Term term[3];
    int n = 0;
    term[n++] = {a.stride[lead], most - 1};
    Wide from = a.stride[lead];
    for (int i = lead + 1; i < 3; ++i) {
      term[n++] = {a.stride[i], 2 * (Wide{a.count[i]} - 1)};
      from -= Wide{a.stride[i]} * (Wide{a.count[i]} - 1);
    }
    if (overlap::sum_within(term, n, -Wide{a.run} + 1 - from, Wide{a.run} - 1 - from)) return true;
  }
  return false;
}

// The same memory index by index.
inline bool same_view(const View& a, const View& b) {
  if (a.begin != b.begin || a.run != b.run) return false;
  for (int i = 0; i < 3; ++i)
    if (a.count[i] != b.count[i] || (a.count[i] > 1 && a.stride[i] != b.stride[i])) return false;
  return true;
}

// An output that shares memory with itself or with one of `others`.
inline bool clashes(const View& out, std::initializer_list<View> others) {
  if (overlaps_itself(out)) return true;
  for (const View& other : others)
    if (overlaps(out, other)) return true;
  return false;
}

}  // namespace sq
