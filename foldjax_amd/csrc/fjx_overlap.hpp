// Whether two strided sets of rows share memory. Host only, standard headers only.
//
// Two views of one buffer, such as the queries and the keys of a projection that writes
// both, lie within each other's first and last byte without a byte in common: ranges of
// addresses alone would refuse them.
#pragma once

#include <algorithm>
#include <cstdint>

namespace fjx {

// rows of `width` bytes at `at`, n[i] of them at steps of stride[i] >= 0 bytes along axis i
struct RowSet {
  static constexpr int kAxes = 3;
  uintptr_t at;
  int64_t n[kAxes], stride[kAxes];
  int64_t width;
};

namespace overlap {

typedef __int128 wide;
// any multiple of `step` with a factor in [lo, hi]
struct Term {
  wide step, lo, hi;
};
inline wide floor_div(wide a, wide b) { return a / b - (a % b < 0); }  // b > 0

// Whether one multiple of each term adds up to `want`, the largest steps first: what the
// others can reach leaves few factors for the largest. `budget`: sums looked at; where they
// are used up the answer is true.
inline bool reaches(const Term* t, int n, wide want, int& budget) {
  if (n == 0) return want == 0;
  if (--budget < 0) return true;
  wide lo = 0, hi = 0;
  for (int i = 1; i < n; ++i) {
    lo += t[i].lo * t[i].step;
    hi += t[i].hi * t[i].step;
  }
  const wide first = std::max(t[0].lo, -floor_div(hi - want, t[0].step)), last = std::min(t[0].hi, floor_div(want - lo, t[0].step));
  for (wide x = first; x <= last; ++x)
    if (reaches(t + 1, n - 1, want - x * t[0].step, budget)) return true;
  return false;
}

}  // namespace overlap

// the same rows at the same places
inline bool rows_equal(const RowSet& a, const RowSet& b) {
  bool same = a.at == b.at && a.width == b.width;
  for (int i = 0; i < RowSet::kAxes; ++i) same = same && a.n[i] == b.n[i] && (a.n[i] <= 1 || a.stride[i] == b.stride[i]);
  return same;
}

// Whether a byte belongs to both: exact for views with steps alike and for most others, and
// true where finding out would take long.
inline bool rows_meet(const RowSet& a, const RowSet& b) {
  using namespace overlap;
  wide a_end = a.width, b_end = b.width;
  for (int i = 0; i < RowSet::kAxes; ++i) {
    if (a.n[i] < 1 || b.n[i] < 1) return false;
    a_end += (wide)(a.n[i] - 1) * a.stride[i];
    b_end += (wide)(b.n[i] - 1) * b.stride[i];
  }
  const wide between = (wide)b.at - (wide)a.at;  // a's place less b's, counted from their starts, must be this
  if (between >= a_end || -between >= b_end) return false;
  // a byte of a is sum x_i stride_i + x, one of b sum y_i stride_i + y: x_i step up, y_i down
  Term t[2 * RowSet::kAxes + 1];
  int n = 0;
  auto add = [&](wide step, wide down, wide up) {
    if (step == 0 || (down == 0 && up == 0)) return;
    for (int i = 0; i < n; ++i)
      if (t[i].step == step) {
        t[i].lo -= down;
        t[i].hi += up;
        return;
      }
    t[n++] = {step, -down, up};
  };
  for (int i = 0; i < RowSet::kAxes; ++i) {
    add(a.stride[i], 0, a.n[i] - 1);
    add(b.stride[i], b.n[i] - 1, 0);
  }
  add(1, b.width - 1, a.width - 1);
  std::sort(t, t + n, [](const Term& x, const Term& y) { return x.step > y.step; });
  int budget = 4096;
  return reaches(t, n, between, budget);
}

}  // namespace fjx
