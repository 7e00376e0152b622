// Rows of equal width at strides in up to three dimensions: do they lie on one another?  Plain
// C++, for the host checks of the operators that write such rows, their Python binding and the host
// tests.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace ypk {

// Rows of `width` units that start at `at` + sum i_k stride[k], 0 <= i_k < count[k]; all of one unit
// (elements or bytes), strides not negative.
struct StridedRows {
  int64_t at, width;
  int64_t stride[3], count[3];
};

// A dimension of the distance between two rows: any whole number of strides from lo to hi.
struct RowSteps {
  int64_t stride, lo, hi;
};

// Is some distance x + sum d_k stride_k shorter than the width, with `moved` or some d_k not 0?
// The widest steps come first (dims[0 .. n)), so that what the rest can reach leaves few d_k: one or two
// where the dimensions are nested, as those of views are.  `budget` bounds the looks; past it the
// answer is yes.
inline bool some_step_meets(const RowSteps *dims, int n, int64_t x, int64_t width, bool moved, int &budget) {
  if (--budget < 0) return true;
  if (n == 0) return moved && x > -width && x < width;
  int64_t lowest = 0, highest = 0;
  for (int i = 1; i < n; ++i) lowest += dims[i].lo * dims[i].stride, highest += dims[i].hi * dims[i].stride;
  const RowSteps &s = dims[0];
  if (s.stride == 0) return some_step_meets(dims + 1, n - 1, x, width, moved || s.lo < 0 || s.hi > 0, budget);
  // -width < x + d stride + rest < width
  const auto floor_of = [&](int64_t a) { return a >= 0 ? a / s.stride : -((-a + s.stride - 1) / s.stride); };
  const int64_t first = std::max(s.lo, floor_of(-width - x - highest) + 1);
  const int64_t last = std::min(s.hi, -floor_of(-(width - x - lowest)) - 1);
  for (int64_t d = first; d <= last; ++d)
    if (some_step_meets(dims + 1, n - 1, x + d * s.stride, width, moved || d != 0, budget)) return true;
  return false;
}

inline void widest_first(RowSteps *dims, int n) {
  std::sort(dims, dims + n, [](const RowSteps &a, const RowSteps &b) { return a.stride > b.stride; });
}

// No two rows share a unit.
inline bool rows_distinct(const StridedRows &r) {
  RowSteps dims[3];
  int n = 0;
  for (int k = 0; k < 3; ++k)
    if (r.count[k] > 1) dims[n++] = {r.stride[k], -(r.count[k] - 1), r.count[k] - 1};
  // nested dimensions, each step over all that the narrower ones reach; most often as they stand
  const auto nested = [&] {
    int64_t extent = r.width;
    for (int i = n - 1; i >= 0; --i) {
      if (dims[i].stride < extent) return false;
      extent += dims[i].hi * dims[i].stride;
    }
    return true;
  };
  if (nested()) return true;
  widest_first(dims, n);
  int budget = 1 << 16;
  return nested() || !some_step_meets(dims, n, 0, r.width, false, budget);
}

// Some row of a shares a unit with one of b (the same width); also where that is too tangled to tell.
inline bool rows_touch(const StridedRows &a, const StridedRows &b) {
  int64_t end_a = a.at + a.width, end_b = b.at + b.width;
  for (int k = 0; k < 3; ++k) {
    if (a.count[k] < 1 || b.count[k] < 1) return false;
    end_a += (a.count[k] - 1) * a.stride[k];
    end_b += (b.count[k] - 1) * b.stride[k];
  }
  if (a.at >= end_b || b.at >= end_a) return false;
  RowSteps dims[6];
  int n = 0;
  const auto step = [&](int64_t stride, int64_t lo, int64_t hi) {      // equal strides make one dimension
    if (lo == hi) return;
    for (int i = 0; i < n; ++i)
      if (dims[i].stride == stride) {
        dims[i].lo += lo, dims[i].hi += hi;
        return;
      }
    dims[n++] = {stride, lo, hi};
  };
  for (int k = 0; k < 3; ++k) {
    step(a.stride[k], -(a.count[k] - 1), 0);
    step(b.stride[k], 0, b.count[k] - 1);
  }
  widest_first(dims, n);
  int budget = 1 << 12;
  return some_step_meets(dims, n, b.at - a.at, a.width, true, budget);
}

}  // namespace ypk
