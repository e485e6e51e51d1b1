// Where a strided array's rows lie, for the checks of what a call writes. Plain C++, no device code.
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>

namespace pdh {

// Rows of `width` bytes, one at every combination of the axes' steps.
struct Spans {
  struct Axis {
    int64_t n, step;  // bytes, >= 0
  };
  uintptr_t at;  // the first row
  int64_t width;
  Axis axis[4];  // ascending by step, those of one entry left out
  int axes = 0;

  Spans(const void* first, int64_t row, std::initializer_list<Axis> of) : at(reinterpret_cast<uintptr_t>(first)), width(row) {
    for (const Axis& a : of)
      if (a.n > 1) axis[axes++] = a;
    std::sort(axis, axis + axes, [](const Axis& a, const Axis& b) { return a.step < b.step; });
  }

  // Bytes from the first row's start to the last one's end, of the first `count` axes.
  __int128 extent(int count) const {
    __int128 e = width;
    for (int i = 0; i < count; ++i) e += static_cast<__int128>(axis[i].n - 1) * axis[i].step;
    return e;
  }

  // No two rows share a byte: every axis steps over all that the ones before it span. (Layouts whose rows interleave
  // without lying inside one another are refused with the overlapping ones.)
  bool apart() const {
    for (int i = 0; i < axes; ++i)
      if (axis[i].step < extent(i)) return false;
    return true;
  }
};

}  // namespace pdh
