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

  // No row of the first `count` axes shares a byte with one of b's first `bcount`, whose first lies `between` bytes behind.
  // What both step over by the longest step, S, is taken off: rests that span no more than S can meet at two distances
  // alone, their own modulo S and S less. (Arrays that this does not tell apart count as overlapping.)
  bool apart_from(int count, const Spans& b, int bcount, __int128 between) const {
    const __int128 ea = extent(count), eb = b.extent(bcount);
    if (between >= ea || -between >= eb) return true;
    const int64_t sa = count > 0 ? axis[count - 1].step : 0, sb = bcount > 0 ? b.axis[bcount - 1].step : 0;
    const int64_t step = sa > sb ? sa : sb;
    if (step == 0) return false;
    const int ca = sa == step ? count - 1 : count, cb = sb == step ? bcount - 1 : bcount;
    if (extent(ca) > step || b.extent(cb) > step) return false;
    const __int128 rest = (between % step + step) % step;
    return apart_from(ca, b, cb, rest) && apart_from(ca, b, cb, rest - step);
  }
  bool apart_from(const Spans& b) const {
    return apart_from(axes, b, b.axes, static_cast<__int128>(b.at) - static_cast<__int128>(at));
  }
};

}  // namespace pdh
