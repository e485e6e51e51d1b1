// Where a strided array's rows lie, for the checks of what a call writes. Plain C++, no device code.
#pragma once

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <utility>

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

  // Bytes from the first row's start to the last one's end, of some of the axes (bits of `some`).
  __int128 extent(unsigned some) const {
    __int128 e = width;
    for (int i = 0; i < axes; ++i)
      if (some >> i & 1) e += static_cast<__int128>(axis[i].n - 1) * axis[i].step;
    return e;
  }

  // No two rows share a byte: every axis steps over all that the ones before it span. (Layouts whose rows interleave
  // without lying inside one another are refused with the overlapping ones.)
  bool apart() const {
    for (int i = 0; i < axes; ++i)
      if (axis[i].step < extent((1u << i) - 1)) return false;
    return true;
  }

  // No row of some of the axes shares a byte with one of b's, whose first lies `between` bytes behind. Any step S of theirs
  // that tells it will do: without the axes that step by multiples of S, blocks that span no more than S can meet at two
  // distances alone, their own modulo S and S less. (Arrays that no step tells apart count as overlapping.)
  bool apart_from(unsigned some, const Spans& b, unsigned of_b, __int128 between) const {
    if (between >= extent(some) || -between >= b.extent(of_b)) return true;
    auto rest = [](const Spans& s, unsigned m, int64_t step) {
      for (int i = 0; i < s.axes; ++i)
        if (s.axis[i].step % step == 0) m &= ~(1u << i);
      return m;
    };
    for (const auto& [s, m] : {std::pair{this, some}, std::pair{&b, of_b}})
      for (int i = s->axes - 1; i >= 0; --i) {
        const int64_t step = s->axis[i].step;
        if (!(m >> i & 1) || step == 0) continue;
        const unsigned ra = rest(*this, some, step), rb = rest(b, of_b, step);
        if (extent(ra) > step || b.extent(rb) > step) continue;
        const __int128 at0 = (between % step + step) % step;
        if (apart_from(ra, b, rb, at0) && apart_from(ra, b, rb, at0 - step)) return true;
      }
    return false;
  }
  bool apart_from(const Spans& b) const {
    return apart_from((1u << axes) - 1, b, (1u << b.axes) - 1, static_cast<__int128>(b.at) - static_cast<__int128>(at));
  }
};

}  // namespace pdh
