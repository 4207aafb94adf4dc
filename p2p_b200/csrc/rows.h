// rows.h -- whether two sets of strided rows share a byte (host code).
#pragma once

#include <cstdint>

namespace p2p {

// n rows each (n > 0): row i of a is the bytes [a + i * pitch_a, + width_a), likewise b; the rows of
// one set do not overlap (width <= pitch, or n is 1).
inline bool rows_overlap(const void* a, int64_t pitch_a, int64_t width_a, const void* b,
                         int64_t pitch_b, int64_t width_b, int64_t n) {
  const int64_t at_a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a));
  const int64_t at_b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b));
  if (at_a + (n - 1) * pitch_a + width_a <= at_b || at_b + (n - 1) * pitch_b + width_b <= at_a)
    return false;
  if (n == 1) return true;
  if (pitch_a == pitch_b && pitch_a > 0) {  // widths within the pitch: only the nearest rows can meet
    const int64_t d = at_b - at_a, near = -d / pitch_a;
    for (int64_t k = near - 1; k <= near + 1; ++k) {  // row i of a against row i + k of b
      const int64_t gap = d + k * pitch_a;
      if (k > -n && k < n && gap < width_a && gap + width_b > 0) return true;
    }
    return false;
  }
  // Rows in order on both sides, whichever ends first goes on to its next.
  for (int64_t i = 0, j = 0; i < n && j < n;) {
    const int64_t x = at_a + i * pitch_a, y = at_b + j * pitch_b;
    if (x + width_a <= y) ++i;
    else if (y + width_b <= x) ++j;
    else return true;
  }
  return false;
}

}  // namespace p2p
