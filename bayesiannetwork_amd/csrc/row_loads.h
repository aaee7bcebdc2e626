// 16 bytes of a row that has n elements and no memory behind them: where a pack's load starts, and how its
// elements get to their places.  Plain arithmetic, for host and device.
#pragma once

#include <algorithm>
#include <cstdint>

namespace bn_rows {

// The 16 bytes as four registers.
struct Raw {
  uint32_t w[4];
};

// The element at which a load of `pack` elements begins that is meant for those from `from` on: there if the row has
// them all, else so that it ends with the row.  Needs n >= pack; a pack wholly behind the row's end loads its last one.
constexpr int pack_start(int from, int n, int pack) { return std::min(from, n - pack); }

// The pack with every element `count` places further down (what comes in at the top is of no meaning; beyond the
// pack's own elements, `count` may be anything).
template <int ELEMENT_BYTES>
constexpr Raw moved_down(Raw r, int count) {
  static_assert(ELEMENT_BYTES == 2 || ELEMENT_BYTES == 4 || ELEMENT_BYTES == 8, "a logit");
  // (word by word: indexed in a loop the words would go through memory)
  uint32_t a = r.w[0], b = r.w[1], c = r.w[2], d = r.w[3];
  if (ELEMENT_BYTES == 2 && (count & 1) != 0) {
    a = (a >> 16) | (b << 16);
    b = (b >> 16) | (c << 16);
    c = (c >> 16) | (d << 16);
    d = d >> 16;
  }
  const int words = ELEMENT_BYTES == 2 ? count >> 1 : ELEMENT_BYTES == 4 ? count : 2 * count;
  if (ELEMENT_BYTES != 8 && (words & 1) != 0) {
    a = b;
    b = c;
    c = d;
  }
  if ((words & 2) != 0) {
    a = c;
    b = d;
  }
  return Raw{{a, b, c, d}};
}

}  // namespace bn_rows
