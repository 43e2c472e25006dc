// Whether tensors share memory, for entry points whose outputs must lie apart
// from what they read.  Host only.
#pragma once

#include <stdint.h>

namespace qs {

// `count` rows of `width` bytes, `apart` bytes from one to the next.
struct Rows {
  const void* at;
  int64_t count, apart, width;
};

inline bool share_memory(const Rows& a, const Rows& b) {
  typedef __int128 wide;
  if (a.count < 1 || b.count < 1 || a.width < 1 || b.width < 1) return false;
  const wide a0 = (wide) reinterpret_cast<uintptr_t>(a.at), b0 = (wide) reinterpret_cast<uintptr_t>(b.at);
  const wide a1 = a0 + (wide)(a.count - 1) * a.apart + a.width, b1 = b0 + (wide)(b.count - 1) * b.apart + b.width;
  if (a1 <= b0 || b1 <= a0) return false;
  if (a.count == 1 && b.count == 1) return true;
  if (a.apart == b.apart || a.count == 1 || b.count == 1) {
    // columns of one tensor, say: row i of a and row j of b meet where (i - j)
    // apart lies between b0 - a0 - a.width and b0 - a0 + b.width
    const wide apart = a.count > 1 ? a.apart : b.apart, d = b0 - a0;
    if (apart == 0) return d < a.width && -d < b.width;
    auto below = [](wide x, wide y) { return x / y - (x % y < 0); };  // the whole quotient, rounded down
    wide first = below(d - a.width, apart) + 1, last = below(d + b.width - 1, apart);
    if (first < 1 - (wide)b.count) first = 1 - (wide)b.count;
    if (last > a.count - 1) last = a.count - 1;
    return first <= last;
  }
  if (a.apart == 0) return share_memory(Rows{a.at, 1, 0, a.width}, b);
  if (b.apart == 0) return share_memory(a, Rows{b.at, 1, 0, b.width});
  wide i = 0, j = 0;
  while (i < a.count && j < b.count) {
    const wide x = a0 + i * a.apart, y = b0 + j * b.apart;
    if (x + a.width <= y) ++i;
    else if (y + b.width <= x) ++j;
    else return true;
  }
  return false;
}

}  // namespace qs
