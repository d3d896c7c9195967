// Whether tensors of the paged cache's calls share memory, from their strides.  Host code, plain C++.
#pragma once

#include <stdint.h>

namespace pa {

typedef __int128 wide;  // (no size times a stride overflows it)

// n[0] x n[1] x .. rows of w bytes, s[i] bytes apart, the lowest one at `at`.
template <int N>
struct Strided {
  wide at, w;
  int64_t n[N];
  wide s[N];
};
// (strides in units of `unit` bytes, of either sign: the same rows counted backwards)
template <int N>
inline Strided<N> strided(const void* p, int64_t w, const int64_t (&n)[N], const int64_t (&s)[N], int unit = 1) {
  Strided<N> x;
  x.at = (wide) reinterpret_cast<uintptr_t>(p);
  x.w = w;
  for (int i = 0; i < N; ++i) {
    x.n[i] = n[i];
    x.s[i] = (s[i] < 0 ? -(wide)s[i] : s[i]) * unit;
    if (s[i] < 0 && n[i] > 0) x.at -= (n[i] - 1) * x.s[i];
  }
  return x;
}
inline Strided<1> flat(const void* p, int64_t bytes) { return strided<1>(p, bytes, {1}, {0}); }

// Bytes from the first to the end of the last.
template <int N>
inline wide span(const Strided<N>& x) {
  wide d = x.w;
  for (int i = 0; i < N; ++i) {
    if (x.n[i] <= 0) return 0;
    d += (x.n[i] - 1) * x.s[i];
  }
  return d;
}
template <int N, int M>
inline bool spans_meet(const Strided<N>& x, const Strided<M>& y) {
  const wide a = span(x), b = span(y);
  return a > 0 && b > 0 && x.at < y.at + b && y.at < x.at + a;
}

// Whether the strides nest: taken from the smallest, each passes all the rows within it.  No two rows
// of such a tensor share a byte.
template <int N>
inline bool nested(const Strided<N>& x) {
  bool done[N] = {};
  wide inside = x.w;
  for (int k = 0; k < N; ++k) {
    int least = -1;
    for (int i = 0; i < N; ++i)
      if (!done[i] && (least < 0 || x.s[i] < x.s[least])) least = i;
    done[least] = true;
    if (x.n[least] < 2) continue;
    if (x.s[least] < inside) return false;
    inside += x.s[least] * (x.n[least] - 1);
  }
  return true;
}

// Whether some row of x and some row of x moved by d bytes and w_y wide share a byte; self (d = 0, w_y =
// w): two different ones.  A difference of indexes j of the second dimension leaves a range of those of
// the first.
inline bool rows_meet(const Strided<2>& x, wide d, wide w_y, bool self) {
  auto floor_div = [](wide a, wide b) { return a / b - (a % b < 0 ? 1 : 0); };
  const wide last = x.n[0] - 1, s = x.s[0];
  for (int64_t j = 1 - x.n[1]; j < x.n[1]; ++j) {
    const wide at = d + j * x.s[1];
    // i in lo .. hi: -w_y < at + i s < w
    wide lo = -last, hi = last;
    if (s > 0) {
      const wide a = floor_div(-w_y - at, s) + 1, b = -floor_div(at - x.w, s) - 1;
      if (a > lo) lo = a;
      if (b < hi) hi = b;
    } else if (at <= -w_y || at >= x.w) {
      continue;
    }
    if (lo <= hi && !(self && j == 0 && lo == 0 && hi == 0)) return true;
  }
  return false;
}

// Whether two rows of x share a byte.
inline bool overlaps_itself(const Strided<2>& x) { return span(x) > 0 && !nested(x) && rows_meet(x, 0, x.w, true); }

// Whether x and y share a byte: exact where they have the same sizes and strides (parts of one buffer's
// rows), else whether their spans do.
template <int N, int M>
inline bool overlap(const Strided<N>& x, const Strided<M>& y) {
  return spans_meet(x, y);
}
inline bool overlap(const Strided<2>& x, const Strided<2>& y) {
  if (!spans_meet(x, y)) return false;
  if (x.n[0] != y.n[0] || x.n[1] != y.n[1] || x.s[0] != y.s[0] || x.s[1] != y.s[1]) return true;
  return rows_meet(x, y.at - x.at, y.w, false);
}

}  // namespace pa
