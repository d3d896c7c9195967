// Integer arithmetic of the paged cache: what a mask leaves live for a range of query
// positions, as hulls of key ranges, verdicts on blocks and words of 32 keys, and which slot a
// position has.  Plain C++ without HIP types, so it also compiles for the host.
//
// Positions and lengths are below 2^30 (checked by the entry points) and a term's parameters
// are clamped to 2^30 - 1, which is larger than every distance: no sum here overflows.
#pragma once

#include <stdint.h>

#include "polyattn_amd.h"

#if defined(__HIP__) || defined(__HIPCC__)
#define PA_HD __host__ __device__ __forceinline__
#else
#define PA_HD inline
#endif

namespace pa {

constexpr int32_t kMaxPosition = (1 << 30) - 1;  // positions and lengths stay at or below it

// The terms of a pa_mask without tables.  They are walked in rolled loops, so there is one copy of
// each term's code: the first one, which most masks consist of, from registers, the others through
// a pointer (on the device one into the kernel's arguments, read by scalar loads).
template <typename Ptr>
struct PageMask {
  int32_t n_include, n_exclude;
  pa_term first;
  Ptr terms;
  PA_HD pa_term term(int i) const {
    return i == 0 ? first : pa_term{terms[i].kind, terms[i].p0, terms[i].p1, terms[i].p2};
  }
};

enum Verdict { kDead = 0, kPartial = 1, kFull = 2 };

PA_HD int32_t imin(int32_t x, int32_t y) { return x < y ? x : y; }
PA_HD int32_t imax(int32_t x, int32_t y) { return x > y ? x : y; }

// One term on every pair of queries q0 .. q1 and keys k0 .. k1: all live (kFull), none (kDead),
// or not decided from the ranges (kPartial).
PA_HD int term_verdict(const pa_term& t, int32_t q0, int32_t q1, int32_t k0, int32_t k1) {
  if (t.kind == PA_FULL) return kFull;
  const int32_t dmin = q0 - k1, dmax = q1 - k0;
  if (t.kind == PA_PREFIX_LM) {
    if (dmin >= 0 || (q1 < t.p0 && k1 < t.p0)) return kFull;
    return dmax < 0 && !(q0 < t.p0 && k0 < t.p0) ? kDead : kPartial;
  }
  if (dmax < 0) return kDead;
  const bool causal = dmin >= 0;
  switch (t.kind) {
    case PA_CAUSAL:
      return causal ? kFull : kPartial;
    case PA_WINDOW:
      if (dmin >= t.p0) return kDead;
      return causal && dmax < t.p0 ? kFull : kPartial;
    case PA_DILATED:
      if (causal && t.p0 == 1) return kFull;
      return dmax / t.p0 * t.p0 < dmin ? kDead : kPartial;
    case PA_LOCAL_STRIDED:
      if (causal && (t.p1 == 1 || dmax < t.p0)) return kFull;
      return dmin >= t.p0 && dmax / t.p1 * t.p1 < dmin ? kDead : kPartial;
    case PA_TWOBAND:
      if (causal && (dmax < t.p0 || (dmin >= t.p1 && dmax < t.p1 + t.p2))) return kFull;
      return dmin >= t.p0 && (dmax < t.p1 || dmin >= t.p1 + t.p2) ? kDead : kPartial;
    case PA_SINKS:
      if (causal && (dmax < t.p0 || k1 < t.p1)) return kFull;
      return dmin >= t.p0 && k0 >= t.p1 ? kDead : kPartial;
    default:
      return kDead;
  }
}

// The mask on the same pairs.
template <typename Ptr>
PA_HD int mask_verdict(const PageMask<Ptr>& m, int32_t q0, int32_t q1, int32_t k0, int32_t k1) {
  int inc = kDead, exc = kDead;
#pragma unroll 1
  for (int i = 0; i < m.n_include + m.n_exclude; ++i) {
    const int v = term_verdict(m.term(i), q0, q1, k0, k1);
    if (i < m.n_include)
      inc = imax(inc, v);
    else
      exc = imax(exc, v);
  }
  if (inc == kDead || exc == kFull) return kDead;
  return exc == kDead ? inc : (int)kPartial;
}

// Bits lo - k0 .. hi - k0 - 1 of a word whose bit b is key k0 + b (k0 >= 0).
PA_HD uint32_t range_word(int32_t lo, int32_t hi, int32_t k0) {
  const int32_t a = imin(imax(imax(lo, 0) - k0, 0), 32), b = imin(imax(imax(hi, 0) - k0, 0), 32);
  if (b <= a) return 0u;
  return (b >= 32 ? 0xffffffffu : (1u << b) - 1u) & ~((1u << a) - 1u);  // (a < b <= 32)
}

// Bits of the keys k0 + b <= q with (q - k0 - b) a multiple of s.
PA_HD uint32_t lattice_word(int32_t q, int32_t s, int32_t k0) {
  if (q < k0) return 0u;
  const int32_t f = (q - k0) % s;
  if (f >= 32) return 0u;
  uint32_t w = 1u << f;
  for (int32_t d = s; d < 32; d *= 2) w |= w << d;
  return w & range_word(k0, q + 1, k0);
}

// Bit b: key k0 + b is live for query q by one term (k0 >= 0).
PA_HD uint32_t term_word(const pa_term& t, int32_t q, int32_t k0) {
  switch (t.kind) {
    case PA_CAUSAL:
      return range_word(0, q + 1, k0);
    case PA_WINDOW:
      return range_word(q - t.p0 + 1, q + 1, k0);
    case PA_DILATED:
      return lattice_word(q, t.p0, k0);
    case PA_LOCAL_STRIDED:
      return range_word(q - t.p0 + 1, q + 1, k0) | lattice_word(q, t.p1, k0);
    case PA_TWOBAND:
      return range_word(q - t.p0 + 1, q + 1, k0) | range_word(imax(q, 0) - t.p1 - t.p2 + 1, q - t.p1 + 1, k0);
    case PA_SINKS:
      return range_word(q - t.p0 + 1, q + 1, k0) | range_word(0, imin(t.p1, q + 1), k0);
    case PA_PREFIX_LM:
      return range_word(0, q + 1, k0) | (q < t.p0 ? range_word(0, t.p0, k0) : 0u);
    case PA_FULL:
      return 0xffffffffu;
    default:
      return 0u;
  }
}

// Bit b: key k0 + b is cached (below len) and live for query q.
template <typename Ptr>
PA_HD uint32_t mask_word(const PageMask<Ptr>& m, int32_t q, int32_t k0, int32_t len) {
  uint32_t inc = 0u, exc = 0u;
#pragma unroll 1
  for (int i = 0; i < m.n_include + m.n_exclude; ++i) {
    const uint32_t w = term_word(m.term(i), q, k0);
    if (i < m.n_include)
      inc |= w;
    else
      exc |= w;
  }
  return inc & ~exc & range_word(0, len, k0);
}

// Keys that may be live for queries q0 .. q1 of a request of len tokens, in blocks of 1 << lg
// keys: blocks 0 .. low - 1 and first .. first + high - 1 (first >= low), as a list of
// low + high entries.
struct KeyList {
  int32_t low, first, high;
  PA_HD int32_t count() const { return low + high; }
  PA_HD int32_t block(int32_t j) const { return j < low ? j : first + j - low; }
  // Entries before block b.
  PA_HD int32_t before(int32_t b) const { return imin(low, imax(b, 0)) + imin(imax(b - first, 0), high); }
};

template <typename Ptr>
PA_HD KeyList key_list(const PageMask<Ptr>& m, int32_t q0, int32_t q1, int32_t len, int lg) {
  int32_t a = 0, b = len, e = 0;  // [0, a) and [b, e)
  const int32_t qc = imax(q0, 0);  // (a query before the first token sees what none of these adds)
#pragma unroll 1
  for (int i = 0; i < m.n_include; ++i) {
    const pa_term t = m.term(i);
    int32_t lo = 0, hi = q1 + 1;
    switch (t.kind) {
      case PA_WINDOW:
        lo = qc - t.p0 + 1;
        break;
      case PA_SINKS:
        lo = qc - t.p0 + 1;
        a = imax(a, imin(t.p1, hi));
        break;
      case PA_TWOBAND:
        lo = qc - imax(t.p0, t.p2 > 0 ? t.p1 + t.p2 : 0) + 1;
        break;
      case PA_PREFIX_LM:
        if (q0 < t.p0) hi = imax(hi, t.p0);
        break;
      case PA_FULL:
        hi = len;
        break;
      default:
        break;
    }
    if (lo < hi) {
      b = imin(b, imax(lo, 0));
      e = imax(e, hi);
    }
  }
  a = imin(imax(a, 0), len);
  e = imin(e, len);
  const int32_t one = (1 << lg) - 1;
  KeyList l;
  l.low = (a + one) >> lg;
  const int32_t end = e > 0 ? (e + one) >> lg : 0;
  l.first = imax(b >> lg, l.low);
  l.high = imax(end - l.first, 0);
  return l;
}

// Queries that may see a key of k0 .. k1: positions lo .. hi.
struct QueryRange {
  int32_t lo, hi;
};
template <typename Ptr>
PA_HD QueryRange query_range(const PageMask<Ptr>& m, int32_t k0, int32_t k1) {
  QueryRange r{kMaxPosition, -1};
#pragma unroll 1
  for (int i = 0; i < m.n_include; ++i) {
    const pa_term t = m.term(i);
    int32_t lo = k0, hi = kMaxPosition;
    switch (t.kind) {
      case PA_WINDOW:
        hi = imin(k1, kMaxPosition - t.p0) + t.p0 - 1;
        break;
      case PA_SINKS:
        if (k0 >= t.p1) hi = imin(k1, kMaxPosition - t.p0) + t.p0 - 1;
        break;
      case PA_TWOBAND: {
        const int32_t far = imax(t.p0, t.p2 > 0 ? imin(t.p1, kMaxPosition - t.p2) + t.p2 : 0);
        hi = imin(k1, kMaxPosition - far) + far - 1;
        break;
      }
      case PA_PREFIX_LM:
        if (k0 < t.p0) lo = 0;
        break;
      case PA_FULL:
        lo = 0;
        break;
      default:
        break;
    }
    r.lo = imin(r.lo, lo);
    r.hi = imax(r.hi, hi);
  }
  return r;
}

// Page of a request's table, or -1 where it names none of the cache.
PA_HD int32_t checked_page(int32_t page, int64_t n_pages) {
  return (uint32_t)page < (uint64_t)n_pages ? page : -1;
}

// Slot (row of the cache) of a position in a page, or -1.
PA_HD int32_t slot_of(int32_t page, int32_t position, int page_lg, int64_t n_pages) {
  const int32_t p = checked_page(page, n_pages);
  return p < 0 ? -1 : (p << page_lg) + (position & ((1 << page_lg) - 1));
}

// Division of numbers below 2^30 by d in 1 .. 65535 as a product: with l = ceil(log2 d), k = max(32,
// 30 + l) and m = ceil(2^k / d), m d - 2^k < d <= 2^(k - 30), so x m / 2^k is above x / d by less
// than 1 / d.
struct Divisor {
  uint32_t d, m, shift;  // shift: k - 32
};
inline Divisor divisor_of(uint32_t d) {
  int l = 0;
  while ((1u << l) < d) ++l;
  const int k = l > 2 ? 30 + l : 32;
  return {d, (uint32_t)(((1ull << k) + d - 1) / d), (uint32_t)(k - 32)};  // (m is not used for d = 1)
}
PA_HD int32_t divide(int32_t x, const Divisor& v) {
  return v.d == 1 ? x : (int32_t)((uint32_t)(((uint64_t)(uint32_t)x * v.m) >> 32) >> v.shift);
}

// Rows and length of a request, whatever its entries hold: rows start .. start + n - 1 of T
// packed ones, len within the table's reach.
struct Request {
  int32_t start, n, len;
};
PA_HD Request request_of(int32_t s0, int32_t s1, int32_t len, int32_t T, int32_t max_len) {
  Request r;
  r.start = imin(imax(s0, 0), T);
  r.n = imin(imax(s1, r.start), T) - r.start;
  r.len = imin(imax(len, 0), max_len);
  return r;
}

}  // namespace pa
