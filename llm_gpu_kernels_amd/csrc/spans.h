// Which memory the tensors of a call take: host side, for checks of arguments.
#pragma once

#include <stdint.h>

#include <numeric>

namespace moe {

// Bytes [from, to).
struct Span {
  uintptr_t from, to;
};
inline Span span_of(const void *p, int64_t bytes) { return Span{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes}; }
inline bool meet(Span a, Span b) { return a.from < b.to && b.from < a.to; }

// `n` rows (at least one) of `row` bytes, `stride` (at least `row`) from one to the next.
struct Rows {
  const void *at;
  int64_t stride, row, n;
};
inline Span span_of(const Rows &a) { return span_of(a.at, (a.n - 1) * a.stride + a.row); }
// Whether two such have bytes in common, or may have: rows that lie between each other's, as those
// of the two halves of one tensor, are apart if no two meet by their offsets modulo both
// strides.
inline bool may_meet(const Rows &a, const Rows &b) {
  if (!meet(span_of(a), span_of(b))) return false;
  const int64_t g = std::gcd(a.n > 1 ? a.stride : b.stride, b.n > 1 ? b.stride : a.stride);
  const int64_t off = ((int64_t)((uintptr_t)b.at - (uintptr_t)a.at) % g + g) % g;
  return off < a.row || off + b.row > g;
}

}  // namespace moe
