// dc_span.h -- what a call's strided buffers cover, for the checks of its
// arguments.  Plain C++, so that a host program can test them.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

namespace dcc {

// The addresses that a strided buffer covers, from its first to behind its
// last byte, for the overlap checks.
struct Dim {
  int64_t n, stride;
};
struct Span {
  uintptr_t lo = 0, hi = 0;
  bool ok = true;
  bool meets(const Span& o) const { return lo < o.hi && o.lo < hi; }
};
static inline Span span(const void* p, int elem, std::initializer_list<Dim> dims) {
  Span s;
  if (!p) return s;
  int64_t last = 0;
  bool empty = false;
  for (const Dim& d : dims) {
    if (d.stride < 0) s.ok = false;
    if (d.n <= 0) empty = true;
    else last += (d.n - 1) * d.stride;
  }
  if (empty || !s.ok) return s;
  s.lo = (uintptr_t)p;
  s.hi = s.lo + (uintptr_t)(last + 1) * elem;
  return s;
}
// Whether a buffer of es-byte elements begins, and each of its rows in these
// dimensions, on a boundary of `align` bytes.
static inline bool aligned(const void* p, int es, int align, std::initializer_list<Dim> dims) {
  uintptr_t m = (uintptr_t)p;
  for (const Dim& d : dims)
    if (d.n > 1) m |= (uintptr_t)(d.stride * es);
  return !(m & (align - 1));
}

// Whether no two elements of a buffer share an address, as those of a written one
// must not (a tensor expanded over a dimension has its stride 0).  Taken from the
// smallest stride up, each dimension has to step over all that lies within it;
// interleaved and permuted layouts do.
static inline bool apart(std::initializer_list<Dim> dims, std::initializer_list<Dim> more = {}) {
  Dim d[8];
  int n = 0;
  for (auto* list : {&dims, &more})
    for (const Dim& x : *list) {
      if (x.n <= 0) return true;
      if (x.n > 1) d[n++] = x;
    }
  std::sort(d, d + n, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  int64_t extent = 1;
  for (int i = 0; i < n; i++) {
    if (d[i].stride < extent) return false;
    extent += d[i].stride * (d[i].n - 1);
  }
  return true;
}
// Whether two written buffers of the same dimensions share no element: apart as a
// whole, or (keys and values of one buffer) with the same strides and interleaved,
// as if one more dimension stepped from the one to the other.
static inline bool twins_apart(const Span& a, const Span& b, int elem, std::initializer_list<Dim> da,
                               std::initializer_list<Dim> db) {
  if (!a.meets(b)) return true;
  if (!std::equal(da.begin(), da.end(), db.begin(), db.end(),
                  [](const Dim& x, const Dim& y) { return x.n == y.n && (x.n < 2 || x.stride == y.stride); }))
    return false;
  const uintptr_t step = a.lo < b.lo ? b.lo - a.lo : a.lo - b.lo;
  return step % elem == 0 && apart(da, {{2, (int64_t)(step / elem)}});
}

}  // namespace dcc
