// Whether the rows of tensors share memory (host).  A call that writes one
// of them while other blocks read or write the other is refused.
#pragma once

#include <stdint.h>

namespace mw8 {

// Rows of `len` bytes at p + i outer + j inner, i < n_outer, j < n_inner
// (strides in bytes, any sign).  A contiguous tensor is one row.
struct RowSet {
  const void* p;
  int64_t len;
  int64_t n_outer, outer, n_inner, inner;
};

using wide_t = __int128;  // row counts times strides pass 64 bits

inline RowSet one_row(const void* p, int64_t len) { return {p, p ? len : 0, 1, 0, 1, 0}; }

inline bool row_set_empty(const RowSet& r) { return r.len <= 0 || r.n_outer <= 0 || r.n_inner <= 0; }

// Puts the rows in order: the strides of single steps 0, the larger one outside.
inline RowSet row_set_sorted(RowSet r) {
  if (r.n_outer == 1) r.outer = 0;
  if (r.n_inner == 1) r.inner = 0;
  if (r.n_outer == 1 || (r.n_inner != 1 && r.outer < r.inner)) {
    const int64_t n = r.n_outer, s = r.outer;
    r.n_outer = r.n_inner, r.outer = r.inner;
    r.n_inner = n, r.inner = s;
  }
  return r;
}

// Whether the rows of one tensor lie apart: one stride holds a row, the other
// all of its steps (strides not negative).
inline bool rows_apart(RowSet r) {
  r = row_set_sorted(r);
  const wide_t span = static_cast<wide_t>(r.n_inner - 1) * r.inner + r.len;
  return (r.n_inner == 1 || r.inner >= r.len) && (r.n_outer == 1 || r.outer >= span);
}

// First and last byte + 1 of a set, from its own p.
inline void row_set_range(const RowSet& r, wide_t& lo, wide_t& hi) {
  const wide_t a = static_cast<wide_t>(r.n_outer - 1) * r.outer, b = static_cast<wide_t>(r.n_inner - 1) * r.inner;
  lo = (a < 0 ? a : 0) + (b < 0 ? b : 0);
  hi = (a > 0 ? a : 0) + (b > 0 ? b : 0) + r.len;
}

// Whether a byte of `at`, `at + 1`, ... `at + len - 1` (from w.p) lies in a row
// of w, whose rows lie apart and which is sorted.
inline bool row_meets(const RowSet& w, wide_t at, int64_t len) {
  const wide_t span = static_cast<wide_t>(w.n_inner - 1) * w.inner + w.len;
  // steps k whose [k stride, k stride + size) meets [at, at + len)
  auto steps = [](wide_t at, int64_t len, wide_t size, int64_t stride, int64_t n, int64_t& k0, int64_t& k1) {
    k0 = 0, k1 = n;
    if (n == 1) {
      if (at >= size || at + len <= 0) k1 = 0;
      return;
    }
    auto floor_div = [](wide_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
    const wide_t first = floor_div(at - size, stride) + 1, last = floor_div(at + len - 1, stride) + 1;
    if (first > k0) k0 = first < n ? static_cast<int64_t>(first) : n;
    if (last < k1) k1 = last > 0 ? static_cast<int64_t>(last) : 0;
  };
  int64_t o0, o1, i0, i1;
  steps(at, len, span, w.outer, w.n_outer, o0, o1);
  for (int64_t k = o0; k < o1; ++k) {
    steps(at - static_cast<wide_t>(k) * w.outer, len, w.len, w.inner, w.n_inner, i0, i1);
    if (i0 < i1) return true;
  }
  return false;
}

// Whether a row of w (rows_apart) shares a byte with a row of x.  Exact: bytes
// ranges and, for views of one buffer (equal strides), the rows' places within a
// stride settle the usual calls at once; any other layout is walked row by row.
inline bool row_sets_meet(RowSet w, RowSet x) {
  if (row_set_empty(w) || row_set_empty(x)) return false;
  w = row_set_sorted(w), x = row_set_sorted(x);
  const wide_t d = static_cast<wide_t>(reinterpret_cast<intptr_t>(x.p)) - reinterpret_cast<intptr_t>(w.p);
  wide_t wl, wh, xl, xh;
  row_set_range(w, wl, wh);
  row_set_range(x, xl, xh);
  if (d + xh <= wl || wh <= d + xl) return false;
  // within a stride that both share: w's bytes [0, size), x's [at, at + size)
  auto beside = [&](int64_t stride, wide_t w_size, wide_t x_size) {
    if (stride <= 0) return false;
    wide_t at = d % stride;
    if (at < 0) at += stride;
    return at >= w_size && at + x_size <= stride;
  };
  if (w.outer == x.outer && x.inner >= 0 &&
      beside(w.outer, static_cast<wide_t>(w.n_inner - 1) * w.inner + w.len, static_cast<wide_t>(x.n_inner - 1) * x.inner + x.len))
    return false;
  if (w.inner == x.inner && w.inner > 0 && w.outer % w.inner == 0 && x.outer % w.inner == 0 && beside(w.inner, w.len, x.len))
    return false;
  for (int64_t i = 0; i < x.n_outer; ++i)
    for (int64_t j = 0; j < x.n_inner; ++j)
      if (row_meets(w, d + static_cast<wide_t>(i) * x.outer + static_cast<wide_t>(j) * x.inner, x.len)) return true;
  return false;
}

// Whether any of `outs` shares a byte with another of them or one of `ins`
// (one_row each).
template <int NO, int NI>
bool any_meet(const RowSet (&outs)[NO], const RowSet (&ins)[NI]) {
  for (int i = 0; i < NO; ++i) {
    for (int j = i + 1; j < NO; ++j)
      if (row_sets_meet(outs[i], outs[j])) return true;
    for (const RowSet& x : ins)
      if (row_sets_meet(outs[i], x)) return true;
  }
  return false;
}

}  // namespace mw8
