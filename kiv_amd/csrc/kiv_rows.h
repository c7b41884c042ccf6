// Whether sets of strided rows share memory, for the arguments' checks.
// Plain C++, so that it is also checked on the host.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace kiv {

// Rows of `row` bytes at p + i0 stride[0] + i1 stride[1] + i2 stride[2],
// 0 <= ij < n[j] (strides in bytes).
struct RowSet {
  const void *p;
  int64_t stride[3], n[3], row;
};

// An axis of two sets: its stride, and the ranges of both.
struct RowAxis {
  int64_t s, na, nb;
};

inline bool rows_empty(const RowSet &a) { return a.n[0] < 1 || a.n[1] < 1 || a.n[2] < 1; }

// Axes by falling stride; true if each steps over all that the axes behind it
// reach, so that a row's place gives its indexes.
inline bool rows_nested(RowAxis *x, int n, int64_t row) {
  std::sort(x, x + n, [](const RowAxis &a, const RowAxis &b) { return a.s > b.s; });
  int64_t reach = row;
  for (int i = n - 1; i >= 0; --i) {
    if (x[i].s < reach) return false;
    reach += x[i].s * (std::max(x[i].na, x[i].nb) - 1);
  }
  return true;
}

// Rows of a set over another of its rows (or maybe so: strides that interleave).
inline bool rows_fold(const RowSet &a) {
  if (rows_empty(a)) return false;
  RowAxis x[3];
  int n = 0;
  for (int i = 0; i < 3; ++i)
    if (a.n[i] > 1) x[n++] = {a.stride[i] < 0 ? -a.stride[i] : a.stride[i], a.n[i], a.n[i]};
  return !rows_nested(x, n, a.row);
}

inline bool rows_meet(int64_t delta, const RowAxis *x, int n, int64_t row) {
  if (n == 0) return delta > -row && delta < row;
  const int64_t d = delta / x->s - (delta % x->s < 0);  // the axes behind this one reach less than s
  for (int64_t k = d; k <= d + 1; ++k)
    if (k > -x->nb && k < x->na && rows_meet(delta - k * x->s, x + 1, n - 1, row)) return true;
  return false;
}

// The sets share memory.  Exact where both have the same strides and these
// nest, as slices of one buffer have; otherwise sets whose ranges of addresses
// meet are taken to share it.
inline bool rows_overlap(const RowSet &a, const RowSet &b) {
  if (rows_empty(a) || rows_empty(b)) return false;
  int64_t pa = (int64_t)(uintptr_t)a.p, pb = (int64_t)(uintptr_t)b.p, ea = pa + a.row, eb = pb + b.row;
  RowAxis x[3];
  int n = 0;
  bool alike = a.row == b.row;
  for (int i = 0; i < 3; ++i) {
    const int64_t wa = a.stride[i] * (a.n[i] - 1), wb = b.stride[i] * (b.n[i] - 1);
    (wa < 0 ? pa : ea) += wa;
    (wb < 0 ? pb : eb) += wb;
    const bool one_a = a.n[i] == 1 || a.stride[i] == 0, one_b = b.n[i] == 1 || b.stride[i] == 0;
    if (one_a && one_b) continue;
    const int64_t sa = one_a ? b.stride[i] : a.stride[i], sb = one_b ? a.stride[i] : b.stride[i];
    const int64_t s = sa < 0 ? -sa : sa;
    alike = alike && s == (sb < 0 ? -sb : sb);
    x[n++] = {s, one_a ? 1 : a.n[i], one_b ? 1 : b.n[i]};
  }
  if (ea <= pb || eb <= pa) return false;
  if (!alike || !rows_nested(x, n, a.row)) return true;
  return rows_meet(pb - pa, x, n, a.row);  // from the lowest row of each
}

// One and the same rows, index by index.
inline bool rows_same(const RowSet &a, const RowSet &b) {
  bool same = a.p == b.p && a.row == b.row;
  for (int i = 0; i < 3; ++i) same = same && a.n[i] == b.n[i] && (a.n[i] == 1 || a.stride[i] == b.stride[i]);
  return same;
}

}  // namespace kiv
