// Rows of an operand along three axes, and whether two such operands meet.
#pragma once

#include "internal.h"

#include <algorithm>

namespace {

// [batch][heads][tokens] rows of dim elements.
struct RowSet {
  const void *p;
  uint64_t ts, hs, bs;
  uint64_t batch, heads, tokens, dim;

  // A block of row stride ld that holds the set, where there is one: axes whose
  // strides are multiples of ld go along its rows, the others into a row.
  bool as_block(uint64_t ld, uint64_t &rows, uint64_t &cols) const {
    rows = 1;
    cols = dim;
    const uint64_t n[3] = {tokens, heads, batch}, st[3] = {ts, hs, bs};
    for (int i = 0; i < 3; ++i) {
      if (n[i] == 1) continue;
      if (st[i] % ld == 0) rows += (n[i] - 1) * (st[i] / ld);
      else cols += (n[i] - 1) * st[i];
    }
    return cols <= ld;
  }
  uint64_t span() const { return (batch - 1) * bs + (heads - 1) * hs + (tokens - 1) * ts + dim; }
};

// Whether two sets may share an element: not where they lie in blocks of one row
// stride, a token's, head's or batch's, that share none (q and k side by side in
// each token's row, or in each batch: heads before tokens); else by byte range.
bool meet(const RowSet &a, const RowSet &b, uint64_t es) {
  if (!a.p || !b.p) return false;
  for (const uint64_t ld : {a.tokens > 1 ? a.ts : 0, a.heads > 1 ? a.hs : 0, a.batch > 1 ? a.bs : 0}) {
    uint64_t ra, ca, rb, cb;
    if (ld && a.as_block(ld, ra, ca) && b.as_block(ld, rb, cb) &&
        !bwpp_hip_blocks_overlap(a.p, ra, ca, ld, b.p, rb, cb, ld, es))
      return false;
  }
  return bwpp_hip_blocks_overlap(a.p, 1, a.span(), 0, b.p, 1, b.span(), 0, es);
}
bool same_rows(const RowSet &a, const RowSet &b) {
  return a.p == b.p && (a.tokens == 1 || a.ts == b.ts) && (a.heads == 1 || a.hs == b.hs) &&
         (a.batch == 1 || a.bs == b.bs);
}
// Whether the rows of an output are disjoint: every stride passes what lies
// inside it, in some order of the three.
bool disjoint_rows(const RowSet &s) {
  struct Axis {
    uint64_t n, st;
  } ax[3] = {{s.tokens, s.ts}, {s.heads, s.hs}, {s.batch, s.bs}};
  std::sort(ax, ax + 3, [](const Axis &a, const Axis &b) { return a.st < b.st; });
  uint64_t inside = s.dim;
  for (const Axis &a : ax) {
    if (a.n == 1) continue;
    if (a.st < inside) return false;
    inside += (a.n - 1) * a.st;
  }
  return true;
}

}  // namespace
