// Memory that a call reads and writes, and the refusal of outputs that lie over an input or another output (host code).
#pragma once
#include <algorithm>
#include <initializer_list>

#include "common.h"

namespace nmtgan {

// `rows` rows of `width` bytes, `ld` bytes from one to the next (ld >= width)
struct Region {
  const char* name;
  uintptr_t at;
  int64_t rows, ld, width;
  Region(const char* n, const void* p, int64_t r, int64_t l, int64_t w)
      : name(n), at((uintptr_t)p), rows(p && w > 0 ? r : 0), ld(std::max(l, w)), width(w) {}
  Region(const char* n, const void* p, int64_t bytes) : Region(n, p, bytes > 0 ? 1 : 0, bytes, bytes) {}
  int64_t end() const { return (int64_t)at + (rows - 1) * ld + width; }
};
// whether a row of (at, rows, ld, width) meets the bytes [a, a + w)
static inline bool rows_meet(int64_t at, int64_t rows, int64_t ld, int64_t width, int64_t a, int64_t w) {
  const int64_t before = a - width - at;         // the last row that ends at or before a
  const int64_t first = before < 0 ? 0 : before / ld + 1;
  return first < rows && at + first * ld < a + w;
}
// Exact: columns of one buffer (q, k and v of a fused projection, their gradients) lie between each other and do not meet.  Rows of
// the same distance are one comparison, whatever their number; other distances are walked, only where the ranges meet.
static inline bool regions_meet(const Region& x, const Region& y) {
  if (x.rows <= 0 || y.rows <= 0 || x.end() <= (int64_t)y.at || y.end() <= (int64_t)x.at) return false;
  if (x.rows == 1) return rows_meet(y.at, y.rows, y.ld, y.width, x.at, x.width);
  if (y.rows == 1) return rows_meet(x.at, x.rows, x.ld, x.width, y.at, y.width);
  if (x.ld == y.ld)                              // row i of x and j of y: j - i decides
    return rows_meet((int64_t)y.at - (x.rows - 1) * y.ld, x.rows + y.rows - 1, y.ld, y.width, x.at, x.width);
  const Region &a = x.rows < y.rows ? x : y, &b = x.rows < y.rows ? y : x;
  for (int64_t i = 0; i < a.rows; ++i)
    if (rows_meet(b.at, b.rows, b.ld, b.width, a.at + i * a.ld, a.width)) return true;
  return false;
}
static inline int refuse_overlaps(const char* what, std::initializer_list<Region> outputs, std::initializer_list<Region> inputs) {
  for (const Region* o = outputs.begin(); o != outputs.end(); ++o) {
    for (const Region* p = o + 1; p != outputs.end(); ++p)
      NMTGAN_REQUIRE(!regions_meet(*o, *p), "%s: %s overlaps %s", what, o->name, p->name);
    for (const Region& i : inputs) NMTGAN_REQUIRE(!regions_meet(*o, i), "%s: %s overlaps %s", what, o->name, i.name);
  }
  return 0;
}

}  // namespace nmtgan
