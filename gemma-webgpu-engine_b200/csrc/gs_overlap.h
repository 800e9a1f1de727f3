// Whether rows that a call writes share bytes with one another or with rows that it reads (host side, no device needed).
#pragma once
#include <cstdint>

namespace gs {

// tokens x heads rows of `row` bytes at base + t · token + h · head (bytes).
struct RowGrid {
  std::uintptr_t base;
  std::int64_t tokens, heads, token, head, row;
};

namespace overlap {
using wide = __int128;  // (a grid's extent passes 2^63 at the limits of its counts and strides)

inline wide extent(const RowGrid& a) {
  return static_cast<wide>(a.tokens - 1) * a.token + static_cast<wide>(a.heads - 1) * a.head + a.row;
}
// Whether some t in (-tokens, tokens) brings x + t · token within a row of 0.
inline bool meets(wide x, const RowGrid& a) {
  wide t = -x / a.token;
  for (wide k = t - 1; k <= t + 1; ++k) {
    const wide at = k >= a.tokens ? a.tokens - 1 : k <= -a.tokens ? 1 - a.tokens : k, y = x + at * a.token;
    if (y < a.row && -y < a.row) return true;
  }
  return false;
}
}  // namespace overlap

// Rows of one grid that share bytes.  (Strides are at least a row; a nested grid, as any slice of a tensor is, has none.)
inline bool rows_overlap(const RowGrid& a) {
  using overlap::wide;
  if (a.tokens < 2 || a.heads < 2) return false;
  if (static_cast<wide>(a.heads - 1) * a.head + a.row <= a.token || static_cast<wide>(a.tokens - 1) * a.token + a.row <= a.head) return false;
  for (std::int64_t h = 1; h < a.heads; ++h)
    if (overlap::meets(static_cast<wide>(h) * a.head, a)) return true;
  return false;
}

// Rows of two grids with the same counts and row size that share bytes.  Exact where the strides are the same, or the heads of a
// token fit into the token stride that both have; any other two grids whose extents meet count as overlapping.
inline bool rows_overlap(RowGrid a, RowGrid b) {
  using overlap::wide;
  if (a.tokens < 1 || a.heads < 1) return false;
  if (a.heads == 1) a.head = b.head = a.row;
  if (a.tokens == 1) a.token = b.token = static_cast<std::int64_t>(1) << 62;  // (never used)
  const wide d = static_cast<wide>(b.base) - static_cast<wide>(a.base);
  if (d >= overlap::extent(a) || -d >= overlap::extent(b)) return false;
  if (a.token == b.token && a.head == b.head) {
    for (std::int64_t h = 1 - a.heads; h < a.heads; ++h)
      if (overlap::meets(d + static_cast<wide>(h) * a.head, a)) return true;
    return false;
  }
  if (a.token != b.token) return true;
  const wide ea = static_cast<wide>(a.heads - 1) * a.head + a.row, eb = static_cast<wide>(b.heads - 1) * b.head + b.row;
  wide r = d % a.token;
  if (r < 0) r += a.token;
  return r < ea || r + eb > a.token;
}

}  // namespace gs
