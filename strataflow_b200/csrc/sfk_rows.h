// sfk_rows.h -- whether strided rows of two tensors share memory.  Host only.
#pragma once
#include <cstdint>

namespace sfk {

struct Rows {
  const void* at;
  int64_t stride, width, n;  // bytes from row to row (>= width), bytes of a row, rows
};

inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0

// Exact: rows of one that lie between the rows of the other (q beside k and v in packed rows) do not meet them.
inline bool rows_meet(const Rows& a, const Rows& b) {
  if (a.n <= 0 || b.n <= 0) return false;
  if (a.n > b.n) return rows_meet(b, a);
  // from b's first byte; a row at x meets b's row j when j stride < x + width_a and j stride + width_b > x
  const int64_t off = (int64_t)((uintptr_t)a.at - (uintptr_t)b.at);
  auto meets = [&](int64_t x, int64_t first, int64_t last) {
    const int64_t lo = floor_div(x - b.width, b.stride) + 1, hi = floor_div(x + a.width - 1, b.stride);
    return (lo > first ? lo : first) <= (hi < last ? hi : last);
  };
  if (off + (a.n - 1) * a.stride + a.width <= 0 || off >= (b.n - 1) * b.stride + b.width) return false;
  // rows i and j of one stride meet by i - j alone
  if (a.stride == b.stride) return meets(off, -(a.n - 1), b.n - 1);
  for (int64_t i = 0; i < a.n; ++i)
    if (meets(off + i * a.stride, 0, b.n - 1)) return true;
  return false;
}

// The same rows: out of q's own memory, each row where it was.
inline bool same_rows(const Rows& a, const Rows& b) {
  return a.at == b.at && a.n == b.n && a.width == b.width && (a.stride == b.stride || a.n == 1);
}

}  // namespace sfk
