// Whether rows of one matrix share bytes with rows of another: the host's check of
// outputs that other workgroups would still read as inputs.  No allocation and no loop
// over rows where the strides are equal, as they are where both are columns of one buffer.
#pragma once

#include <stdint.h>

#include <utility>

namespace mi {

struct Rows {
  const void* base;
  int64_t stride, rows, width;  // bytes from row to row; bytes of a row
};

namespace overlap {

struct Span {
  __int128 at, stride, rows, width;
};

// Span a's row i and b's row j meet where d - a.width < (i - j) stride < d + b.width, d the
// distance from a to b, of one positive stride: some i - j of the rows' range, other than 0 if `apart`.
inline bool meet_in_step(const Span& a, const Span& b, bool apart) {
  const __int128 s = a.stride, d = b.at - a.at, over = d - a.width;
  __int128 m = over / s - (over % s < 0) + 1;  // the least above over / s
  if (m < 1 - b.rows) m = 1 - b.rows;
  for (; m < a.rows && m * s < d + b.width; ++m)
    if (!apart || m) return true;
  return false;
}

}  // namespace overlap

// Whether any byte of a's rows is one of b's; with `apart`, of two rows of unlike number
// (rows of unlike or negative strides that meet count as such).
inline bool rows_meet(const Rows& x, const Rows& y, bool apart = false) {
  using overlap::Span;
  auto span = [](const Rows& r) -> Span {
    Span s = {__int128(reinterpret_cast<uintptr_t>(r.base)), r.stride, r.rows, r.width};
    if (s.stride < 0) s.at += (s.rows - 1) * s.stride, s.stride = -s.stride;
    return s;
  };
  Span a = span(x), b = span(y);
  if (a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  if (a.at + (a.rows - 1) * a.stride + a.width <= b.at || b.at + (b.rows - 1) * b.stride + b.width <= a.at) return false;
  if (x.stride < 0 || y.stride < 0) apart = false;
  if ((a.stride == 0 && a.rows > 1) || (b.stride == 0 && b.rows > 1)) apart = false;  // every row is every other
  if (a.stride == 0) a.rows = 1;
  if (b.stride == 0) b.rows = 1;
  if (a.rows == 1) a.stride = b.stride;
  if (b.rows == 1) b.stride = a.stride;
  if (a.stride == 0) return !apart;  // one row each, which meet
  if (a.stride == b.stride) return overlap::meet_in_step(a, b, apart);
  if (a.rows > b.rows) std::swap(a, b);
  for (Span row = {a.at, b.stride, 1, a.width}; a.rows > 0; --a.rows, row.at += a.stride)
    if (overlap::meet_in_step(row, b, false)) return true;
  return false;
}

}  // namespace mi
