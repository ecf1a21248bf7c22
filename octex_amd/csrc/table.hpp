// Launchers of rows of a table by ids, and of the table's gradient (table.hip).  Shapes, types and pointers are checked by the
// callers (operators.cpp).
#pragma once

#include "rows.hpp"

#include <algorithm>

namespace cuvs::neighbors::octex::detail {

constexpr int64_t kMaxRowWidth = int64_t{1} << 24;  // values of a row

/** A table [n, d], rows `stride` apart; scales [n] of int8 rows, else null. */
struct table_rows {
  const void* x;
  elem type;
  int64_t n, stride;
  const float* scales;
};

/** m ids, `stride` apart; ids outside [0, n) are padding. */
struct row_ids {
  const void* ids;
  bool wide;  // int64, else int32
  int64_t stride, m;
};

/** A matrix of rows of d values that is read or written. */
struct value_rows {
  void* x;
  elem type;
  int64_t stride;
};

/** out[i] = scale * table[ids[i]], padding 0. */
void launch_embed(table_rows const& table, row_ids const& ids, int64_t d, float scale, value_rows const& out, hipStream_t s);

/** The bytes of workspace (at a multiple of 256) that launch_embed_backward needs. */
auto embed_backward_workspace(int64_t m, int64_t n, int64_t d) -> int64_t;

constexpr int kClearRows = 4096;  // of a workgroup, at most

/** Rows that a workgroup clears of the `left` ones that a gradient's sort has not: up to 32 KB (1 MB: 288 us for what takes 276),
 * in 2048 workgroups or more.  At most 2^23 of them, whatever the table's size: with those that sum, fewer than 2^21, a launch
 * stays below 2^32 work-items. */
inline auto rows_to_clear(int64_t left, int64_t row_bytes) -> int64_t
{
  const int64_t enough = std::min((int64_t{32} << 10) / row_bytes, (left + 2047) / 2048);
  return std::clamp<int64_t>(std::max(enough, (left + (1 << 23) - 1) >> 23), 1, kClearRows);
}

/** out[v] = scale * the sum of grad[i] with ids[i] = v, of n rows; with `add` that much more than it held. */
void launch_embed_backward(value_rows const& grad, row_ids const& ids, int64_t n, int64_t d, float scale, bool add,
                           value_rows const& out, void* workspace, hipStream_t s);

}  // namespace cuvs::neighbors::octex::detail
