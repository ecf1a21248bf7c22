// Launchers of the product in 8-bit integers (scores.hip): scores[i][j] = qs[i] * rs[j] * sum_d q[i][d] * r[j][d] +
// bias[j], and of the quantization of rows that feeds it.  Shapes, types and pointers are checked by the callers
// (operators.cpp).
#pragma once

#include "rows.hpp"

namespace cuvs::neighbors::octex::detail {

// the products of k values of -128 x -128 stay within an int32 sum
constexpr int kMaxInt8Width = 131071;

/** codes [m, k] (rows cstride apart) and scales [m] of x [m, k] (rows `stride` apart). */
void launch_quantize_rows(const void* x, elem type, int64_t m, int k, int64_t stride, int8_t* codes, int64_t cstride,
                          float* scales, hipStream_t s);

/** Bytes from row to row of quantized queries of k values: whole 16-byte chunks, and no multiple of 1024, at which the same
 * columns of many rows meet in few channels of the L2 (8192 x 4096 x 16,384 takes 14 % longer there). */
inline auto int8_pitch(int k) -> int64_t
{
  const int64_t pitch = (int64_t{k} + 15) / 16 * 16;
  return pitch % 1024 == 0 ? pitch + 128 : pitch;
}

struct int8_rows {
  const int8_t* x;
  int64_t stride;
  const float* scales;
};

/** Queries: int8 codes with their scales, or floats (no scales) that the product quantizes. */
struct int8_query {
  const void* x;
  elem type;
  int64_t stride;
  const float* scales;
};

/** The bytes that launch_int8_scores needs for the same operands. */
auto int8_scores_workspace(int8_query const& q, int64_t m, int8_rows const& r, int64_t n, int k) -> int64_t;

/** out [m, n] of `type`, rows ostride apart; bias [n] may be null.  workspace at a multiple of 256 bytes. */
void launch_int8_scores(int8_query const& q, int64_t m, int8_rows const& r, int64_t n, int k, const float* bias, void* out,
                        elem type, int64_t ostride, void* workspace, hipStream_t s);

}  // namespace cuvs::neighbors::octex::detail
