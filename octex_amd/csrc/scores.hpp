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

struct int8_rows {
  const int8_t* x;
  int64_t stride;
  const float* scales;
};

/** out [m, n] of `type`, rows ostride apart; bias [n] may be null. */
void launch_int8_scores(int8_rows const& q, int64_t m, int8_rows const& r, int64_t n, int k, const float* bias, void* out,
                        elem type, int64_t ostride, hipStream_t s);

}  // namespace cuvs::neighbors::octex::detail
