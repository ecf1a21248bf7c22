// Launchers of the balance of rows over experts, and of its gradient (balance.hip).  Shapes, types and pointers are checked
// by the callers (operators.cpp).
#pragma once

#include "rows.hpp"

namespace cuvs::neighbors::octex::detail {

constexpr int kMaxExperts = 2048;  // 32 logits a lane

/** The weights of the balance's term and of the squared log-sum-exp's. */
struct balance_weights {
  float balance, z;
};

/** What a forward pass gives: the loss, the choices of each expert [e], the rows that count, the experts' mean probabilities
 * [e], and the rows' log-sum-exp [m]. */
struct balance_out {
  float* loss;
  int64_t *counts, *rows;
  float *probs, *lse;
};

/** The bytes of workspace (at a multiple of 256) that launch_balance needs. */
auto balance_workspace(int64_t m, int e, int k, elem type) -> int64_t;

/** in: m rows of e logits (their temperature is not read); experts: k choices a row.  grad [m, e] (in's type, rows gstride
 * apart) of grad_loss * loss, or null. */
void launch_balance(score_rows const& in, listed_ids const& experts, balance_weights const& w, balance_out const& out,
                    const float* grad_loss, void* grad, int64_t gstride, void* workspace, hipStream_t s);

/** The gradient alone, from the counts and rows that launch_balance gave. */
void launch_balance_backward(score_rows const& in, listed_ids const& experts, balance_weights const& w, const int64_t* counts,
                             const int64_t* rows, const float* grad_loss, void* grad, int64_t gstride, hipStream_t s);

}  // namespace cuvs::neighbors::octex::detail
