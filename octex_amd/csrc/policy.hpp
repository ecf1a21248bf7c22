// Launchers of a policy's clipped loss on rows of logits, and of its gradient (policy.hip).  Shapes, types and pointers are
// checked by the callers (operators.cpp).
#pragma once

#include "rows.hpp"

namespace cuvs::neighbors::octex::detail {

/** What a row's loss is made of beside its logits, each [m]: the log probabilities of the ids when they were sampled, their
 * advantages, and (null: no KL term) a reference model's log probabilities; the bounds of an unclipped ratio, and the terms'
 * weights. */
struct policy_terms {
  const float *sampled, *advantages, *reference;
  float low, high, kl, entropy;
};

/** What a forward pass gives of each row [m]; a row whose id is padding has 0 everywhere. */
struct policy_out {
  float *loss, *logp, *entropy, *lse;
};

/** The bytes of workspace (at a multiple of 256) that launch_policy needs. */
auto policy_workspace(int64_t m, int n) -> int64_t;

/** ids: one a row. */
void launch_policy(score_rows const& in, listed_ids const& ids, policy_terms const& terms, policy_out const& out,
                   void* workspace, hipStream_t s);

/** grad [m, n] (in's type, rows gstride apart) of sum(grad_loss * loss); saved: what launch_policy gave (loss is not read). */
void launch_policy_backward(score_rows const& in, listed_ids const& ids, policy_terms const& terms, policy_out const& saved,
                            const float* grad_loss, void* grad, int64_t gstride, hipStream_t s);

/** Whether launch_policy_step holds a row in registers (up to 256 KB of one, 128 KB of fewer than 512 rows); else it needs
 * launch_policy's workspace. */
auto policy_step_held(int64_t m, int n, elem type) -> bool;

/** Both directions; the logits are read once if a workgroup can hold a row. */
void launch_policy_step(score_rows const& in, listed_ids const& ids, policy_terms const& terms, const float* grad_loss,
                        policy_out const& out, void* grad, int64_t gstride, void* workspace, hipStream_t s);

}  // namespace cuvs::neighbors::octex::detail
