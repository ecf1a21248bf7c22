// Launchers of the operators on rows of scores (rows.hip): log probabilities of given ids with entropy and top
// alternatives, distillation from a teacher's top logits, and the gradients of both.  Shapes, types and pointers are
// checked by the callers (operators.cpp); a launcher splits what does not fit one grid.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace cuvs::neighbors::octex::detail {

/** Element types of the operators' arrays, as the C ABI numbers them (octexType). */
enum class elem : int { f32 = 0, f16 = 1, bf16 = 2, i8 = 3 };

inline auto elem_size(elem e) -> int { return e == elem::f32 ? 4 : e == elem::i8 ? 1 : 2; }

constexpr int kMaxTop        = 64;       // top alternatives of a row: a lane each
constexpr int kMaxListed     = 512;      // given ids, or the teacher's entries, of a row (LDS)
constexpr int64_t kMaxScores = 1 << 30;  // scores of a row: its offsets are 32-bit

/** A matrix of scores [m, n] with `stride` elements from row to row, and the scale its logits take: z = x / temperature. */
struct score_rows {
  const void* x;
  elem type;
  int64_t m, stride;
  int n;
  float temperature;
};

/** Ids [m, k] (rows `stride` apart) of a row's columns; ids outside [0, n) are padding. */
struct listed_ids {
  const void* ids;
  bool wide;  // int64, else int32
  int64_t stride;
  int k;
};

/** The outputs of a log_probs pass, each dense: logp [m, k], entropy, lse [m], top_logp, top_ids [m, top]. */
struct log_probs_out {
  float* logp;
  float* entropy;
  float* lse;
  float* top_logp;
  int64_t* top_ids;
  int top;
};

/** The teacher's logits [m, k] of the listed ids. */
struct teacher_logits {
  const void* x;
  elem type;
  int64_t stride;
};

/** The bytes of workspace (at a multiple of 256) that launch_log_probs and launch_distill need: rows that do not fill the
 * GPU are split into parts, whose sums meet there. */
auto log_probs_workspace(int64_t m, int n, int top) -> int64_t;
auto distill_workspace(int64_t m, int n) -> int64_t;

void launch_log_probs(score_rows const& in, listed_ids const& ids, log_probs_out const& out, void* workspace, hipStream_t s);

/** grad [m, n] (in's type, rows gstride apart) of sum(grad_logp * logp) + sum(grad_entropy * entropy); either may be null. */
void launch_log_probs_backward(score_rows const& in, listed_ids const& ids, const float* grad_logp,
                               const float* grad_entropy, const float* lse, const float* entropy, void* grad,
                               int64_t gstride, hipStream_t s);

void launch_distill(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, float* loss, float* lse,
                    void* workspace, hipStream_t s);

void launch_distill_backward(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher,
                             const float* grad_loss, const float* lse, void* grad, int64_t gstride, hipStream_t s);

/** Whether launch_distill_step holds a row in registers; else it needs launch_distill's workspace. */
auto distill_step_held(int64_t m, int n, elem type) -> bool;

/** Both directions; the logits are read once if a workgroup can hold a row. */
void launch_distill_step(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, const float* grad_loss,
                         float* loss, float* lse, void* grad, int64_t gstride, void* workspace, hipStream_t s);

}  // namespace cuvs::neighbors::octex::detail
