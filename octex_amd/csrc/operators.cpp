// C entries of the operators on rows of scores (octex_amd/octex_amd.h): arguments checked, the operands' GPU made current,
// the kernels launched on the caller's stream.  No call waits or allocates.

#include "balance.hpp"
#include "common.hpp"
#include "policy.hpp"
#include "rows.hpp"
#include "scores.hpp"
#include "table.hpp"

#include <cuvs/core/c_api.h>
#include <octex_amd/octex_amd.h>

#include <algorithm>
#include <cmath>
#include <exception>

namespace {

using namespace cuvs::neighbors::octex::detail;

template <typename Fn>
auto run(Fn fn) -> cuvsError_t
{
  try {
    fn();
    cuvsSetLastErrorText(nullptr);
    return CUVS_SUCCESS;
  } catch (std::exception const& e) {
    cuvsSetLastErrorText(e.what());
  } catch (...) {
    cuvsSetLastErrorText("unknown exception");
  }
  return CUVS_ERROR;
}

/** The operands of a call: all in the memory of one GPU, which is current while this lives. */
class on_gpu {
 public:
  on_gpu()                               = default;
  on_gpu(on_gpu const&)                  = delete;
  auto operator=(on_gpu const&) -> on_gpu& = delete;
  ~on_gpu()
  {
    if (changed_) (void)hipSetDevice(before_);
  }

  void take(const void* p, const char* what)
  {
    OCTEX_EXPECTS(p != nullptr, "octex: %s is NULL", what);
    hipPointerAttribute_t a{};
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
      (void)hipGetLastError();  // not memory that the runtime knows
      a.type = hipMemoryTypeHost;
    }
    OCTEX_EXPECTS(a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged,
                  "octex: %s must lie in GPU memory", what);
    if (device_ < 0) {
      device_ = a.device;
      OCTEX_HIP(hipGetDevice(&before_));
      if (before_ != device_) {
        OCTEX_HIP(hipSetDevice(device_));
        changed_ = true;
      }
    }
    OCTEX_EXPECTS(a.device == device_, "octex: %s lies on GPU %d, the other operands on GPU %d", what, a.device, device_);
  }

 private:
  int device_ = -1, before_ = -1;
  bool changed_ = false;
};

auto is_float(octexMatrix const& m) -> bool
{
  return m.type == OCTEX_FLOAT32 || m.type == OCTEX_FLOAT16 || m.type == OCTEX_BFLOAT16;
}

auto elem_of(octexMatrix const& m) -> elem { return static_cast<elem>(m.type); }

void shape(const octexMatrix* m, const char* what, int64_t rows, int64_t cols)
{
  OCTEX_EXPECTS(m != nullptr, "octex: %s is NULL", what);
  OCTEX_EXPECTS(m->rows >= 0 && m->cols >= 0 && m->stride >= m->cols, "octex: %s has a negative size or rows that overlap",
                what);
  OCTEX_EXPECTS((rows < 0 || m->rows == rows) && (cols < 0 || m->cols == cols),
                "octex: %s is [%lld, %lld], expected [%lld, %lld]", what, static_cast<long long>(m->rows),
                static_cast<long long>(m->cols), static_cast<long long>(rows < 0 ? m->rows : rows),
                static_cast<long long>(cols < 0 ? m->cols : cols));
}

void float_type(octexMatrix const& m, const char* what)
{
  OCTEX_EXPECTS(is_float(m), "octex: %s must be float32, float16 or bfloat16", what);
}

auto logits_of(const octexMatrix* x, float temperature) -> score_rows
{
  shape(x, "logits", -1, -1);
  float_type(*x, "logits");
  OCTEX_EXPECTS(x->cols >= 1 && x->cols <= kMaxScores, "octex: logits have 1 to 2^30 columns, not %lld",
                static_cast<long long>(x->cols));
  OCTEX_EXPECTS(temperature >= 1e-30f && temperature <= 1e30f, "octex: the temperature must be positive (1e-30 to 1e30)");
  return {x->data, elem_of(*x), x->rows, x->stride, static_cast<int>(x->cols), temperature};
}

auto ids_of(const octexMatrix* ids, int64_t m) -> listed_ids
{
  shape(ids, "ids", m, -1);
  OCTEX_EXPECTS(ids->type == OCTEX_INT32 || ids->type == OCTEX_INT64, "octex: ids must be int32 or int64");
  OCTEX_EXPECTS(ids->cols <= kMaxListed, "octex: at most %d ids a row, not %lld", kMaxListed,
                static_cast<long long>(ids->cols));
  return {ids->data, ids->type == OCTEX_INT64, ids->stride, static_cast<int>(ids->cols)};
}

auto teacher_of(const octexMatrix* t, listed_ids const& ids, int64_t m) -> teacher_logits
{
  shape(t, "teacher", m, ids.k);
  float_type(*t, "teacher");
  return {t->data, elem_of(*t), t->stride};
}

void grad_of(const octexMatrix* grad, const octexMatrix* logits)
{
  shape(grad, "grad", logits->rows, logits->cols);
  OCTEX_EXPECTS(grad->type == logits->type, "octex: grad must have the type of the logits");
}

/** Answers a question for the workspace's size; else checks what was given. */
auto asked_size(int64_t need, int64_t bytes, int64_t* size) -> bool
{
  if (size != nullptr) {
    *size = need;
    return true;
  }
  OCTEX_EXPECTS(bytes >= need, "octex: the workspace has %lld bytes, %lld are needed", static_cast<long long>(bytes),
                static_cast<long long>(need));
  return false;
}

void take_workspace(on_gpu& gpu, const void* workspace, int64_t need)
{
  if (need == 0) return;
  gpu.take(workspace, "workspace");
  OCTEX_EXPECTS(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "octex: the workspace must lie at a multiple of 256 bytes");
}

}  // namespace

extern "C" cuvsError_t octexQuantizeRows(const octexMatrix* x, const octexMatrix* codes, float* scales, void* stream)
{
  return run([&] {
    shape(x, "x", -1, -1);
    float_type(*x, "x");
    OCTEX_EXPECTS(x->cols >= 1 && x->cols <= kMaxInt8Width, "octex: rows of 1 to %d values, not %lld", kMaxInt8Width,
                  static_cast<long long>(x->cols));
    shape(codes, "codes", x->rows, x->cols);
    OCTEX_EXPECTS(codes->type == OCTEX_INT8, "octex: codes must be int8");
    if (x->rows == 0) return;
    on_gpu gpu;
    gpu.take(x->data, "x"), gpu.take(codes->data, "codes"), gpu.take(scales, "scales");
    launch_quantize_rows(x->data, elem_of(*x), x->rows, static_cast<int>(x->cols), x->stride,
                         static_cast<int8_t*>(codes->data), codes->stride, scales, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexInt8Scores(const octexMatrix* queries, const float* query_scales, const octexMatrix* rows,
                                       const float* row_scales, const float* bias, const octexMatrix* out, void* workspace,
                                       int64_t bytes, int64_t* size, void* stream)
{
  return run([&] {
    shape(queries, "queries", -1, -1);
    const bool coded = queries->type == OCTEX_INT8;
    OCTEX_EXPECTS(coded || is_float(*queries), "octex: queries must be int8, float32, float16 or bfloat16");
    OCTEX_EXPECTS(coded || query_scales == nullptr, "octex: only int8 queries have query_scales");
    const int64_t m = queries->rows, k = queries->cols;
    OCTEX_EXPECTS(k >= 1 && k <= kMaxInt8Width, "octex: rows of 1 to %d values, not %lld", kMaxInt8Width,
                  static_cast<long long>(k));
    shape(rows, "rows", -1, k);
    OCTEX_EXPECTS(rows->type == OCTEX_INT8, "octex: rows must be int8");
    const int64_t n = rows->rows;
    shape(out, "out", m, n);
    float_type(*out, "out");
    const int8_query q{queries->data, elem_of(*queries), queries->stride, query_scales};
    const int8_rows r{static_cast<const int8_t*>(rows->data), rows->stride, row_scales};
    const int64_t need = m == 0 || n == 0 ? 0 : int8_scores_workspace(q, m, r, n, static_cast<int>(k));
    if (asked_size(need, bytes, size)) return;
    if (m == 0 || n == 0) return;
    on_gpu gpu;
    gpu.take(queries->data, "queries"), gpu.take(rows->data, "rows"), gpu.take(row_scales, "row_scales");
    gpu.take(out->data, "out");
    if (coded) gpu.take(query_scales, "query_scales");
    if (bias != nullptr) gpu.take(bias, "bias");
    take_workspace(gpu, workspace, need);
    launch_int8_scores(q, m, r, n, static_cast<int>(k), bias, out->data, elem_of(*out), out->stride, workspace,
                       static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexLogProbs(const octexMatrix* logits, const octexMatrix* ids, float temperature, int32_t top,
                                     float* log_probs, float* entropy, float* lse, float* top_log_probs, int64_t* top_ids,
                                     void* workspace, int64_t bytes, int64_t* size, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = ids_of(ids, in.m);
    OCTEX_EXPECTS(top >= 0 && top <= kMaxTop, "octex: 0 to %d top entries, not %d", kMaxTop, top);
    const int64_t need = in.m == 0 ? 0 : log_probs_workspace(in.m, in.n, top);
    if (asked_size(need, bytes, size)) return;
    if (in.m == 0) return;
    on_gpu gpu;
    take_workspace(gpu, workspace, need);
    gpu.take(in.x, "logits"), gpu.take(entropy, "entropy"), gpu.take(lse, "lse");
    if (id.k > 0) gpu.take(id.ids, "ids"), gpu.take(log_probs, "log_probs");
    if (top > 0) gpu.take(top_log_probs, "top_log_probs"), gpu.take(top_ids, "top_ids");
    launch_log_probs(in, id, {log_probs, entropy, lse, top_log_probs, top_ids, top}, workspace,
                     static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexLogProbsBackward(const octexMatrix* logits, const octexMatrix* ids, float temperature,
                                             const float* grad_log_probs, const float* grad_entropy, const float* lse,
                                             const float* entropy, const octexMatrix* grad, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = ids_of(ids, in.m);
    grad_of(grad, logits);
    if (in.m == 0) return;
    on_gpu gpu;
    gpu.take(in.x, "logits"), gpu.take(lse, "lse"), gpu.take(grad->data, "grad");
    if (id.k > 0) gpu.take(id.ids, "ids");
    if (grad_log_probs != nullptr && id.k > 0) gpu.take(grad_log_probs, "grad_log_probs");
    if (grad_entropy != nullptr) gpu.take(grad_entropy, "grad_entropy"), gpu.take(entropy, "entropy");
    launch_log_probs_backward(in, id, grad_log_probs, grad_entropy, lse, entropy, grad->data, grad->stride,
                              static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexDistill(const octexMatrix* logits, const octexMatrix* ids, const octexMatrix* teacher,
                                    float temperature, float* loss, float* lse, void* workspace, int64_t bytes,
                                    int64_t* size, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = ids_of(ids, in.m);
    const auto t  = teacher_of(teacher, id, in.m);
    const int64_t need = in.m == 0 ? 0 : distill_workspace(in.m, in.n);
    if (asked_size(need, bytes, size)) return;
    if (in.m == 0) return;
    on_gpu gpu;
    take_workspace(gpu, workspace, need);
    gpu.take(in.x, "logits"), gpu.take(loss, "loss"), gpu.take(lse, "lse");
    if (id.k > 0) gpu.take(id.ids, "ids"), gpu.take(t.x, "teacher");
    launch_distill(in, id, t, loss, lse, workspace, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexDistillBackward(const octexMatrix* logits, const octexMatrix* ids, const octexMatrix* teacher,
                                            float temperature, const float* grad_loss, const float* lse,
                                            const octexMatrix* grad, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = ids_of(ids, in.m);
    const auto t  = teacher_of(teacher, id, in.m);
    grad_of(grad, logits);
    if (in.m == 0) return;
    on_gpu gpu;
    gpu.take(in.x, "logits"), gpu.take(grad_loss, "grad_loss"), gpu.take(lse, "lse"), gpu.take(grad->data, "grad");
    if (id.k > 0) gpu.take(id.ids, "ids"), gpu.take(t.x, "teacher");
    launch_distill_backward(in, id, t, grad_loss, lse, grad->data, grad->stride, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexDistillStep(const octexMatrix* logits, const octexMatrix* ids, const octexMatrix* teacher,
                                        float temperature, const float* grad_loss, float* loss, float* lse,
                                        const octexMatrix* grad, void* workspace, int64_t bytes, int64_t* size, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = ids_of(ids, in.m);
    const auto t  = teacher_of(teacher, id, in.m);
    grad_of(grad, logits);
    const int64_t need = in.m == 0 || distill_step_held(in.m, in.n, in.type) ? 0 : distill_workspace(in.m, in.n);
    if (asked_size(need, bytes, size)) return;
    if (in.m == 0) return;
    on_gpu gpu;
    take_workspace(gpu, workspace, need);
    gpu.take(in.x, "logits"), gpu.take(grad_loss, "grad_loss"), gpu.take(loss, "loss"), gpu.take(lse, "lse");
    gpu.take(grad->data, "grad");
    if (id.k > 0) gpu.take(id.ids, "ids"), gpu.take(t.x, "teacher");
    launch_distill_step(in, id, t, grad_loss, loss, lse, grad->data, grad->stride, workspace,
                        static_cast<hipStream_t>(stream));
  });
}

namespace {

/** The ids of a policy's rows: one a row. */
auto row_ids_of(const octexMatrix* ids, int64_t m) -> listed_ids
{
  shape(ids, "ids", m, 1);
  return ids_of(ids, m);
}

auto terms_of(const float* sampled, const float* advantages, const float* reference, float low, float high, float kl,
              float entropy) -> policy_terms
{
  OCTEX_EXPECTS(low >= 0.f && low <= 1.f && high >= 1.f, "octex: a ratio is clipped to bounds from 0 to 1 and from 1 on");
  OCTEX_EXPECTS(std::isfinite(kl) && std::isfinite(entropy), "octex: the weights of the KL and entropy terms must be finite");
  OCTEX_EXPECTS(kl == 0.f || reference != nullptr, "octex: the KL term needs ref_log_probs");
  return {sampled, advantages, kl != 0.f ? reference : nullptr, low, high, kl, entropy};
}

void take_terms(on_gpu& gpu, score_rows const& in, listed_ids const& ids, policy_terms const& t)
{
  gpu.take(in.x, "logits"), gpu.take(ids.ids, "ids"), gpu.take(t.sampled, "old_log_probs");
  gpu.take(t.advantages, "advantages");
  if (t.reference != nullptr) gpu.take(t.reference, "ref_log_probs");
}

void take_results(on_gpu& gpu, policy_out const& out)
{
  gpu.take(out.loss, "loss"), gpu.take(out.logp, "log_probs"), gpu.take(out.entropy, "entropy"), gpu.take(out.lse, "lse");
}

/** Logits over experts and the rows' choices of them. */
auto experts_of(const octexMatrix* logits, const octexMatrix* experts, score_rows& in) -> listed_ids
{
  in = logits_of(logits, 1.f);
  OCTEX_EXPECTS(in.n <= kMaxExperts, "octex: at most %d experts, not %d", kMaxExperts, in.n);
  shape(experts, "experts", in.m, -1);
  OCTEX_EXPECTS(experts->type == OCTEX_INT32 || experts->type == OCTEX_INT64, "octex: experts must be int32 or int64");
  OCTEX_EXPECTS(experts->cols <= kMaxListed, "octex: at most %d experts a row, not %lld", kMaxListed,
                static_cast<long long>(experts->cols));
  OCTEX_EXPECTS(in.m <= INT32_MAX / std::max<int64_t>(experts->cols, 1), "octex: at most 2^31 - 1 choices");
  return {experts->data, experts->type == OCTEX_INT64, experts->stride, static_cast<int>(experts->cols)};
}

auto weights_of(float balance, float z) -> balance_weights
{
  OCTEX_EXPECTS(std::isfinite(balance) && std::isfinite(z), "octex: the balance's weights must be finite");
  return {balance, z};
}

auto table_ids(const octexMatrix* ids, int64_t m) -> row_ids
{
  shape(ids, "ids", m, 1);
  OCTEX_EXPECTS(ids->type == OCTEX_INT32 || ids->type == OCTEX_INT64, "octex: ids must be int32 or int64");
  return {ids->data, ids->type == OCTEX_INT64, ids->stride, ids->rows};
}

void table_size(int64_t m, int64_t n, int64_t d)
{
  OCTEX_EXPECTS(m <= INT32_MAX && n <= INT32_MAX, "octex: at most 2^31 - 1 ids and rows");
  OCTEX_EXPECTS(d <= kMaxRowWidth, "octex: rows of at most %lld values, not %lld", static_cast<long long>(kMaxRowWidth),
                static_cast<long long>(d));
}

}  // namespace

extern "C" cuvsError_t octexPolicyLoss(const octexMatrix* logits, const octexMatrix* ids, float temperature,
                                       const float* old_log_probs, const float* advantages, const float* ref_log_probs,
                                       float low, float high, float kl, float entropy_weight, float* loss, float* log_probs,
                                       float* entropy, float* lse, void* workspace, int64_t bytes, int64_t* size, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = row_ids_of(ids, in.m);
    const auto t  = terms_of(old_log_probs, advantages, ref_log_probs, low, high, kl, entropy_weight);
    const int64_t need = in.m == 0 ? 0 : policy_workspace(in.m, in.n);
    if (asked_size(need, bytes, size)) return;
    if (in.m == 0) return;
    const policy_out out{loss, log_probs, entropy, lse};
    on_gpu gpu;
    take_workspace(gpu, workspace, need);
    take_terms(gpu, in, id, t), take_results(gpu, out);
    launch_policy(in, id, t, out, workspace, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexPolicyLossBackward(const octexMatrix* logits, const octexMatrix* ids, float temperature,
                                               const float* old_log_probs, const float* advantages,
                                               const float* ref_log_probs, float low, float high, float kl,
                                               float entropy_weight, const float* grad_loss, const float* log_probs,
                                               const float* entropy, const float* lse, const octexMatrix* grad, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = row_ids_of(ids, in.m);
    const auto t  = terms_of(old_log_probs, advantages, ref_log_probs, low, high, kl, entropy_weight);
    grad_of(grad, logits);
    if (in.m == 0) return;
    on_gpu gpu;
    take_terms(gpu, in, id, t);
    gpu.take(grad_loss, "grad_loss"), gpu.take(log_probs, "log_probs"), gpu.take(entropy, "entropy"), gpu.take(lse, "lse");
    gpu.take(grad->data, "grad");
    // what a forward pass gave is read only
    const policy_out saved{nullptr, const_cast<float*>(log_probs), const_cast<float*>(entropy), const_cast<float*>(lse)};
    launch_policy_backward(in, id, t, saved, grad_loss, grad->data, grad->stride, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexPolicyLossStep(const octexMatrix* logits, const octexMatrix* ids, float temperature,
                                           const float* old_log_probs, const float* advantages, const float* ref_log_probs,
                                           float low, float high, float kl, float entropy_weight, const float* grad_loss,
                                           float* loss, float* log_probs, float* entropy, float* lse, const octexMatrix* grad,
                                           void* workspace, int64_t bytes, int64_t* size, void* stream)
{
  return run([&] {
    const auto in = logits_of(logits, temperature);
    const auto id = row_ids_of(ids, in.m);
    const auto t  = terms_of(old_log_probs, advantages, ref_log_probs, low, high, kl, entropy_weight);
    grad_of(grad, logits);
    const int64_t need = in.m == 0 || policy_step_held(in.m, in.n, in.type) ? 0 : policy_workspace(in.m, in.n);
    if (asked_size(need, bytes, size)) return;
    if (in.m == 0) return;
    const policy_out out{loss, log_probs, entropy, lse};
    on_gpu gpu;
    take_workspace(gpu, workspace, need);
    take_terms(gpu, in, id, t), take_results(gpu, out);
    gpu.take(grad_loss, "grad_loss"), gpu.take(grad->data, "grad");
    launch_policy_step(in, id, t, grad_loss, out, grad->data, grad->stride, workspace, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexBalanceLoss(const octexMatrix* logits, const octexMatrix* experts, float weight, float z_weight,
                                        float* loss, int64_t* counts, int64_t* rows, float* probs, float* lse,
                                        const float* grad_loss, const octexMatrix* grad, void* workspace, int64_t bytes,
                                        int64_t* size, void* stream)
{
  return run([&] {
    score_rows in{};
    const auto id = experts_of(logits, experts, in);
    const auto w  = weights_of(weight, z_weight);
    if (grad != nullptr) grad_of(grad, logits);
    const int64_t need = balance_workspace(in.m, in.n, id.k, in.type);
    if (asked_size(need, bytes, size)) return;
    on_gpu gpu;
    gpu.take(loss, "loss"), gpu.take(counts, "counts"), gpu.take(rows, "rows"), gpu.take(probs, "probs");
    take_workspace(gpu, workspace, need);
    if (in.m > 0) {
      gpu.take(in.x, "logits"), gpu.take(lse, "lse");
      if (id.k > 0) gpu.take(id.ids, "experts");
      if (grad != nullptr) gpu.take(grad->data, "grad");
    }
    if (grad_loss != nullptr) gpu.take(grad_loss, "grad_loss");
    launch_balance(in, id, w, {loss, counts, rows, probs, lse}, grad_loss, grad != nullptr ? grad->data : nullptr,
                   grad != nullptr ? grad->stride : 0, workspace, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexBalanceLossBackward(const octexMatrix* logits, const octexMatrix* experts, float weight,
                                                float z_weight, const int64_t* counts, const int64_t* rows,
                                                const float* grad_loss, const octexMatrix* grad, void* stream)
{
  return run([&] {
    score_rows in{};
    const auto id = experts_of(logits, experts, in);
    const auto w  = weights_of(weight, z_weight);
    grad_of(grad, logits);
    if (in.m == 0) return;
    on_gpu gpu;
    gpu.take(in.x, "logits"), gpu.take(counts, "counts"), gpu.take(rows, "rows"), gpu.take(grad->data, "grad");
    if (id.k > 0) gpu.take(id.ids, "experts");
    if (grad_loss != nullptr) gpu.take(grad_loss, "grad_loss");
    launch_balance_backward(in, id, w, counts, rows, grad_loss, grad->data, grad->stride, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexEmbed(const octexMatrix* table, const float* row_scales, const octexMatrix* ids, float scale,
                                  const octexMatrix* out, void* stream)
{
  return run([&] {
    shape(table, "table", -1, -1);
    const bool coded = table->type == OCTEX_INT8;
    OCTEX_EXPECTS(coded || is_float(*table), "octex: the table must be int8, float32, float16 or bfloat16");
    OCTEX_EXPECTS(coded || row_scales == nullptr, "octex: only int8 rows have row_scales");
    const auto id = table_ids(ids, -1);
    shape(out, "out", id.m, table->cols);
    float_type(*out, "out");
    table_size(id.m, table->rows, table->cols);
    if (id.m == 0 || table->cols == 0) return;
    on_gpu gpu;
    gpu.take(id.ids, "ids"), gpu.take(out->data, "out");
    if (table->rows > 0) {
      gpu.take(table->data, "table");
      if (coded) gpu.take(row_scales, "row_scales");
    }
    launch_embed({table->data, elem_of(*table), table->rows, table->stride, row_scales}, id, table->cols, scale,
                 {out->data, elem_of(*out), out->stride}, static_cast<hipStream_t>(stream));
  });
}

extern "C" cuvsError_t octexEmbedBackward(const octexMatrix* grad, const octexMatrix* ids, float scale, int32_t add,
                                          const octexMatrix* out, void* workspace, int64_t bytes, int64_t* size, void* stream)
{
  return run([&] {
    shape(grad, "grad", -1, -1);
    float_type(*grad, "grad");
    const auto id = table_ids(ids, grad->rows);
    shape(out, "out", -1, grad->cols);
    float_type(*out, "out");
    const int64_t n = out->rows, d = grad->cols;
    table_size(id.m, n, d);
    const bool none    = n == 0 || d == 0 || (add != 0 && id.m == 0);
    const int64_t need = none ? 0 : embed_backward_workspace(id.m, n, d);
    if (asked_size(need, bytes, size)) return;
    if (none) return;
    on_gpu gpu;
    gpu.take(out->data, "out");
    take_workspace(gpu, workspace, need);
    if (id.m > 0) gpu.take(grad->data, "grad"), gpu.take(id.ids, "ids");
    launch_embed_backward({grad->data, elem_of(*grad), grad->stride}, id, n, d, scale, add != 0,
                          {out->data, elem_of(*out), out->stride}, workspace, static_cast<hipStream_t>(stream));
  });
}
