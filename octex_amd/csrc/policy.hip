// A policy's clipped loss on rows of logits x, read as z = x / T: row i's id a was sampled when its log probability was `old`
// and earned the advantage A.
//
//   lp   = z_a - ln sum exp z;  r = exp(lp - old);  pg = -min(r A, clip(r, low, high) A)
//   k    = exp(d) - 1 - d,  d = reference's log probability - lp      (an estimate of the KL divergence that is never below 0)
//   loss = pg + kl k - entropy H,  H = -sum p ln p
//   dx_v = g / T (c (1[v = a] - p_v) + entropy p_v (ln p_v + H)),  c = (-r A, or 0 where clipped) + kl (1 - exp(d))
//
// A row's sums are those of log_probs (rows_device.hpp), and its gradient p (a + b ln p) with one share w at the id:
// a = g / T (entropy H - c), b = g / T entropy, w = g / T c.  A row whose id is padding (a prompt's token) is not read.
//
// Bound by the logits' bytes: a large copy takes 5.06 TB/s of this GPU.  Both directions of 4096 x 128,000 bfloat16 take 456 us,
// 4.6 TB/s; 333 x 50,021 float16 11 and 13; 16 x 32,000 float32 10, where a row is one CU's and its exponentials bound it.  Rows
// that no workgroup holds are read twice, by a kernel a direction: 4096 x 150,000 bfloat16 756 us, 2048 x 128,000 float32 592.

#include "policy.hpp"
#include "rows_device.hpp"

namespace cuvs::neighbors::octex::detail {

namespace {

/** What a row's loss takes beside its logits; id -1: padding. */
struct policy_row {
  int id;
  float sampled, advantage, reference, grad_loss;
};

__device__ inline auto row_of(score_rows const& in, listed_ids const& ids, policy_terms const& t, const float* grad_loss,
                              int64_t r) -> policy_row
{
  const int64_t id = id_at(ids, r, 0);
  return {id >= 0 && id < in.n ? static_cast<int>(id) : -1, t.sampled[r], t.advantages[r],
          t.reference != nullptr ? t.reference[r] : 0.f, grad_loss != nullptr ? grad_loss[r] : 0.f};
}

/** exp(d) - 1 - d, given e = exp(d) - 1.  Near 0 that difference would keep few of its digits (1e-4 of it lost at d = 1e-3) or
 * fall below 0; there it is d^2 (1/2 + d/6 + d^2/24 ...), whose next term is 2^-28 of it at |d| = 1/2. */
__device__ inline auto kl_of(float d, float e) -> float
{
  if (!(fabsf(d) < 0.5f)) return e == INFINITY ? e : e - d;
  float s = 1.f / 362880.f;
  s       = fmaf(s, d, 1.f / 40320.f);
  s       = fmaf(s, d, 1.f / 5040.f);
  s       = fmaf(s, d, 1.f / 720.f);
  s       = fmaf(s, d, 1.f / 120.f);
  s       = fmaf(s, d, 1.f / 24.f);
  s       = fmaf(s, d, 1.f / 6.f);
  s       = fmaf(s, d, 0.5f);
  return d * d * s;
}

/** A row's loss but for the entropy's term, and its slope by the log probability. */
struct policy_loss {
  float loss, slope;
};

/** At a bound itself the ratio counts as unclipped. */
__device__ inline auto loss_of(float logp, policy_row const& p, policy_terms const& t) -> policy_loss
{
  const float r = expf(logp - p.sampled), bound = p.advantage < 0.f ? t.low : t.high;
  const bool clipped = p.advantage < 0.f ? r < bound : p.advantage >= 0.f && r > bound;
  policy_loss l{-p.advantage * (clipped ? bound : r), clipped ? 0.f : -p.advantage * r};
  if (t.reference != nullptr) {
    const float d = p.reference - logp, e = expm1f(d);
    l.loss += t.kl * kl_of(d, e);
    l.slope -= t.kl * e;
  }
  return l;
}

__device__ inline void write_row(policy_out const& out, int64_t r, float loss, float logp, float entropy, float lse)
{
  out.loss[r]    = loss;
  out.logp[r]    = logp;
  out.entropy[r] = entropy;
  out.lse[r]     = lse;
}

__device__ inline void write_row(policy_out const& out, int64_t r, policy_loss const& l, float logp, row_sums const& o,
                                 policy_terms const& t)
{
  write_row(out, r, t.entropy != 0.f ? l.loss - t.entropy * o.entropy : l.loss, logp, o.entropy, o.lse);
}

/** A workgroup a row, or with kSplit a workgroup a part of a row, which leaves its sums to finish_policy_kernel. */
template <typename T, int NT, bool kSplit>
__global__ __launch_bounds__(NT) void policy_kernel(score_rows in, listed_ids ids, policy_terms terms, policy_out out,
                                                    row_split split, part_sums* part, int64_t row0)
{
  __shared__ run parts[NT / 64];
  const int64_t b = row0 + blockIdx.x, r = kSplit ? b / split.parts : b;
  const int c0    = kSplit ? static_cast<int>(b - r * split.parts) * split.width : 0;
  const int c1    = kSplit ? min(c0 + split.width, in.n) : in.n;
  const T* row    = static_cast<const T*>(in.x) + r * in.stride;
  const float c   = kLog2e / in.temperature;
  const auto mine = row_of(in, ids, terms, nullptr, r);
  if (mine.id < 0) {
    if (!kSplit && threadIdx.x == 0) write_row(out, r, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  auto added = nothing_long();
  for_scores<T, NT>(row, c0, c1, [](float) {}, [&](const auto& v, int) { add_scores<true>(added, v, c); },
                    [&] { added.fold<true>(c); });
  const run sums = join_block<NT, true>(added.whole(), c, parts);
  if (threadIdx.x != 0) return;
  if constexpr (kSplit) {
    part[b] = {sums.m, sums.s, sums.t};
  } else {
    const auto o     = finish(sums, in.temperature);
    const float logp = log_prob(static_cast<float>(row[mine.id]), o, in.temperature);
    write_row(out, r, loss_of(logp, mine, terms), logp, o, terms);
  }
}

template <typename T>
__global__ __launch_bounds__(64) void finish_policy_kernel(score_rows in, listed_ids ids, policy_terms terms, policy_out out,
                                                           row_split split, const part_sums* part, int64_t row0)
{
  const int64_t r = row0 + blockIdx.x;
  const auto mine = row_of(in, ids, terms, nullptr, r);
  if (mine.id < 0) {
    if (threadIdx.x == 0) write_row(out, r, 0.f, 0.f, 0.f, 0.f);
    return;
  }
  const auto o     = finish(join_parts<true>(part, r, split.parts, kLog2e / in.temperature), in.temperature);
  const float logp = log_prob(static_cast<float>(static_cast<const T*>(in.x)[r * in.stride + mine.id]), o, in.temperature);
  if (threadIdx.x == 0) write_row(out, r, loss_of(logp, mine, terms), logp, o, terms);
}

/** A row's gradient: p (a + b ln p), and w more at the id. */
struct policy_slopes {
  float a, b, w;
};

__device__ inline auto slopes_of(policy_loss const& l, float entropy, policy_row const& p, policy_terms const& t,
                                 float temperature) -> policy_slopes
{
  const float g = p.grad_loss / temperature;
  return {g * (t.entropy != 0.f ? t.entropy * entropy - l.slope : -l.slope), g * t.entropy, g * l.slope};
}

template <typename T, int NT>
__device__ inline void write_zeros(T* grad, int c0, int c1)
{
  constexpr int N = kPer16<T>;
  if (c1 - c0 < N) {
    if (c0 + static_cast<int>(threadIdx.x) < c1) grad[c0 + threadIdx.x] = static_cast<T>(0.f);
    return;
  }
  for (int at = c0 + static_cast<int>(threadIdx.x) * N; at < c1; at += NT * N)
    store16(grad + min(at, c1 - N), uint4{0, 0, 0, 0});
}

/** A workgroup a row or a part of one. */
template <typename T, int NT>
__global__ __launch_bounds__(NT) void policy_backward_kernel(score_rows in, listed_ids ids, policy_terms terms,
                                                             policy_out saved, const float* grad_loss, T* grad,
                                                             int64_t gstride, bool by_cache, row_split split, int64_t row0)
{
  __shared__ listed_shares shares;
  __shared__ run parts[NT / 64];
  const int64_t b = row0 + blockIdx.x, r = b / split.parts;
  const int c0 = static_cast<int>(b - r * split.parts) * split.width, c1 = min(c0 + split.width, in.n);
  const T* row    = static_cast<const T*>(in.x) + r * in.stride;
  const auto mine = row_of(in, ids, terms, grad_loss, r);
  if (mine.id < 0) return write_zeros<T, NT>(grad + r * gstride, c0, c1);
  write_gradient<T, true, NT>(row, grad + r * gstride, by_cache, c0, c1, shares, 1, [&](bool&) {
    const auto s = slopes_of(loss_of(saved.logp[r], mine, terms), saved.entropy[r], mine, terms, in.temperature);
    if (threadIdx.x == 0) shares.id[0] = mine.id, shares.w[0] = s.w;
    lds_barrier();
    auto g = gradient_base<T, NT>(row, in.n, saved.lse[r], in.temperature, parts);
    g.a    = s.a;
    g.b    = s.b;
    return g;
  });
}

/**
 * Both directions of rows that a workgroup holds in registers, H pieces of 16 bytes a thread: each is read once and its
 * gradient written once.  A workgroup takes every gridDim-th row; as a piece of a row's gradient is stored, the same piece
 * of its next row is loaded in its place, and pieces that have arrived enter that row's sums.  What a row has beside its
 * logits comes a row ahead.
 */
template <typename T, int NT, int H>
__global__ __launch_bounds__(NT) void policy_step_kernel(score_rows in, listed_ids ids, policy_terms terms,
                                                         const float* grad_loss, policy_out out, T* grad, int64_t gstride,
                                                         bool by_cache)
{
  constexpr int N = kPer16<T>, kStep = NT * N, kLag = 4;  // pieces on their way
  __shared__ run parts[2][NT / 64];  // in turn: a row's are read until the next row's barrier
  const int last = in.n - N, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64 * N;
  int mine       = static_cast<int>(threadIdx.x) * N;
  const float c  = kLog2e / in.temperature;
  uint4 held[H];
  run sums = nothing();
  float v[N];
  const auto row_at = [&](int64_t r) { return static_cast<const T*>(in.x) + r * in.stride; };
  const auto load   = [&](int64_t r, int h) { held[h] = load16(row_at(r) + min(h * kStep + mine, last)); };
  const auto add    = [&](int h) {
    unpack16<T>(held[h], v);
    if (h * kStep + kStep > in.n) {  // columns that another thread holds
      const int at = h * kStep + mine, from = min(at, last);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (from + i < at) v[i] = -INFINITY;
    }
    add_scores<true>(sums, v, c);
  };
  policy_row row   = row_of(in, ids, terms, grad_loss, blockIdx.x);
  policy_row after = blockIdx.x + int64_t{gridDim.x} < in.m ? row_of(in, ids, terms, grad_loss, blockIdx.x + int64_t{gridDim.x})
                                                            : policy_row{-1, 0.f, 0.f, 0.f, 0.f};
  float x_id = 0.f, x_after = 0.f;
  if (row.id >= 0) {
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (h * kStep < in.n) load(blockIdx.x, h);
    x_id = static_cast<float>(row_at(blockIdx.x)[row.id]);
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (h * kStep < in.n) add(h);
  }
  int turn = 0;
  for (int64_t r = blockIdx.x; r < in.m; r += gridDim.x) {
    asm volatile("" : "+v"(mine));  // the pieces' places are made again for every row: kept, they would take H registers
    const int64_t next = r + gridDim.x, third = next + gridDim.x;
    const bool more    = after.id >= 0;
    const auto later   = third < in.m ? row_of(in, ids, terms, grad_loss, third) : policy_row{-1, 0.f, 0.f, 0.f, 0.f};
    gradient_row g{0.f, c, INFINITY, 0.f, 0.f};
    float w = 0.f;
    if (row.id >= 0) {
      sums             = join_block<NT, true>(sums, c, parts[turn]);
      const auto o     = finish(sums, in.temperature);
      const float logp = log_prob(x_id, o, in.temperature);
      const auto l     = loss_of(logp, row, terms);
      if (threadIdx.x == 0) write_row(out, r, l, logp, o, terms);
      const auto slopes = slopes_of(l, o.entropy, row, terms, in.temperature);
      g = {sums.ref, c, sums.s > 0.f ? log2f(sums.s) : sums.s == 0.f ? INFINITY : sums.s, slopes.a, slopes.b};
      w = slopes.w;
      turn ^= 1;
    } else if (threadIdx.x == 0) {
      write_row(out, r, 0.f, 0.f, 0.f, 0.f);
    }
    T* to = grad + r * gstride;
    sums  = nothing();
#pragma unroll
    for (int h = 0; h < H + kLag; ++h) {
      if (h < H && h * kStep < in.n) {
        const int at = min(h * kStep + mine, last), w0 = h * kStep + wave;
        if (row.id >= 0) {
          unpack16<T>(held[h], v);
#pragma unroll
          for (int i = 0; i < N; ++i)
            v[i] = gradient<true>(v[i], g);
          if (row.id >= min(w0, last) && row.id < w0 + 64 * N) {  // a lane of this wavefront has it
#pragma unroll
            for (int i = 0; i < N; ++i)
              v[i] += row.id - at == i ? w : 0.f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i)
            v[i] = 0.f;
        }
        if (h * kStep + mine < in.n) {
          if (by_cache)
            store16(to + at, pack16<T>(v));
          else
            store16_nt(to + at, pack16<T>(v));
        }
        if (more) load(next, h);
      }
      if (h == H / 2 && more) x_after = static_cast<float>(row_at(next)[after.id]);
      if (more && h >= kLag && (h - kLag) * kStep < in.n) add(h - kLag);
    }
    row   = after;
    after = later;
    x_id  = x_after;
  }
}

}  // namespace

auto policy_workspace(int64_t m, int n) -> int64_t
{
  const auto split = forward_split_of(m, n, 0);
  return split.parts == 1 ? 0 : m * split.parts * static_cast<int64_t>(sizeof(part_sums));
}

void launch_policy(score_rows const& in, listed_ids const& ids, policy_terms const& terms, policy_out const& out,
                   void* workspace, hipStream_t s)
{
  const auto split = forward_split_of(in.m, in.n, 0);
  auto* part       = static_cast<part_sums*>(workspace);
  with_type(in.type, [&](auto e) {
    using T           = decltype(e);
    const auto launch = [&](auto kernel, int threads, int64_t total) {
      for_grids(total, threads, [&](int64_t first, unsigned count) {
        kernel<<<count, threads, 0, s>>>(in, ids, terms, out, split, part, first);
        OCTEX_HIP(hipGetLastError());
      });
    };
    // by a wavefront a row, by 256 threads: 8192 x 1000 float32 11.5 us, 15.5; 8192 x 4000 bfloat16 18.4, 21.5; of 1500 rows 8.2,
    // 7.8.  512 or 1024 threads gain nothing: 333 x 50,021 float16 14.6, 15.1, 15.0, of 250 rows 11.3, 10.6, 11.1
    if (split.parts > 1) {
      launch(policy_kernel<T, kThreads, true>, kThreads, in.m * split.parts);
      launch(finish_policy_kernel<T>, 64, in.m);
    } else if (by_wavefront(in.m, in.n, 1)) {
      launch(policy_kernel<T, 64, false>, 64, in.m);
    } else {
      launch(policy_kernel<T, kThreads, false>, kThreads, in.m);
    }
  });
}

void launch_policy_backward(score_rows const& in, listed_ids const& ids, policy_terms const& terms, policy_out const& saved,
                            const float* grad_loss, void* grad, int64_t gstride, hipStream_t s)
{
  const auto split = split_of(in.m, in.n);
  with_type(in.type, [&](auto e) {
    using T           = decltype(e);
    const auto launch = [&](auto kernel, int threads) {
      for_grids(in.m * split.parts, threads, [&](int64_t first, unsigned count) {
        kernel<<<count, threads, 0, s>>>(in, ids, terms, saved, grad_loss, static_cast<T*>(grad), gstride, passes_cache(in),
                                         split, first);
        OCTEX_HIP(hipGetLastError());
      });
    };
    // 2048 x 1000 float32 7.1 us, by 256 threads 8.5; 8192 x 4000 bfloat16 27.7, 28.1; of 1500 rows 10.3, 9.6
    if (by_wavefront(in.m, in.n, 1))
      launch(policy_backward_kernel<T, 64>, 64);
    else
      launch(policy_backward_kernel<T, kThreads>, kThreads);
  });
}

auto policy_step_held(int64_t m, int n, elem type) -> bool { return distill_step_held(m, n, type); }

void launch_policy_step(score_rows const& in, listed_ids const& ids, policy_terms const& terms, const float* grad_loss,
                        policy_out const& out, void* grad, int64_t gstride, void* workspace, hipStream_t s)
{
  if (!policy_step_held(in.m, in.n, in.type)) {
    launch_policy(in, ids, terms, out, workspace, s);
    launch_policy_backward(in, ids, terms, out, grad_loss, grad, gstride, s);
    return;
  }
  with_type(in.type, [&](auto e) {
    using T           = decltype(e);
    const auto launch = [&](auto kernel, int threads, int64_t slots) {
      kernel<<<static_cast<unsigned>(std::min(in.m, slots)), threads, 0, s>>>(in, ids, terms, grad_loss, out,
                                                                              static_cast<T*>(grad), gstride, passes_cache(in));
      OCTEX_HIP(hipGetLastError());
    };
    // How a row is held, measured on both sides (us):
    // - a wavefront, 4 pieces a lane: 8192 x 1000 float32 17.6, of 16 pieces 20.6, by 256 threads 27.8; 2048 rows 8.7, 9.9, 10.9;
    //   500 x 2000 bfloat16 6.7 by a wavefront, 6.1 by 256 threads
    // - a wavefront, 16 pieces: 8192 x 4000 float32 57.9, by 256 threads 60.5; but 2048 rows 19.7, 17.1
    // - 256 threads, 4 pieces: 300 x 8000 bfloat16 8.2, by a wavefront 13.4, by 1024 threads 11.7
    // - 256 threads, 16 pieces: 4096 x 32,000 bfloat16 123, by 1024 threads 139; 512 rows 22.7, 22.2
    // - 1024 threads, 4 pieces, of no more rows than CUs: 256 x 16,000 float32 12.2, by 256 threads 15.7
    // - 1024 threads, 8 pieces: 16 x 32,000 float32 11.2, of 16 pieces 12.4; 2048 rows 118, 123
    // - 1024 threads, 16 pieces: 4096 x 128,000 bfloat16 460, in two kernels 597
    const int pieces = (in.n + kPer16<T> - 1) / kPer16<T>;
    if (pieces <= 256 && in.m >= 2048)
      launch(policy_step_kernel<T, 64, 4>, 64, 8192);
    else if (pieces <= 1024 && in.m >= 2048)
      launch(policy_step_kernel<T, 64, 16>, 64, 4096);
    else if (pieces <= 1024)
      launch(policy_step_kernel<T, 256, 4>, 256, 2048);
    else if (pieces <= 4096 && in.m > 256)
      launch(policy_step_kernel<T, 256, 16>, 256, 1024);
    else if (pieces <= 4096)
      launch(policy_step_kernel<T, 1024, 4>, 1024, 256);
    else if (pieces <= 8192)
      launch(policy_step_kernel<T, 1024, 8>, 1024, 256);
    else
      launch(policy_step_kernel<T, 1024, 16>, 1024, 256);
  });
}

}  // namespace cuvs::neighbors::octex::detail
