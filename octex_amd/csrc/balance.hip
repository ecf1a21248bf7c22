// The balance of m rows over e experts: p = softmax of a row's logits, k choices a row.
//
//   f_v  = choices of expert v / all choices;  P_v = sum of p_v over the R rows that count / R
//   loss = balance e sum_v f_v P_v + z (sum of l^2) / R,  l = ln sum exp x
//   dx_v = g p_v / R (balance e (f_v - sum_u f_u p_u) + 2 z l)          (the choices have no gradient)
//
// A row counts if it names an expert; the others (a batch's padding) change nothing.  A row without a finite logit has p = 0
// and no l^2.  A NaN or +inf makes its own row's gradient NaN, and the loss.
//
// The gradient needs all choices first, which come from the ids alone: one kernel counts them by parts, the next adds the
// parts up, takes the logits once, writes the gradient and adds up p, a third joins those sums.  Every sum has a fixed order;
// p's are fp32 within a workgroup and fp64 over them.  Bound by the logits' bytes, or by the launches.

#include "balance.hpp"
#include "rows_device.hpp"

namespace cuvs::neighbors::octex::detail {

namespace {

constexpr int kCountThreads = 1024;
constexpr int kRounds       = 4;  // in which a workgroup's wavefronts add up their sums in LDS

/** The sum over all lanes of a wavefront; of W lanes apart, the same in each of them. */
template <int W, typename V>
__device__ inline auto sum_apart(V v) -> V
{
#pragma unroll
  for (int d = W; d < 64; d *= 2)
    v += __shfl_xor(v, d);
  return v;
}

/** Adds the choices of rows [r0, r1) to counts[0, e), and the rows that count to counts[e]; LDS. */
__device__ inline void count_rows(listed_ids const& experts, int e, int64_t r0, int64_t r1, int* counts)
{
  int rows = 0;
  for (int64_t r = r0 + threadIdx.x; r < r1; r += blockDim.x) {
    bool some = false;
    for (int j = 0; j < experts.k; ++j) {
      const int64_t id = id_at(experts, r, j);
      if (id < 0 || id >= e) continue;
      some = true;
      atomicAdd(counts + id, 1);
    }
    rows += some;
  }
  rows = sum_apart<1>(rows);
  if (threadIdx.x % 64 == 0 && rows > 0) atomicAdd(counts + e, rows);
}

/** The choices of `width` rows a workgroup: parts [gridDim, e + 1]. */
__global__ __launch_bounds__(kCountThreads) void count_choices_kernel(listed_ids experts, int e, int64_t m, int64_t width,
                                                                      int* parts)
{
  __shared__ int counts[kMaxExperts + 1];
  for (int i = threadIdx.x; i <= e; i += kCountThreads)
    counts[i] = 0;
  lds_barrier();
  const int64_t r0 = blockIdx.x * width;
  count_rows(experts, e, r0, min(r0 + width, m), counts);
  lds_barrier();
  for (int i = threadIdx.x; i <= e; i += kCountThreads)
    parts[static_cast<int64_t>(blockIdx.x) * (e + 1) + i] = counts[i];
}

/** Adds n parts up to counts [e + 1] (LDS). */
template <int NT>
__device__ inline void add_parts(const int* parts, int n, int e, int* counts)
{
  for (int i = threadIdx.x; i <= e; i += NT) {
    int sum = 0;
#pragma unroll 8
    for (int p = 0; p < n; ++p)
      sum += parts[static_cast<int64_t>(p) * (e + 1) + i];
    counts[i] = sum;
  }
}

/** The sum of all threads' v; sums [NT / 64] is LDS. */
template <int NT, typename V>
__device__ inline auto sum_block(V v, V* sums) -> V
{
  v = sum_apart<1>(v);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = v;
  lds_barrier();
  v = sums[0];
  for (int w = 1; w < NT / 64; ++w)
    v += sums[w];
  lds_barrier();
  return v;
}

/** The last step of a forward pass, of one workgroup: counts [e + 1] (LDS), the rows that count last, and p(i), the sum of the
 * rows' p_i, of l^2 for i = e. */
template <int NT, typename P>
__device__ inline void write_balance(balance_out const& out, balance_weights const& w, int e, const int* counts, P p,
                                     double* sums)
{
  double choices = 0.;
  for (int i = threadIdx.x; i < e; i += NT)
    choices += counts[i];
  choices           = fmax(sum_block<NT>(choices, sums), 1.);
  const double rows = max(counts[e], 1);
  double sum        = 0.;
  for (int i = threadIdx.x; i < e; i += NT) {
    const double mean = p(i) / rows;
    out.probs[i]      = static_cast<float>(mean);
    out.counts[i]     = counts[i];
    sum += mean * (counts[i] / choices);
  }
  sum = sum_block<NT>(sum, sums);
  if (threadIdx.x != 0) return;
  double loss = double{w.balance} * e * sum;
  if (w.z != 0.f) loss += w.z * (p(e) / rows);
  *out.loss = static_cast<float>(loss);
  *out.rows = counts[e];
}

/** Where a pass takes the choices from: `n` parts; a forward pass's outputs; or (alone) the ids themselves, which its only
 * workgroup counts. */
struct count_source {
  const int* parts;
  int n;
  const int64_t *counts, *rows;
  bool alone;
};

/**
 * Rows by W lanes each, H pieces of 16 bytes a lane, the next row's on their way meanwhile.  A lane keeps the sums of its
 * columns' p in registers over all of its rows; a workgroup's meet in LDS and go to p_parts [gridDim, e + 1] (l^2 last), or,
 * of a workgroup that is alone, to the outputs.
 */
template <typename T, int NT, int W, int H>
__global__ __launch_bounds__(NT) void balance_kernel(score_rows in, listed_ids experts, balance_weights w, balance_out out,
                                                     const float* grad_loss, T* grad, int64_t gstride, bool by_cache,
                                                     count_source from, float* p_parts)
{
  constexpr int N = kPer16<T>, kTeams = NT / W, kWavesHere = NT / 64, kPerRound = kWavesHere / kRounds;
  __shared__ int counts[kMaxExperts + 1];
  __shared__ float p_sums[kPerRound][W * H * N + 1];
  __shared__ double sums[kWavesHere];
  const int e = in.n, sub = static_cast<int>(threadIdx.x) % W;
  const bool forward = from.counts == nullptr;
  if (from.alone) {
    for (int i = threadIdx.x; i <= e; i += NT)
      counts[i] = 0;
    lds_barrier();
    count_rows(experts, e, 0, in.m, counts);
    lds_barrier();
  } else if (from.parts != nullptr) {
    add_parts<NT>(from.parts, from.n, e, counts);
    lds_barrier();
  }
  int at[H];  // a lane's columns; a piece that would pass the row's end is moved back to it
  float f[H][N], p_sum[H][N], z_sum = 0.f, c_balance = 0.f, c_z = 0.f;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    at[h] = (h * W + sub) * N;
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[h][i] = p_sum[h][i] = 0.f;
  }
  if (grad != nullptr) {
    double choices = 0.;
    for (int i = threadIdx.x; i < e; i += NT)
      choices += forward ? static_cast<double>(counts[i]) : static_cast<double>(from.counts[i]);
    choices          = fmax(sum_block<NT>(choices, sums), 1.);
    const double all = forward ? static_cast<double>(counts[e]) : static_cast<double>(*from.rows);
    const float g    = grad_loss != nullptr ? *grad_loss : 1.f, per_row = static_cast<float>(1. / fmax(all, 1.));
    c_balance = g * (w.balance * static_cast<float>(e) * per_row);
    c_z       = g * (2.f * w.z * per_row);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int column = max(min(at[h], e - N), 0) + i;
        if (column >= at[h] && column < e)
          f[h][i] = static_cast<float>((forward ? static_cast<double>(counts[column]) : static_cast<double>(from.counts[column])) /
                                       choices);
      }
  }
  const auto row_at = [&](int64_t r) { return static_cast<const T*>(in.x) + r * in.stride; };
  uint4 next[H];
  int64_t first_id = -1;  // the lane's first choice of the row
  const auto load  = [&](int64_t r) {
    first_id = sub < experts.k ? id_at(experts, r, sub) : -1;
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (h == 0 || at[h] < e || h * W * N < e)
        next[h] = e >= N ? load16(row_at(r) + min(at[h], e - N)) : load_row16(row_at(r), 0, e);
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTeams;
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / W;
  // a wavefront's teams go on together: those past the last row take it again, without a result
  const int64_t leader = static_cast<int64_t>(blockIdx.x) * kTeams + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * (64 / W);
  if (leader < in.m) load(min(mine, in.m - 1));
  for (int64_t r0 = leader; r0 < in.m; r0 += step) {
    const int64_t r = r0 + (mine - leader);
    const bool here = r < in.m;
    bool some       = first_id >= 0 && first_id < e;
    uint4 cur[H];
#pragma unroll
    for (int h = 0; h < H; ++h)
      cur[h] = next[h];
    for (int j = W + sub; j < experts.k; j += W) {
      const int64_t id = id_at(experts, min(r, in.m - 1), j);
      some             = some || (id >= 0 && id < e);
    }
    if (r0 + step < in.m) load(min(r + step, in.m - 1));
    const key64 lanes  = __ballot(some) >> (threadIdx.x % 64 / W * W);
    const bool counted = here && (W == 64 ? lanes : lanes & ((key64{1} << (W % 64)) - 1)) != 0;
    float v[H][N], top = -INFINITY;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      unpack16<T>(cur[h], v[h]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int column = max(min(at[h], e - N), 0) + i;
        if (column < at[h] || column >= e) v[h][i] = -INFINITY;
        top = fmaxf(top, v[h][i]);
      }
    }
    top             = reduce_lanes<W>(top, [](float x, float y) { return fmaxf(x, y); });
    const float ref = top == -INFINITY ? 0.f : top;
    float s         = 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[h][i] = exp2_fast((v[h][i] - ref) * kLog2e);
        s += v[h][i];
      }
    s                 = sum_lanes<W>(s);
    const float lse   = s > 0.f ? ref + logf(s) : s + top;  // nothing: 0 - inf; a NaN stays one
    const float per_s = s > 0.f ? 1.f / s : s;
    const float l     = s == 0.f ? 0.f : lse;
    float inner       = 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[h][i] *= per_s;
        p_sum[h][i] += counted ? v[h][i] : 0.f;
        inner = fmaf(f[h][i], v[h][i], inner);
      }
    if (forward && sub == 0) {
      z_sum += counted ? l * l : 0.f;
      if (here) out.lse[r] = counted ? lse : 0.f;
    }
    if (grad == nullptr) continue;
    inner          = sum_lanes<W>(inner);
    const float cz = c_z * l;
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[h][i] = counted ? v[h][i] * fmaf(c_balance, f[h][i] - inner, cz) : 0.f;
    }
    if (!here) continue;
    T* to = grad + r * gstride;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (at[h] >= e) continue;
      if (at[h] + N <= e) {
        if (by_cache)
          store16(to + at[h], pack16<T>(v[h]));
        else
          store16_nt(to + at[h], pack16<T>(v[h]));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int column = max(e - N, 0) + i;
          if (column >= at[h] && column < e) to[column] = static_cast<T>(v[h][i]);
        }
      }
    }
  }
  if (!forward) return;
  z_sum = sum_apart<1>(z_sum);
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < N; ++i)
      p_sum[h][i] = sum_apart<W>(p_sum[h][i]);
  const int wave = static_cast<int>(threadIdx.x) / 64;
  for (int round = 0; round < kRounds; ++round) {
    if (wave / kPerRound == round && threadIdx.x % 64 < W) {
      float* to       = p_sums[wave % kPerRound];
      const auto join = [&](int i, float v) { to[i] = round == 0 ? v : to[i] + v; };
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int column = max(min(at[h], e - N), 0) + i;
          if (column >= at[h] && column < e) join(column, p_sum[h][i]);
        }
      if (sub == 0) join(e, z_sum);
    }
    lds_barrier();
  }
  const auto total = [&](int i) {
    float sum = p_sums[0][i];
    for (int q = 1; q < kPerRound; ++q)
      sum += p_sums[q][i];
    return sum;
  };
  if (from.alone) return write_balance<NT>(out, w, e, counts, total, sums);
  for (int i = threadIdx.x; i <= e; i += NT)
    p_parts[static_cast<int64_t>(blockIdx.x) * (e + 1) + i] = total(i);
}

constexpr int kFinishThreads = 1024;

/** Joins the parts of the choices and of p. */
__global__ __launch_bounds__(kFinishThreads) void finish_balance_kernel(balance_weights w, balance_out out, int e,
                                                                        const int* parts, int n, const float* p_parts, int np)
{
  __shared__ int counts[kMaxExperts + 1];
  __shared__ double p[kMaxExperts + 1];
  __shared__ double sums[kFinishThreads / 64];
  add_parts<kFinishThreads>(parts, n, e, counts);
  for (int i = threadIdx.x; i <= e; i += kFinishThreads) {
    double sum = 0.;
#pragma unroll 8
    for (int q = 0; q < np; ++q)
      sum += p_parts[static_cast<int64_t>(q) * (e + 1) + i];
    p[i] = sum;
  }
  lds_barrier();
  write_balance<kFinishThreads>(out, w, e, counts, [&](int i) { return p[i]; }, sums);
}

constexpr int kMaxCountParts = 64, kMaxWorkgroups = 512;

/** How a pass is shared out. */
struct balance_plan {
  bool alone;
  int count_parts, workgroups, teams;
  int64_t width;  // rows of a part
};

auto per_row(int e, elem type) -> int { return (e * elem_size(type) + 15) / 16; }

auto plan_of(int64_t m, int e, int k, elem type) -> balance_plan
{
  balance_plan p{};
  const int pieces = per_row(e, type);
  int lanes        = 1;
  while (lanes < 64 && lanes < pieces)
    lanes *= 2;
  const int threads = pieces > 64 ? 512 : 1024;
  p.teams           = threads / lanes;
  p.alone           = m * e <= 32768 && m * k <= 8192;
  p.workgroups      = p.alone ? 1 : static_cast<int>(std::min<int64_t>((m + p.teams - 1) / p.teams, kMaxWorkgroups));
  p.count_parts     = static_cast<int>(std::clamp<int64_t>(m / kCountThreads, 1, kMaxCountParts));
  p.width           = (m + p.count_parts - 1) / p.count_parts;
  return p;
}

template <typename T, typename F>
void with_team(int pieces, F f)
{
  const auto call = [&](auto nt, auto w, auto h) { f(nt, w, h); };
  constexpr auto kSmall = std::integral_constant<int, 1024>{};
  constexpr auto kLarge = std::integral_constant<int, 512>{};
  constexpr auto one    = std::integral_constant<int, 1>{};
  if (pieces <= 1) return call(kSmall, one, one);
  if (pieces <= 2) return call(kSmall, std::integral_constant<int, 2>{}, one);
  if (pieces <= 4) return call(kSmall, std::integral_constant<int, 4>{}, one);
  if (pieces <= 8) return call(kSmall, std::integral_constant<int, 8>{}, one);
  if (pieces <= 16) return call(kSmall, std::integral_constant<int, 16>{}, one);
  if (pieces <= 32) return call(kSmall, std::integral_constant<int, 32>{}, one);
  if (pieces <= 64) return call(kSmall, std::integral_constant<int, 64>{}, one);
  if (pieces <= 128) return call(kLarge, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  if (sizeof(T) == 2 || pieces <= 256) return call(kLarge, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  if constexpr (sizeof(T) == 4) call(kLarge, std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
}

template <typename T>
void run_balance(score_rows const& in, listed_ids const& experts, balance_weights const& w, balance_out const& out,
                 const float* grad_loss, void* grad, int64_t gstride, count_source const& from, float* p_parts, int workgroups,
                 hipStream_t s)
{
  with_team<T>(per_row(in.n, in.type), [&](auto nt, auto lanes, auto h) {
    balance_kernel<T, nt(), lanes(), h()><<<workgroups, nt(), 0, s>>>(in, experts, w, out, grad_loss, static_cast<T*>(grad),
                                                                       gstride, passes_cache(in), from, p_parts);
    OCTEX_HIP(hipGetLastError());
  });
}

}  // namespace

auto balance_workspace(int64_t m, int e, int k, elem type) -> int64_t
{
  const auto p = plan_of(m, e, k, type);
  return p.alone ? 0 : int64_t{4} * (p.count_parts + p.workgroups) * (e + 1);
}

void launch_balance(score_rows const& in, listed_ids const& experts, balance_weights const& w, balance_out const& out,
                    const float* grad_loss, void* grad, int64_t gstride, void* workspace, hipStream_t s)
{
  const auto p  = plan_of(in.m, in.n, experts.k, in.type);
  auto* parts   = static_cast<int*>(workspace);
  auto* p_parts = reinterpret_cast<float*>(parts + int64_t{p.count_parts} * (in.n + 1));
  if (!p.alone) {
    count_choices_kernel<<<p.count_parts, kCountThreads, 0, s>>>(experts, in.n, in.m, p.width, parts);
    OCTEX_HIP(hipGetLastError());
  }
  const count_source from{p.alone || grad == nullptr ? nullptr : parts, p.count_parts, nullptr, nullptr, p.alone};
  with_type(in.type, [&](auto e) {
    run_balance<decltype(e)>(in, experts, w, out, grad_loss, grad, gstride, from, p_parts, p.workgroups, s);
  });
  if (!p.alone) {
    finish_balance_kernel<<<1, kFinishThreads, 0, s>>>(w, out, in.n, parts, p.count_parts, p_parts, p.workgroups);
    OCTEX_HIP(hipGetLastError());
  }
}

void launch_balance_backward(score_rows const& in, listed_ids const& experts, balance_weights const& w, const int64_t* counts,
                             const int64_t* rows, const float* grad_loss, void* grad, int64_t gstride, hipStream_t s)
{
  const auto p = plan_of(in.m, in.n, experts.k, in.type);
  const int workgroups = static_cast<int>(std::min<int64_t>((in.m + p.teams - 1) / p.teams, kMaxWorkgroups));
  const count_source from{nullptr, 0, counts, rows, false};
  with_type(in.type, [&](auto e) {
    run_balance<decltype(e)>(in, experts, w, {}, grad_loss, grad, gstride, from, nullptr, workgroups, s);
  });
}

}  // namespace cuvs::neighbors::octex::detail
