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
// p's are fp32 within a workgroup and fp64 over several (up to 32,768 logits are one's alone).  Bound by the logits' bytes, or by
// the launches: 131,072 x 256 bfloat16 with 8 choices in both directions take 46 us (7.7 + 31.9, at 4.2 TB/s, + 6.5), 64 x 8
// float32 5.8.

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

constexpr int kIdsAhead = 8;  // of a row, that a thread has on their way

/** Adds the choices of rows [r0, r1) to counts[0, e), and the rows that count to counts[e]; LDS. */
__device__ inline void count_rows(listed_ids const& experts, int e, int64_t r0, int64_t r1, int* counts)
{
  int rows = 0;
  for (int64_t r = r0 + threadIdx.x; r < r1; r += blockDim.x) {
    bool some = false;
    for (int j = 0; j < experts.k; j += kIdsAhead) {
      int64_t id[kIdsAhead];
      if (experts.wide) {
#pragma unroll
        for (int q = 0; q < kIdsAhead; ++q)
          id[q] = static_cast<const int64_t*>(experts.ids)[r * experts.stride + min(j + q, experts.k - 1)];
      } else {
#pragma unroll
        for (int q = 0; q < kIdsAhead; ++q)
          id[q] = static_cast<const int32_t*>(experts.ids)[r * experts.stride + min(j + q, experts.k - 1)];
      }
#pragma unroll
      for (int q = 0; q < kIdsAhead; ++q) {
        if (j + q >= experts.k || id[q] < 0 || id[q] >= e) continue;
        some = true;
        atomicAdd(counts + id[q], 1);
      }
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

/** Adds n parts up to counts [e + 1] (LDS), as many threads a count as there are. */
template <int NT>
__device__ inline void add_parts(const int* parts, int n, int e, int* counts)
{
  for (int i = threadIdx.x; i <= e; i += NT)
    counts[i] = 0;
  lds_barrier();
  const int columns = e + 1, groups = max(NT / columns, 1);
  for (int i = threadIdx.x; i < columns * groups; i += NT) {
    const int group = i / columns, column = i - group * columns;
    int sum = 0;
#pragma unroll 16
    for (int p = group; p < n; p += groups)
      sum += parts[static_cast<int64_t>(p) * columns + column];
    if (sum > 0) atomicAdd(counts + column, sum);
  }
  lds_barrier();
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

/** Where a pass takes the choices from: `n` parts; a forward pass's outputs; or (alone) the ids themselves, which its only
 * workgroup counts. */
struct count_source {
  const int* parts;
  int n;
  const int64_t *counts, *rows;
  bool alone;
};

/** Columns that a pass leaves in its parts beside the experts' sums of p: the sums of l^2, and of the rows' sum_v f_v p_v. */
constexpr int kMoreSums = 2;

__device__ inline auto loss_of(balance_weights const& w, int e, double rows, double squares, double inner) -> float
{
  double loss = w.balance != 0.f ? double{w.balance} * e * (inner / rows) : 0.;
  if (w.z != 0.f) loss += w.z * (squares / rows);
  return static_cast<float>(loss);
}

/**
 * Rows by W lanes each, H pieces of 16 bytes a lane, the next row's on their way meanwhile.  A lane keeps the sums of its
 * columns' p in registers over all of its rows; a workgroup's meet in LDS and go to p_parts [gridDim, e + kMoreSums], or, of a
 * workgroup that is alone, to the outputs.  kWhole: rows are whole pieces; else a piece that would pass the row's end is moved
 * back to it, and columns that it shares with its neighbor are masked.
 */
template <typename T, int NT, int W, int H, bool kWhole>
__global__ __launch_bounds__(NT) void balance_kernel(score_rows in, listed_ids experts, balance_weights w, balance_out out,
                                                     const float* grad_loss, T* grad, int64_t gstride, bool by_cache,
                                                     count_source from, float* p_parts)
{
  constexpr int N = kPer16<T>, kTeams = NT / W, kWavesHere = NT / 64, kPerRound = kWavesHere / kRounds;
  __shared__ int counts[kMaxExperts + 1];
  __shared__ float p_sums[kPerRound][W * H * N + kMoreSums];
  __shared__ double sums[kWavesHere];
  __shared__ float shares[kMaxExperts];
  const int e = in.n, sub = static_cast<int>(threadIdx.x) % W;
  const bool forward = from.counts == nullptr;
  // a lane's columns, and where their piece lies
  const auto at_of    = [&](int h) { return (h * W + sub) * N; };
  const auto place_of = [&](int h) { return kWhole ? at_of(h) : max(min(at_of(h), e - N), 0); };
  const auto own      = [&](int h, int i) { return kWhole || (place_of(h) + i >= at_of(h) && place_of(h) + i < e); };
  const auto row_at   = [&](int64_t r) { return static_cast<const T*>(in.x) + r * in.stride; };
  uint4 next[H];
  int64_t first_id = -1;  // the lane's first choice of the row
  {
    float nothing_here[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      nothing_here[i] = -INFINITY;
#pragma unroll
    for (int h = 0; h < H; ++h)
      next[h] = pack16<T>(nothing_here);
  }
  const auto load = [&](int64_t r) {
    first_id = sub < experts.k ? id_at(experts, r, sub) : -1;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (kWhole ? at_of(h) >= e : h * W * N >= e) continue;
      next[h] = kWhole || e >= N ? load16(row_at(r) + place_of(h)) : load_row16(row_at(r), 0, e);
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTeams;
  // a wavefront's teams go on together: those past the last row take that again, without a result
  const int64_t leader = static_cast<int64_t>(blockIdx.x) * kTeams + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * (64 / W);
  const int team       = static_cast<int>(threadIdx.x) % 64 / W;
  if (leader < in.m) load(min(leader + team, in.m - 1));
  if (from.alone) {
    for (int i = threadIdx.x; i <= e; i += NT)
      counts[i] = 0;
    lds_barrier();
    count_rows(experts, e, 0, in.m, counts);
    lds_barrier();
  } else if (forward) {
    add_parts<NT>(from.parts, from.n, e, counts);
  }
  const auto count_of = [&](int i) { return forward ? static_cast<double>(counts[i]) : static_cast<double>(from.counts[i]); };
  double choices      = 0.;
  for (int i = threadIdx.x; i < e; i += NT)
    choices += count_of(i);
  choices = fmax(sum_block<NT>(choices, sums), 1.);
  for (int i = threadIdx.x; i < e; i += NT)
    shares[i] = static_cast<float>(count_of(i) / choices);
  lds_barrier();
  const double rows = fmax(forward ? static_cast<double>(counts[e]) : static_cast<double>(*from.rows), 1.);
  const float g = grad_loss != nullptr ? *grad_loss : 1.f, per_row = static_cast<float>(1. / rows);
  const float c_balance = g * (w.balance * static_cast<float>(e) * per_row), c_z = g * (2.f * w.z * per_row);
  float f[H][N], p_sum[H][N], z_sum = 0.f, inner_sum = 0.f;
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      p_sum[h][i] = 0.f;
      f[h][i]     = own(h, i) && at_of(h) < e ? shares[place_of(h) + i] : 0.f;
    }
  for (int64_t r0 = leader; r0 < in.m; r0 += step) {
    const int64_t r = r0 + team;
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
      // rows that do not count are read as zeros, whatever they hold
      unpack16<T>(counted ? cur[h] : uint4{0, 0, 0, 0}, v[h]);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!own(h, i)) v[h][i] = -INFINITY;
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
    const float per_s = !counted ? 0.f : s > 0.f ? 1.f / s : s;
    const float l     = counted && s != 0.f ? lse : 0.f;
    float inner       = 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[h][i] *= per_s;
        p_sum[h][i] += v[h][i];
        inner = fmaf(f[h][i], v[h][i], inner);
      }
    inner = sum_lanes<W>(inner);
    z_sum += l * l;
    inner_sum += inner;
    if (forward && sub == 0 && here) out.lse[r] = counted ? lse : 0.f;
    if (grad == nullptr) continue;
    // a row that does not count has none, also where the loss weighs infinitely much
    const float cb = counted ? c_balance : 0.f, cz = counted ? c_z * l : 0.f;
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[h][i] *= fmaf(cb, f[h][i] - inner, cz);
    }
    if (!here) continue;
    T* to = grad + r * gstride;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (at_of(h) >= e) continue;
      if (kWhole || at_of(h) + N <= e) {
        if (by_cache)
          store16(to + at_of(h), pack16<T>(v[h]));
        else
          store16_nt(to + at_of(h), pack16<T>(v[h]));
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (own(h, i)) to[place_of(h) + i] = static_cast<T>(v[h][i]);
      }
    }
  }
  if (!forward) return;
  // every lane of a team has its z_sum and inner_sum
  z_sum     = sum_apart<W>(z_sum);
  inner_sum = sum_apart<W>(inner_sum);
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < N; ++i)
      p_sum[h][i] = sum_apart<W>(p_sum[h][i]);
  const int wave = static_cast<int>(threadIdx.x) / 64;
  for (int round = 0; round < kRounds; ++round) {
    if (wave / kPerRound == round && threadIdx.x % 64 < W) {
      float* to       = p_sums[wave % kPerRound];
      const auto join = [&](int i, float x) { to[i] = round == 0 ? x : to[i] + x; };
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (own(h, i) && at_of(h) < e) join(place_of(h) + i, p_sum[h][i]);
      if (sub == 0) join(e, z_sum), join(e + 1, inner_sum);
    }
    lds_barrier();
  }
  const auto total = [&](int i) {
    float sum = p_sums[0][i];
    for (int q = 1; q < kPerRound; ++q)
      sum += p_sums[q][i];
    return sum;
  };
  if (!from.alone) {
    for (int i = threadIdx.x; i < e + kMoreSums; i += NT)
      p_parts[static_cast<int64_t>(blockIdx.x) * (e + kMoreSums) + i] = total(i);
    return;
  }
  for (int i = threadIdx.x; i < e; i += NT) {
    out.probs[i]  = static_cast<float>(total(i) / rows);
    out.counts[i] = counts[i];
  }
  if (threadIdx.x != 0) return;
  *out.loss = loss_of(w, e, rows, total(e), total(e + 1));
  *out.rows = counts[e];
}

constexpr int kFinishThreads = 1024, kFinishWaves = kFinishThreads / 64;

/** Joins the parts of p, 64 columns a workgroup; one more joins those of the choices and gives the loss. */
__global__ __launch_bounds__(kFinishThreads) void finish_balance_kernel(balance_weights w, balance_out out, int e,
                                                                        const int* parts, int n, const float* p_parts, int np)
{
  __shared__ double sums[kFinishWaves][64];
  __shared__ int counts[kMaxExperts + 1];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const bool last  = blockIdx.x + 1 == gridDim.x;
  const int column = last ? e + min(lane, kMoreSums - 1) : min(static_cast<int>(blockIdx.x) * 64 + lane, e - 1);
  const int rows   = sum_apart<1>(lane < n ? parts[lane * (e + 1) + e] : 0);
  double sum       = 0.;
#pragma unroll 16
  for (int q = wave; q < np; q += kFinishWaves)
    sum += p_parts[static_cast<int64_t>(q) * (e + kMoreSums) + column];
  sums[wave][lane] = sum;
  if (last) {
    add_parts<kFinishThreads>(parts, n, e, counts);
    for (int i = threadIdx.x; i < e; i += kFinishThreads)
      out.counts[i] = counts[i];
    if (threadIdx.x == 0) *out.rows = counts[e];
  }
  lds_barrier();
  if (wave > 0) return;
  const double rows_here = max(rows, 1);
  for (int q = 1; q < kFinishWaves; ++q)
    sum += sums[q][lane];
  if (!last) {
    if (static_cast<int>(blockIdx.x) * 64 + lane < e) out.probs[column] = static_cast<float>(sum / rows_here);
    return;
  }
  const double inner = __shfl(sum, 1);
  if (lane == 0) *out.loss = loss_of(w, e, rows_here, sum, inner);
}

constexpr int kMaxCountParts = 64;
/** Threads of a pass: two workgroups of 512 a CU, or one of 1024 (30,000 x 128 bfloat16: 20 us; two 28). */
constexpr int kMaxThreads = 1 << 18;

auto pieces_of(int e, elem type) -> int { return (e * elem_size(type) + 15) / 16; }

constexpr int kManyRows = 32768;

/** Calls f with the threads of a workgroup, the lanes of a row and the pieces of a lane.  Many rows take 16 values a lane: what
 * a row's lanes exchange, and a lane's steps beside its pieces, are fewer then (131,072 x 256 bfloat16: 34 us; 8 values 51, 32
 * values 46, whose registers leave a CU half of the wavefronts).  Few rows take as many lanes as they have pieces. */
template <typename T, typename F>
void with_team(int64_t m, int pieces, F f)
{
  using std::integral_constant;
  constexpr auto one         = integral_constant<int, 1>{};
  constexpr auto many        = integral_constant<int, sizeof(T) == 4 ? 4 : 2>{};
  constexpr auto most        = integral_constant<int, sizeof(T) == 4 ? 8 : 4>{};
  constexpr auto wide        = integral_constant<int, 64>{};
  constexpr auto small_group = integral_constant<int, 512>{};
  constexpr auto group       = integral_constant<int, 1024>{};
  if (pieces > 64 * many()) return f(small_group, wide, most);
  if (m >= kManyRows || pieces > 64) {
    if (pieces <= many()) return f(small_group, one, many);
    if (pieces <= 2 * many()) return f(small_group, integral_constant<int, 2>{}, many);
    if (pieces <= 4 * many()) return f(small_group, integral_constant<int, 4>{}, many);
    if (pieces <= 8 * many()) return f(small_group, integral_constant<int, 8>{}, many);
    if (pieces <= 16 * many()) return f(small_group, integral_constant<int, 16>{}, many);
    if (pieces <= 32 * many()) return f(small_group, integral_constant<int, 32>{}, many);
    return f(small_group, wide, many);
  }
  if (pieces <= 1) return f(group, one, one);
  if (pieces <= 2) return f(group, integral_constant<int, 2>{}, one);
  if (pieces <= 4) return f(group, integral_constant<int, 4>{}, one);
  if (pieces <= 8) return f(group, integral_constant<int, 8>{}, one);
  if (pieces <= 16) return f(group, integral_constant<int, 16>{}, one);
  if (pieces <= 32) return f(group, integral_constant<int, 32>{}, one);
  f(group, wide, one);
}

/** How a pass is shared out. */
struct balance_plan {
  bool alone;
  int count_parts, workgroups;
  int64_t width;  // rows of a part
};

auto plan_of(int64_t m, int e, int k, elem type) -> balance_plan
{
  balance_plan p{};
  int threads = 1, teams = 1;
  with_type(type, [&](auto x) {
    with_team<decltype(x)>(m, pieces_of(e, type), [&](auto nt, auto w, auto) { threads = nt(), teams = nt() / w(); });
  });
  p.alone       = m * e <= 32768 && m * k <= 8192;
  p.workgroups  = p.alone ? 1 : static_cast<int>(std::min<int64_t>((m + teams - 1) / teams, kMaxThreads / threads));
  p.count_parts = static_cast<int>(std::clamp<int64_t>(m / kCountThreads, 1, kMaxCountParts));
  p.width       = (m + p.count_parts - 1) / p.count_parts;
  return p;
}

void run_balance(score_rows const& in, listed_ids const& experts, balance_weights const& w, balance_out const& out,
                 const float* grad_loss, void* grad, int64_t gstride, count_source const& from, float* p_parts, int workgroups,
                 hipStream_t s)
{
  with_type(in.type, [&](auto x) {
    using T = decltype(x);
    with_team<T>(in.m, pieces_of(in.n, in.type), [&](auto nt, auto lanes, auto h) {
      const auto kernel = in.n % kPer16<T> == 0 ? balance_kernel<T, nt(), lanes(), h(), true>
                                                : balance_kernel<T, nt(), lanes(), h(), false>;
      kernel<<<workgroups, nt(), 0, s>>>(in, experts, w, out, grad_loss, static_cast<T*>(grad), gstride, passes_cache(in), from,
                                         p_parts);
      OCTEX_HIP(hipGetLastError());
    });
  });
}

}  // namespace

auto balance_workspace(int64_t m, int e, int k, elem type) -> int64_t
{
  const auto p = plan_of(m, e, k, type);
  return p.alone ? 0 : int64_t{4} * (int64_t{p.count_parts} * (e + 1) + int64_t{p.workgroups} * (e + kMoreSums));
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
  run_balance(in, experts, w, out, grad_loss, grad, gstride, {parts, p.count_parts, nullptr, nullptr, p.alone}, p_parts,
              p.workgroups, s);
  if (!p.alone) {
    finish_balance_kernel<<<(in.n + 63) / 64 + 1, kFinishThreads, 0, s>>>(w, out, in.n, parts, p.count_parts, p_parts, p.workgroups);
    OCTEX_HIP(hipGetLastError());
  }
}

void launch_balance_backward(score_rows const& in, listed_ids const& experts, balance_weights const& w, const int64_t* counts,
                             const int64_t* rows, const float* grad_loss, void* grad, int64_t gstride, hipStream_t s)
{
  auto p = plan_of(in.m, in.n, experts.k, in.type);
  if (p.alone) p.workgroups = 1;
  run_balance(in, experts, w, {}, grad_loss, grad, gstride, {nullptr, 0, counts, rows, false}, nullptr, p.workgroups, s);
}

}  // namespace cuvs::neighbors::octex::detail
