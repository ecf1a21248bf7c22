// Operators on rows of scores: a row holds one query's (or token's) n logits x, read as z = x / T.
//
//   log_probs   l = ln sum exp z;  log p_v = z_v - l of the given ids;  H = l - sum p z;  the top entries by (value, id)
//   distill     q = softmax(teacher / T) over the listed ids;  loss = sum q_j (ln q_j - log p_{id_j})
//   backward    dx_v = p_v (A + B ln p_v) + sum over the listed j with id_j = v of w_j, with
//               log_probs: A = -(sum g + h H) / T, B = -h / T, w = g / T;  distill: A = g / T, B = 0, w = -g q / T
//
// One pass over a row holds, a thread, the running maximum m, s = sum 2^u and t = sum 2^u u with u = (x - m) log2(e) / T:
// then l = m / T + ln s and H = ln s - ln 2 t / s, a difference of small numbers.  All sums are fp32, in a fixed order.
// A row without a finite score has p = 0 everywhere: l = -inf, H = 0, log p = -inf.  A NaN or +inf makes its row NaN.

#include "common.hpp"
#include "elems_device.hpp"
#include "rows.hpp"

#include <algorithm>

namespace cuvs::neighbors::octex::detail {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2   = 0.693147180559945309417f;
constexpr float kFloor = -200.f;  // an exponent whose power of two is 0; keeps 0 * -inf out of the sums
constexpr int kThreads = 256;
constexpr int kWaves   = kThreads / 64;
constexpr int kUnroll  = 4;     // 16-byte loads a thread keeps in flight
constexpr int kList    = 256;   // a wavefront's candidate keys: four a lane
constexpr int kSlack   = 12;    // entries that a compaction may keep beyond the k best

__device__ inline auto exp2_fast(float v) -> float { return __builtin_amdgcn_exp2f(v); }

__device__ inline void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

/** The running sums of a part of a row; ref is m, or 0 while there is no finite score. */
struct run {
  float m, ref, s, t;
};

__device__ inline auto nothing() -> run { return {-INFINITY, 0.f, 0.f, 0.f}; }

/** Adds N scores; returns their largest. */
template <bool kEntropy, int N>
__device__ inline auto add_scores(run& r, const float (&v)[N], float c) -> float
{
  float cm = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    cm = fmaxf(cm, v[i]);
  if (cm > r.m) {
    const float d = fmaxf((r.m - cm) * c, kFloor), f = exp2_fast(d);
    if constexpr (kEntropy) r.t = (r.t + r.s * d) * f;
    r.s *= f;
    r.m = r.ref = cm;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float u = (v[i] - r.ref) * c, e = exp2_fast(u);
    r.s += e;
    if constexpr (kEntropy) r.t = fmaf(e, fmaxf(u, kFloor), r.t);
  }
  return cm;
}

__device__ inline auto join(run const& a, run const& b, float c) -> run
{
  run r;
  r.m   = fmaxf(a.m, b.m);
  r.ref = r.m == -INFINITY ? 0.f : r.m;
  const float da = fmaxf((a.m - r.ref) * c, kFloor), db = fmaxf((b.m - r.ref) * c, kFloor);
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  r.s = a.s * fa + b.s * fb;
  r.t = (a.t + a.s * da) * fa + (b.t + b.s * db) * fb;
  return r;
}

__device__ inline auto shuffle_xor(run const& a, int mask) -> run
{
  run r;
  r.m = __shfl_xor(a.m, mask);
  r.s = __shfl_xor(a.s, mask);
  r.t = __shfl_xor(a.t, mask);
  return r;
}

/** The whole workgroup's sums, the same in every thread; parts [kWaves] is LDS. */
__device__ inline auto join_block(run r, float c, run* parts) -> run
{
#pragma unroll
  for (int mask = 32; mask > 0; mask >>= 1)
    r = join(r, shuffle_xor(r, mask), c);
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = r;
  __syncthreads();
  r = parts[0];
  for (int w = 1; w < kWaves; ++w)
    r = join(r, parts[w], c);
  return r;
}

struct row_sums {
  float m, ln_s, lse, entropy;
};

__device__ inline auto finish(run const& r, float temperature) -> row_sums
{
  row_sums o;
  o.m       = r.m;
  o.ln_s    = logf(r.s);
  o.lse     = r.s > 0.f ? r.m / temperature + o.ln_s : r.s + r.m;  // nothing: 0 - inf; a NaN stays one
  o.entropy = r.s > 0.f ? o.ln_s - kLn2 * r.t / r.s : r.s;
  return o;
}

__device__ inline auto log_prob(float x, row_sums const& o, float temperature) -> float
{
  if (x == -INFINITY && !isnan(o.lse)) return x;
  return (x - o.m) / temperature - o.ln_s;
}

// ---- the top entries: a wavefront's list of keys (order of the value, ~column), compacted when it fills

using key64 = unsigned long long;

__device__ inline auto key_of(float v, int column) -> key64
{
  const unsigned b = __float_as_uint(v + 0.f);  // -0 and 0 are one value
  const unsigned o = b >> 31 ? ~b : b | 0x80000000u;
  return key64{o} << 32 | static_cast<unsigned>(~column);
}

__device__ inline auto value_of_order(unsigned o) -> float { return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ inline auto value_of(key64 k) -> float { return value_of_order(static_cast<unsigned>(k >> 32)); }
__device__ inline auto column_of(key64 k) -> int { return static_cast<int>(~static_cast<unsigned>(k)); }

/** A floor such that at least k and at most k + slack of the wavefront's distinct keys (0: none) reach it; 0 if there are
 * not k. */
__device__ inline auto floor_of(const key64 (&key)[4], int k, int slack) -> key64
{
  key64 p = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const key64 q = p | key64{1} << bit;
    int c         = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c += __popcll(__ballot(key[j] >= q));
    if (c >= k) {
      p = q;
      if (c <= k + slack) break;
    }
  }
  return p;
}

/** Writes the keys at or above floor to list, dense; returns their count. */
__device__ inline auto keep_from(const key64 (&key)[4], key64 floor, key64* list) -> int
{
  const int lane = threadIdx.x % 64;
  int n          = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in  = key[j] != 0 && key[j] >= floor;
    const key64 at = __ballot(in);
    if (in) list[n + __popcll(at & ((key64{1} << lane) - 1))] = key[j];
    n += __popcll(at);
  }
  wave_fence();
  return n;
}

struct top_list {
  key64* list;  // [kList] in LDS, this wavefront's
  int k;
  int n     = 0;
  float thr = -INFINITY;  // no later score at or below it is among the k best

  __device__ void compact(int slack)
  {
    const int lane = threadIdx.x % 64;
    key64 key[4];
    wave_fence();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      key[j] = lane + 64 * j < n ? list[lane + 64 * j] : 0;
    wave_fence();
    const key64 p    = floor_of(key, k, slack);
    n                = keep_from(key, p, list);
    const unsigned o = static_cast<unsigned>(p >> 32);
    if (o >= 0x00800000u) thr = value_of_order(o);  // below: not a number's order
  }

  /** Scores v of columns at + i, above every column of earlier calls; cm is their largest. */
  template <int N>
  __device__ void add(const float (&v)[N], float cm, int at)
  {
    const float before = thr;
    if (__ballot(cm > before) == 0) return;
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // equal scores of lower columns may come in this very call, so a floor it raised lets them in
      const bool in  = v[i] > before && v[i] >= thr;
      const key64 at_lanes = __ballot(in);
      if (at_lanes == 0) continue;
      if (in) list[n + __popcll(at_lanes & ((key64{1} << lane) - 1))] = key_of(v[i], at + i);
      n += __popcll(at_lanes);
      if (n > kList - 64) compact(kSlack);
    }
  }
};

/** The k best of `lists` lists of at most 64 keys each, lists[i * kList + ..] with counts n[i]; into list 0. */
__device__ inline void merge_lists(key64* lists, int* n, int count, int k)
{
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  while (count > 1) {
    const int groups = (count + 3) / 4;
    key64 key[4]     = {0, 0, 0, 0};
    if (wave < groups) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int l = 4 * wave + j;
        if (l < count && lane < n[l]) key[j] = lists[l * kList + lane];
      }
    }
    __syncthreads();
    if (wave < groups) {
      const int kept = keep_from(key, floor_of(key, k, 0), lists + wave * kList);
      if (lane == 0) n[wave] = kept;
    }
    __syncthreads();
    count = groups;
  }
}

// ---- one pass over a row

/** Calls f(v, at) for the scores of columns [c0, c1) that this thread takes, 16 bytes at a time in ascending order; a
 * score outside the range, or one that another thread takes, comes as -inf.  Every lane of a wavefront calls f alike. */
template <typename T, typename F>
__device__ inline void for_scores(const T* row, int c0, int c1, F f)
{
  constexpr int N = kPer16<T>;
  float v[N];
  if (c1 - c0 < N) {
    const int at = c0 + static_cast<int>(threadIdx.x);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = -INFINITY;
    if (at < c1) v[0] = static_cast<float>(row[at]);
    f(v, at);
    return;
  }
  const int last = c1 - N;  // a load that would pass the range's end is moved back to it
  const int wave = c0 + static_cast<int>(threadIdx.x / 64) * 64 * N, mine = static_cast<int>(threadIdx.x % 64) * N;
  constexpr int kStep = kThreads * N;
  uint4 next[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    next[u] = load16(row + min(wave + u * kStep + mine, last));
  for (int w = wave; w < c1; w += kUnroll * kStep) {
    uint4 cur[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      cur[u] = next[u];
    if (w + kUnroll * kStep < c1) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        next[u] = load16(row + min(w + (kUnroll + u) * kStep + mine, last));
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int w0 = w + u * kStep;
      if (w0 >= c1) break;
      unpack16<T>(cur[u], v);
      int at = w0 + mine;
      if (w0 + 64 * N > c1) {
        const int from = min(at, last);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (from + i < at) v[i] = -INFINITY;
        at = from;
      }
      f(v, at);
    }
  }
}

__device__ inline auto id_at(listed_ids const& ids, int64_t row, int j) -> int64_t
{
  const int64_t i = row * ids.stride + j;
  return ids.wide ? static_cast<const int64_t*>(ids.ids)[i] : static_cast<const int32_t*>(ids.ids)[i];
}

template <typename T, bool kTop>
__global__ __launch_bounds__(kThreads) void log_probs_kernel(score_rows in, listed_ids ids, log_probs_out out,
                                                             int64_t row0)
{
  __shared__ run parts[kWaves];
  __shared__ key64 lists[kTop ? kWaves * kList : 1];
  __shared__ int counts[kWaves];
  const int64_t r = row0 + blockIdx.x;
  const T* row    = static_cast<const T*>(in.x) + r * in.stride;
  const float c   = kLog2e / in.temperature;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  run sums        = nothing();
  top_list top{lists + (kTop ? wave * kList : 0), out.top};
  for_scores<T>(row, 0, in.n, [&](const auto& v, int at) {
    const float cm = add_scores<true>(sums, v, c);
    if constexpr (kTop) top.add(v, cm, at);
  });
  const auto o = finish(join_block(sums, c, parts), in.temperature);
  if (threadIdx.x == 0) {
    out.lse[r]     = o.lse;
    out.entropy[r] = o.entropy;
  }
  for (int j = threadIdx.x; j < ids.k; j += kThreads) {
    const int64_t id = id_at(ids, r, j);
    out.logp[r * ids.k + j] =
      id < 0 || id >= in.n ? 0.f : log_prob(static_cast<float>(row[id]), o, in.temperature);
  }
  if constexpr (kTop) {
    top.compact(0);
    if (lane == 0) counts[wave] = top.n;
    __syncthreads();
    merge_lists(lists, counts, kWaves, out.top);
    if (wave == 0 && lane < out.top) {
      const bool bad  = isnan(o.lse);
      const int n     = bad ? 0 : min(counts[0], out.top);
      const key64 key = lane < n ? lists[lane] : 0;
      int rank        = lane;
      if (lane < n) {
        rank = 0;
        for (int j = 0; j < n; ++j)
          rank += lists[j] > key;
      }
      const int64_t at    = r * out.top + rank;
      out.top_logp[at] = lane < n ? log_prob(value_of(key), o, in.temperature) : (bad ? o.lse : -INFINITY);
      out.top_ids[at]  = lane < n ? column_of(key) : -1;
    }
  }
}

// ---- the teacher's distribution: the first wavefront's work, kListed entries a lane

constexpr int kListed = kMaxListed / 64;

struct teacher_row {
  int id[kListed];        // -1: not listed
  float z[kListed];       // teacher / T, -inf where not listed
  float top, ln_w;        // the largest z; ln sum exp(z - top)
  bool some;              // whether an entry has a probability
};

__device__ inline auto wave_max(float v) -> float
{
#pragma unroll
  for (int mask = 32; mask > 0; mask >>= 1)
    v = fmaxf(v, __shfl_xor(v, mask));
  return v;
}

__device__ inline auto wave_sum(float v) -> float
{
#pragma unroll
  for (int mask = 32; mask > 0; mask >>= 1)
    v += __shfl_xor(v, mask);
  return v;
}

__device__ inline auto read_teacher(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, int64_t r)
  -> teacher_row
{
  const int lane = threadIdx.x % 64;
  teacher_row t;
  float top = -INFINITY, bad = 0.f;
#pragma unroll
  for (int q = 0; q < kListed; ++q) {
    t.id[q] = -1;
    t.z[q]  = -INFINITY;
    const int j = lane + 64 * q;
    if (64 * q < ids.k && j < ids.k) {
      const int64_t id = id_at(ids, r, j);
      if (id >= 0 && id < in.n) {
        t.id[q] = static_cast<int>(id);
        t.z[q]  = load_any(teacher.x, teacher.type, r * teacher.stride + j) / in.temperature;
        top     = fmaxf(top, t.z[q]);
        if (isnan(t.z[q])) bad = t.z[q];
      }
    }
  }
  t.top  = wave_max(top);
  bad    = wave_sum(bad);
  t.some = t.top != -INFINITY || isnan(bad);
  float w = 0.f;
#pragma unroll
  for (int q = 0; q < kListed; ++q)
    if (64 * q < ids.k && t.id[q] >= 0 && t.z[q] != -INFINITY) w += expf(t.z[q] - t.top);
  t.ln_w = logf(wave_sum(w));
  return t;
}

__device__ inline auto teacher_log_q(teacher_row const& t, int q) -> float { return t.z[q] - t.top - t.ln_w; }

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_kernel(score_rows in, listed_ids ids, teacher_logits teacher,
                                                           float* loss, float* lse, int64_t row0)
{
  __shared__ run parts[kWaves];
  const int64_t r = row0 + blockIdx.x;
  const T* row    = static_cast<const T*>(in.x) + r * in.stride;
  const float c   = kLog2e / in.temperature;
  run sums        = nothing();
  for_scores<T>(row, 0, in.n, [&](const auto& v, int) { add_scores<false>(sums, v, c); });
  const auto o = finish(join_block(sums, c, parts), in.temperature);
  if (threadIdx.x >= 64) return;
  const auto t = read_teacher(in, ids, teacher, r);
  float sum    = 0.f;
#pragma unroll
  for (int q = 0; q < kListed; ++q) {
    if (64 * q >= ids.k || t.id[q] < 0 || t.z[q] == -INFINITY) continue;
    const float lq = teacher_log_q(t, q), p = expf(lq);
    if (p != 0.f) sum += p * (lq - log_prob(static_cast<float>(row[t.id[q]]), o, in.temperature));
  }
  sum = wave_sum(sum);
  if (threadIdx.x == 0) {
    loss[r] = t.some ? sum : 0.f;
    lse[r]  = o.lse;
  }
}

// ---- gradients

constexpr float kMaxLse = 100.f;

/** What a row's gradient needs: p = 2^((x - ref) c - l2), dx = p (a + b ln p). */
struct gradient_row {
  float ref, c, l2, a, b;
};

template <bool kEntropy>
__device__ inline auto gradient(float x, gradient_row const& g) -> float
{
  const float u = fmaf(x - g.ref, g.c, -g.l2), p = exp2_fast(u);
  if constexpr (kEntropy) return p * fmaf(g.b * kLn2, fmaxf(u, kFloor), g.a);
  return p * g.a;
}

/** Writes the gradient of columns [c0, c1), then that of the listed ids among them again with their shares w.  ids and w
 * are LDS; an id that is listed more than once gets the sum of its shares, in their order. */
template <typename T, bool kEntropy>
__device__ inline void write_gradient(const T* row, T* grad, int c0, int c1, gradient_row const& g, const int* ids,
                                      const float* w, int k)
{
  constexpr int N = kPer16<T>;
  float v[N];
  if (c1 - c0 < N) {
    const int at = c0 + static_cast<int>(threadIdx.x);
    if (at < c1) grad[at] = static_cast<T>(gradient<kEntropy>(static_cast<float>(row[at]), g));
  } else {
    const int last = c1 - N;
    for (int at0 = c0 + static_cast<int>(threadIdx.x) * N; at0 < c1; at0 += kThreads * N) {
      const int at = min(at0, last);  // the moved-back lane writes what its neighbor writes
      unpack16<T>(load16(row + at), v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = gradient<kEntropy>(v[i], g);
      store16(grad + at, pack16<T>(v));
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const int id = ids[j];
    if (id < c0 || id >= c1) continue;
    bool first = true;
    for (int i = 0; i < j && first; ++i)
      first = ids[i] != id;
    if (!first) continue;
    float sum = 0.f;
    for (int i = j; i < k; ++i)
      if (ids[i] == id) sum += w[i];
    grad[id] = static_cast<T>(gradient<kEntropy>(static_cast<float>(row[id]), g) + sum);
  }
}

/** A gradient of 0 in columns [c0, c1). */
template <typename T>
__device__ inline void write_zeros(T* grad, int c0, int c1)
{
  constexpr int N = kPer16<T>;
  if (c1 - c0 < N) {
    const int at = c0 + static_cast<int>(threadIdx.x);
    if (at < c1) grad[at] = static_cast<T>(0.f);
    return;
  }
  for (int at = c0 + static_cast<int>(threadIdx.x) * N; at < c1; at += kThreads * N)
    store16(grad + min(at, c1 - N), uint4{0, 0, 0, 0});
}

/**
 * ref, c and l2 of a row from its saved log-sum-exp; a row with nothing has p = 0 everywhere.  An l of more than kMaxLse
 * has lost too much of ln s to its rounding (all of it in a row of the type's lowest values), so such a row's sums are made
 * again.  All threads call this; parts [kWaves] is LDS.
 */
template <typename T>
__device__ inline auto gradient_base(const T* row, int n, float lse, float temperature, run* parts) -> gradient_row
{
  gradient_row g{};
  g.c  = kLog2e / temperature;
  g.l2 = lse == -INFINITY ? INFINITY : lse * kLog2e;
  if (fabsf(lse) > kMaxLse && fabsf(lse) != INFINITY) {
    run sums = nothing();
    for_scores<T>(row, 0, n, [&](const auto& v, int) { add_scores<false>(sums, v, g.c); });
    sums  = join_block(sums, g.c, parts);
    g.ref = sums.ref;
    g.l2  = log2f(sums.s);
  }
  return g;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void log_probs_backward_kernel(score_rows in, listed_ids ids, const float* grad_logp,
                                                                      const float* grad_entropy, const float* lse,
                                                                      const float* entropy, T* grad, int64_t gstride,
                                                                      int64_t row0)
{
  __shared__ int listed[kMaxListed];
  __shared__ float w[kMaxListed];
  __shared__ float total;
  __shared__ run parts[kWaves];
  const int64_t r = row0 + blockIdx.x;
  if (threadIdx.x < 64) {
    float sum = 0.f;
    for (int j = threadIdx.x; j < ids.k; j += 64) {
      const int64_t id = id_at(ids, r, j);
      const bool in_row = id >= 0 && id < in.n;
      const float gj    = in_row && grad_logp != nullptr ? grad_logp[r * ids.k + j] : 0.f;
      listed[j]         = in_row ? static_cast<int>(id) : -1;
      w[j]              = gj / in.temperature;
      sum += gj;
    }
    sum = wave_sum(sum);
    if (threadIdx.x == 0) total = sum;
  }
  __syncthreads();
  const float h = grad_entropy != nullptr ? grad_entropy[r] : 0.f;
  const T* row  = static_cast<const T*>(in.x) + r * in.stride;
  auto g        = gradient_base(row, in.n, lse[r], in.temperature, parts);
  g.a           = -(total + (h != 0.f ? h * entropy[r] : 0.f)) / in.temperature;
  g.b           = -h / in.temperature;
  write_gradient<T, true>(row, grad + r * gstride, 0, in.n, g, listed, w, ids.k);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_backward_kernel(score_rows in, listed_ids ids, teacher_logits teacher,
                                                                    const float* grad_loss, const float* lse, T* grad,
                                                                    int64_t gstride, int64_t row0)
{
  __shared__ int listed[kMaxListed];
  __shared__ float w[kMaxListed];
  __shared__ int some;
  __shared__ run parts[kWaves];
  const int64_t r = row0 + blockIdx.x;
  const float a   = grad_loss[r] / in.temperature;
  if (threadIdx.x < 64) {
    const auto t = read_teacher(in, ids, teacher, r);
#pragma unroll
    for (int q = 0; q < kListed; ++q) {
      const int j = threadIdx.x + 64 * q;
      if (64 * q >= ids.k || j >= ids.k) continue;
      listed[j] = t.id[q];
      w[j]      = t.id[q] >= 0 && t.z[q] != -INFINITY ? -a * expf(teacher_log_q(t, q)) : 0.f;
    }
    if (threadIdx.x == 0) some = t.some;
  }
  __syncthreads();
  grad += r * gstride;
  if (!some) {  // nothing to learn from
    write_zeros(grad, 0, in.n);
    return;
  }
  const T* row = static_cast<const T*>(in.x) + r * in.stride;
  auto g       = gradient_base(row, in.n, lse[r], in.temperature, parts);
  g.a          = a;
  write_gradient<T, false>(row, grad, 0, in.n, g, listed, w, ids.k);
}

/** Calls f with a value of the element type. */
template <typename F>
void with_type(elem type, F f)
{
  if (type == elem::f32)
    f(float{});
  else if (type == elem::f16)
    f(f16{});
  else
    f(bf16{});
}

/** Calls f(first row, rows) for parts of m rows whose grids of a workgroup a row have less than 2^32 work-items. */
template <typename F>
void for_row_grids(int64_t m, F f)
{
  constexpr int64_t kRows = (int64_t{1} << 32) / kThreads - 1;
  for (int64_t r = 0; r < m; r += kRows)
    f(r, static_cast<unsigned>(std::min(kRows, m - r)));
}

}  // namespace

void launch_log_probs(score_rows const& in, listed_ids const& ids, log_probs_out const& out, hipStream_t s)
{
  with_type(in.type, [&](auto e) {
    using T = decltype(e);
    for_row_grids(in.m, [&](int64_t row0, unsigned rows) {
      if (out.top > 0)
        log_probs_kernel<T, true><<<rows, kThreads, 0, s>>>(in, ids, out, row0);
      else
        log_probs_kernel<T, false><<<rows, kThreads, 0, s>>>(in, ids, out, row0);
      OCTEX_HIP(hipGetLastError());
    });
  });
}

void launch_log_probs_backward(score_rows const& in, listed_ids const& ids, const float* grad_logp,
                               const float* grad_entropy, const float* lse, const float* entropy, void* grad,
                               int64_t gstride, hipStream_t s)
{
  with_type(in.type, [&](auto e) {
    using T = decltype(e);
    for_row_grids(in.m, [&](int64_t row0, unsigned rows) {
      log_probs_backward_kernel<T><<<rows, kThreads, 0, s>>>(in, ids, grad_logp, grad_entropy, lse, entropy,
                                                             static_cast<T*>(grad), gstride, row0);
      OCTEX_HIP(hipGetLastError());
    });
  });
}

void launch_distill(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, float* loss, float* lse,
                    hipStream_t s)
{
  with_type(in.type, [&](auto e) {
    using T = decltype(e);
    for_row_grids(in.m, [&](int64_t row0, unsigned rows) {
      distill_kernel<T><<<rows, kThreads, 0, s>>>(in, ids, teacher, loss, lse, row0);
      OCTEX_HIP(hipGetLastError());
    });
  });
}

void launch_distill_backward(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher,
                             const float* grad_loss, const float* lse, void* grad, int64_t gstride, hipStream_t s)
{
  with_type(in.type, [&](auto e) {
    using T = decltype(e);
    for_row_grids(in.m, [&](int64_t row0, unsigned rows) {
      distill_backward_kernel<T><<<rows, kThreads, 0, s>>>(in, ids, teacher, grad_loss, lse, static_cast<T*>(grad),
                                                           gstride, row0);
      OCTEX_HIP(hipGetLastError());
    });
  });
}

}  // namespace cuvs::neighbors::octex::detail
