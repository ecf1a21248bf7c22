// Device code that the operators on rows of scores share (rows.hip, policy.hip; balance.hip takes its reductions over lanes):
// the sums of a row's exponentials, their joins over lanes and workgroups, one pass over a row, one that writes a gradient, and
// how rows are shared out.  Every file that includes it has its own.
#pragma once

#include "common.hpp"
#include "elems_device.hpp"
#include "rows.hpp"

#include <algorithm>
#include <cfloat>

namespace cuvs::neighbors::octex::detail {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2   = 0.693147180559945309417f;
constexpr float kFloor = -200.f;  // an exponent whose power of two is 0; keeps 0 * -inf out of the sums
constexpr int kThreads = 256;
constexpr int kWaves   = kThreads / 64;

using key64 = unsigned long long;

__device__ inline auto exp2_fast(float v) -> float { return __builtin_amdgcn_exp2f(v); }

/** The running sums of a part of a row; ref is m, or 0 while there is no finite score. */
struct run {
  float m, ref, s, t;
};

__device__ inline auto nothing() -> run { return {-INFINITY, 0.f, 0.f, 0.f}; }

/** The sums of a thread that may add many: those of a few scores, folded from time to time into s_all and t_all (by the largest
 * score at the last fold, m_all); s_low and t_low are what these additions have lost. */
struct long_run : run {
  float m_all, s_all, s_low, t_all, t_low;

  template <bool kEntropy>
  __device__ void fold(float c)
  {
    if (m > m_all) {
      const float d = fmaxf((m_all - m) * c, kFloor), f = exp2_fast(d);
      if constexpr (kEntropy) {
        t_all = (t_all + s_all * d) * f;
        t_low = (t_low + s_low * d) * f;
      }
      s_all *= f;
      s_low *= f;
      m_all = m;
    }
    add_kept(s_all, s_low, s);
    s = 0.f;
    if constexpr (kEntropy) {
      add_kept(t_all, t_low, t);
      t = 0.f;
    }
  }

  /** The sums of folded scores. */
  __device__ auto whole() const -> run { return {m, ref, s_all + s_low, t_all + t_low}; }

 private:
  /** sum += v; low takes what that loses (exactly while |v| is at most |sum|, which all but a row's first few are). */
  __device__ static void add_kept(float& sum, float& low, float v)
  {
    const float to = sum + v;
    low += v - (to - sum);
    sum = to;
  }
};

__device__ inline auto nothing_long() -> long_run { return {nothing(), -INFINITY, 0.f, 0.f, 0.f, 0.f}; }

/** Adds N scores, to each other first; returns their largest.  One by one to a large sum, equal terms round alike: a row of
 * 4,000,000 columns would be off by 1e-4. */
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
  float s, t;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float u = (v[i] - r.ref) * c, e = exp2_fast(u);
    s = i == 0 ? e : s + e;
    if constexpr (kEntropy) t = i == 0 ? e * fmaxf(u, kFloor) : fmaf(e, fmaxf(u, kFloor), t);
  }
  r.s += s;
  if constexpr (kEntropy) r.t += t;
  return cm;
}

// Reductions over groups of W lanes without LDS: a lane meets lanes that hold the other halves' results, and as f(a, b) is
// f(b, a) every lane ends with the same.  (By shuffles through LDS both directions of distill took 7 % longer for 4096 x
// 128,000 bfloat16, 24 % for 16 x 32,000 float32.)

template <int kControl>
__device__ inline auto from_lane(float v) -> float
{
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, 15, 15, true));
}

template <int W, typename F>
__device__ inline auto reduce_lanes(float v, F f) -> float
{
  if constexpr (W > 1) v = f(v, from_lane<0xb1>(v));   // lane ^ 1
  if constexpr (W > 2) v = f(v, from_lane<0x4e>(v));   // lane ^ 2
  if constexpr (W > 4) v = f(v, from_lane<0x141>(v));  // 7 - lane of 8
  if constexpr (W > 8) v = f(v, from_lane<0x140>(v));  // 15 - lane of 16
  if constexpr (W > 16) {
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v               = f(__uint_as_float(both[0]), __uint_as_float(both[1]));
  }
  if constexpr (W > 32) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v               = f(__uint_as_float(both[0]), __uint_as_float(both[1]));
  }
  return v;
}

template <int W = 64>
__device__ inline auto sum_lanes(float v) -> float
{
  return reduce_lanes<W>(v, [](float a, float b) { return a + b; });
}

/** The sums of W lanes' parts. */
template <int W, bool kEntropy>
__device__ inline auto join_lanes(run const& a, float c) -> run
{
  run r         = nothing();
  r.m           = reduce_lanes<W>(a.m, [](float x, float y) { return fmaxf(x, y); });
  r.ref         = r.m == -INFINITY ? 0.f : r.m;
  const float d = fmaxf((a.m - r.ref) * c, kFloor), f = exp2_fast(d);
  r.s           = sum_lanes<W>(a.s * f);
  if constexpr (kEntropy) r.t = sum_lanes<W>((a.t + a.s * d) * f);
  return r;
}

/** The whole workgroup's sums, the same in every thread; parts is LDS, one a wavefront. */
template <int NT, bool kEntropy>
__device__ inline auto join_block(run r, float c, run* parts) -> run
{
  r = join_lanes<64, kEntropy>(r, c);
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = r;
  lds_barrier();
  return join_lanes<NT / 64, kEntropy>(parts[threadIdx.x % (NT / 64)], c);
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

// ---- one pass over a row

constexpr int kRun    = 8;  // scores that a thread takes at a time: 16 bytes, of fp32 two times 16
constexpr int kPieces = 4;  // of 16 bytes, that a thread has on their way
/** Rounds of such loads whose sums are folded at a time: 64 or 128 scores, which lose 13 e (e = 2^-24) at most.  Both sums and
 * the 20 best of 4096 x 128,000 bfloat16: 207 us (never folded 205, after every round 214). */
constexpr int kFoldRounds = 4;

template <typename T>
struct run_bytes {
  uint4 raw[kRun / kPer16<T>];
};

template <typename T>
__device__ inline auto load_run(const T* p) -> run_bytes<T>
{
  run_bytes<T> r;
#pragma unroll
  for (int i = 0; i < kRun / kPer16<T>; ++i)
    r.raw[i] = load16(p + i * kPer16<T>);
  return r;
}

template <typename T>
__device__ inline void unpack_run(run_bytes<T> const& r, float (&v)[kRun])
{
#pragma unroll
  for (int i = 0; i < kRun / kPer16<T>; ++i) {
    float e[kPer16<T>];
    unpack16<T>(r.raw[i], e);
#pragma unroll
    for (int j = 0; j < kPer16<T>; ++j)
      v[i * kPer16<T> + j] = e[j];
  }
}

/** Calls f(v, at) for the scores of columns [c0, c1) that this thread takes, 8 at a time in ascending order; a score outside
 * the range, or one that another thread takes, comes as -inf.  Every lane of a wavefront calls f alike.  start(largest) is
 * called before, by all threads, with the largest of some of the thread's scores (-inf: none), none of them another's too;
 * fold() after every few rounds of f's, and at the end. */
template <typename T, int NT, typename G, typename F, typename H>
__device__ inline void for_scores(const T* row, int c0, int c1, G start, F f, H fold)
{
  constexpr int N = kRun, kAhead = kPieces * kPer16<T> / kRun;
  float v[N];
  if (c1 - c0 < N) {
    const int at = c0 + static_cast<int>(threadIdx.x);
#pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = -INFINITY;
    if (at < c1) v[0] = static_cast<float>(row[at]);
    start(v[0]);
    f(v, at);
    fold();
    return;
  }
  const int last = c1 - N;  // a load that would pass the range's end is moved back to it
  const int wave = c0 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64 * N;
  const int mine = static_cast<int>(threadIdx.x % 64) * N;
  constexpr int kStep = NT * N;
  run_bytes<T> next[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    next[u] = load_run(row + min(wave + u * kStep + mine, last));
  float largest = -INFINITY;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    if (wave + u * kStep + 64 * N > c1) break;  // this run's scores would not be its own
    unpack_run<T>(next[u], v);
#pragma unroll
    for (int i = 0; i < N; ++i)
      largest = fmaxf(largest, v[i]);
  }
  start(largest);
  int round = 0;
  for (int w = wave; w < c1; w += kAhead * kStep) {
    run_bytes<T> cur[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      cur[u] = next[u];
    if (w + kAhead * kStep < c1) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        next[u] = load_run(row + min(w + (kAhead + u) * kStep + mine, last));
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int w0 = w + u * kStep;
      if (w0 >= c1) break;
      unpack_run<T>(cur[u], v);
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
    if (++round % kFoldRounds == 0) fold();
  }
  fold();
}

__device__ inline auto id_at(listed_ids const& ids, int64_t row, int j) -> int64_t
{
  const int64_t i = row * ids.stride + j;
  return ids.wide ? static_cast<const int64_t*>(ids.ids)[i] : static_cast<const int32_t*>(ids.ids)[i];
}

/** How rows are shared out: `parts` workgroups a row take `width` columns each. */
struct row_split {
  int parts, width;
};

/** What a workgroup found in its columns, for the row's last step. */
struct part_sums {
  float m, s, t;
};

__device__ inline auto as_run(part_sums const& p) -> run { return {p.m, p.m == -INFINITY ? 0.f : p.m, p.s, p.t}; }

/** The sums of all parts of row r (at most 64), the same in every lane of the calling wavefront. */
template <bool kEntropy>
__device__ inline auto join_parts(const part_sums* part, int64_t r, int parts, float c) -> run
{
  const int lane = threadIdx.x % 64;
  return join_lanes<64, kEntropy>(lane < parts ? as_run(part[r * parts + lane]) : nothing(), c);
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

/** The ids of a row's list (-1: not listed) and their shares of its gradient, k of them in LDS. */
struct listed_shares {
  int id[kMaxListed];
  float w[kMaxListed];
};

/** The list's entry of a lane's number, id -1 past the end. */
struct listed_share {
  int id;
  float w;
};

__device__ inline auto share_at(listed_shares const& s, int j, int k) -> listed_share
{
  return j < k ? listed_share{s.id[j], s.w[j]} : listed_share{-1, 0.f};
}

/**
 * Adds the shares of the list's ids to the gradients v of columns at + i, in the list's order; the wavefront's columns are
 * the 64 * N from w0 (a multiple of N) on that lie below end, and a lane whose own would pass the end has those from `last`
 * on.  first is the lane's of the first 64 entries.  So every gradient is stored once, by one thread, with no atomics: an id
 * that is listed twice gets the same sum in every run.
 *
 * A wavefront that has the whole list to itself (kAlone) meets many entries at a time: it takes them by their place among a
 * lane's columns, which is the same for all lanes but where some were moved back, at one addition each instead of N.
 * 8000 x 1000 float32 with 64 ids, distill's gradient: 23 us against 26; but 4096 x 128,000 bfloat16 in both directions,
 * where most pieces meet none, takes 3 % longer.
 */
template <bool kAlone, int N>
__device__ inline void add_shares(float (&v)[N], int at, int w0, int last, int end, listed_share first, listed_shares const& s,
                                  int k)
{
  const int lane = static_cast<int>(threadIdx.x % 64), lo = min(w0, last), hi = min(w0 + 64 * N, end);
  for (int q = 0; q < k; q += 64) {
    const listed_share mine = q == 0 ? first : share_at(s, q + lane, k);
    const key64 all         = __ballot(mine.id >= lo && mine.id < hi);
    if (all == 0) continue;
    if (kAlone && w0 + 64 * N <= end) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        for (key64 in = all & __ballot(mine.id % N == e); in != 0; in &= in - 1) {
          const int i = __builtin_ctzll(in), owner = (__builtin_amdgcn_readlane(mine.id, i) - w0) / N;
          const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine.w), i));
          v[e] += lane == owner ? w : 0.f;
        }
    } else {
      for (key64 in = all; in != 0; in &= in - 1) {
        const int i = __builtin_ctzll(in), column = __builtin_amdgcn_readlane(mine.id, i) - at;
        const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine.w), i));
#pragma unroll
        for (int e = 0; e < N; ++e)
          v[e] += column == e ? w : 0.f;
      }
    }
  }
}

/** Writes the gradient of columns [c0, c1), a thread 64 bytes while the next 64 are on their way.  prepare() gives what a
 * row needs, its list's shares in LDS and, in `some`, whether the gradient is other than 0; it may hold barriers, and runs
 * while the first scores are on their way. */
template <typename T, bool kEntropy, int NT, typename P>
__device__ inline void write_gradient(const T* row, T* grad, bool by_cache, int c0, int c1, listed_shares const& s, int k,
                                      P prepare)
{
  constexpr int N = kPer16<T>, kStep = NT * N;
  const bool tiny = c1 - c0 < N;
  const int last  = c1 - N;
  const int wave = c0 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64 * N;
  const int mine = static_cast<int>(threadIdx.x % 64) * N;
  uint4 next[kPieces];
  if (!tiny) {
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
      next[u] = load16(row + min(wave + u * kStep + mine, last));
  }
  bool some            = true;
  const gradient_row g = prepare(some);
  const listed_share first = share_at(s, static_cast<int>(threadIdx.x % 64), k);
  if (tiny) {
    const int at = c0 + static_cast<int>(threadIdx.x);
    float v[1]   = {0.f};
    if (at < c1 && some) v[0] = gradient<kEntropy>(static_cast<float>(row[at]), g);
    if (some) add_shares<NT == 64>(v, at, c0, c0, c1, first, s, k);
    if (at < c1) grad[at] = static_cast<T>(v[0]);
    return;
  }
  float v[N];
  for (int w = wave; w < c1; w += kPieces * kStep) {
    uint4 cur[kPieces];
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
      cur[u] = next[u];
    if (w + kPieces * kStep < c1) {
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
        next[u] = load16(row + min(w + (kPieces + u) * kStep + mine, last));
    }
#pragma unroll
    for (int u = 0; u < kPieces; ++u) {
      const int w0 = w + u * kStep;
      if (w0 >= c1) break;
      const int at = min(w0 + mine, last);  // a lane that was moved back writes what its neighbor does
      unpack16<T>(cur[u], v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = some ? gradient<kEntropy>(v[i], g) : 0.f;
      if (some) add_shares<NT == 64>(v, at, w0, last, c1, first, s, k);
      if (w0 + mine >= c1) continue;
      if (by_cache)
        store16(grad + at, pack16<T>(v));
      else
        store16_nt(grad + at, pack16<T>(v));
    }
  }
}

/**
 * ref, c and l2 of a row from its saved log-sum-exp l; a row with nothing has p = 0 everywhere.  With ref = l T the difference
 * x - ref is small where p is not, and p is as near as the fp32 l: 3.8e-6 of it at l = 98 (by x c - l log2(e), whose terms are
 * rounded apart, up to 6.0e-6 more).  An l of more than kMaxLse has lost too much of ln s to its rounding (all of it in a row
 * of the type's lowest values), so such a row's sums are made again.  That is so for infinite l too: a row of lowest values has
 * one at temperatures below 1, as a row of nothing has.  All threads call this; parts [NT / 64] is LDS.
 */
template <typename T, int NT>
__device__ inline auto gradient_base(const T* row, int n, float lse, float temperature, run* parts) -> gradient_row
{
  gradient_row g{};
  g.c   = kLog2e / temperature;
  g.ref = lse * temperature;
  g.l2  = fmaf(lse, temperature, -g.ref) / temperature * kLog2e;  // what that product lost
  if (fabsf(lse) > kMaxLse) {
    auto added = nothing_long();
    for_scores<T, NT>(row, 0, n, [](float) {}, [&](const auto& v, int) { add_scores<false>(added, v, g.c); },
                      [&] { added.fold<false>(g.c); });
    const run sums = join_block<NT, false>(added.whole(), g.c, parts);
    g.ref          = sums.ref;
    g.l2           = sums.s == 0.f ? INFINITY : log2f(sums.s);
  }
  return g;
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

/** Calls f(first, count) for parts of `total` workgroups whose grids have less than 2^32 work-items. */
template <typename F>
void for_grids(int64_t total, int threads, F f)
{
  const int64_t most = (int64_t{1} << 32) / threads - 1;
  for (int64_t first = 0; first < total; first += most)
    f(first, static_cast<unsigned>(std::min(most, total - first)));
}

constexpr int kEnough   = 1024;  // workgroups of 256 threads that fill the GPU
constexpr int kMinWidth = 4096;  // columns of a part
constexpr int kMaxParts = 32;    // of a row

/** The longest list of ids that a single wavefront takes. */
constexpr int kShortList = 128;

/** Rows are split into parts of whole 16-byte pieces while they are fewer than the workgroups that fill the GPU. */
inline auto split_of(int64_t m, int n, int64_t most = kMaxParts) -> row_split
{
  const int64_t want = std::min<int64_t>({kEnough / std::min<int64_t>(m, kEnough), (n + kMinWidth - 1) / kMinWidth, most});
  if (want <= 1) return {1, n};
  const int width = static_cast<int>((n + want - 1) / want + 63) / 64 * 64;
  return {(n + width - 1) / width, width};
}

/** Up to kFewRows rows of kWideRow columns or more are split in a forward pass, at a second launch (and a workspace, 4 us of
 * a caller's time): 16 x 128,000 bfloat16 in 5.6 us against 16.7 whole, with the 20 best 12.5 against 25; 128 rows in 12.6
 * against 17.3, but 256 in 17.5 either way and with the 20 best in 30 against 27; 16 x 32,000 in 5.1 against 6.1, with the 20
 * best 12.8 against 11.1. */
constexpr int kFewRows = 128, kWideRow = 65536;

/** Of a forward pass, whose parts' best entries are at most four a thread of the kernel that joins them. */
inline auto forward_split_of(int64_t m, int n, int top) -> row_split
{
  if (m > kFewRows || n < kWideRow) return {1, n};
  return split_of(m, n, std::min(kMaxParts, 4 * kThreads / std::max(top, 1)));
}

/** Whether a gradient is stored through the caches: one of up to half of the last-level cache's 256 MB, that its reader may
 * find there.  A larger one would drive out the logits that a forward pass has left there (4096 x 32,000
 * bfloat16, both directions of log_probs: 135 us in place of 165). */
inline auto passes_cache(score_rows const& in) -> bool { return in.m * in.n * elem_size(in.type) <= int64_t{128} << 20; }

/** Rows of few columns take a wavefront each where there are enough of them. */
inline auto by_wavefront(int64_t m, int n, int k) -> bool { return m >= 2048 && n <= 4096 && k <= kShortList; }

}  // namespace

}  // namespace cuvs::neighbors::octex::detail
