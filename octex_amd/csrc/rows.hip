// Operators on rows of scores: a row holds one query's (or token's) n logits x, read as z = x / T.
//
//   log_probs   l = ln sum exp z;  log p_v = z_v - l of the given ids;  H = l - sum p z;  the top entries by (value, id)
//   distill     q = softmax(teacher / T) over the listed ids;  loss = sum q_j (ln q_j - log p_{id_j})
//   backward    dx_v = p_v (A + B ln p_v) + sum over the listed j with id_j = v of w_j, with
//               log_probs: A = -(sum g + h H) / T, B = -h / T, w = g / T;  distill: A = g / T, B = 0, w = -g q / T
//
// One pass over a row holds, a thread, the running maximum m, s = sum 2^u and t = sum 2^u u with u = (x - m) log2(e) / T:
// then l = m / T + ln s and H = ln s - ln 2 t / s, a difference of small numbers.  All sums are fp32, in a fixed order, and
// keep what their additions lose, so that their error does not grow with the row.
// A row without a finite score has p = 0 everywhere: l = -inf, H = 0, log p = -inf.  A NaN or +inf makes its row NaN.
//
// All of it is bound by the logits' bytes: a large copy takes 4.77 TB/s of this GPU, a kernel that only reads up to 5.5.
// The times below are a launch's among others of its kind, its inputs changing from launch to launch; "TB/s" counts the logits,
// and a gradient, once.  Two sides of a choice were timed together, some before later steps made both quicker.

#include "rows_device.hpp"

namespace cuvs::neighbors::octex::detail {

namespace {

constexpr int kList    = 256;  // a wavefront's candidate keys: four a lane
constexpr int kFull    = 128;  // keys from which a list is compacted
/** New keys of a call that are listed column by column; more of them are quicker one of every lane at a time.  2048 x 128,000
 * bfloat16, top 20: 117 us (all one a lane: 135); 8000 x 1000 float32: 18 us (all column by column: 20). */
constexpr int kSparse = 8;

// ---- the top entries: a wavefront's list of keys (order of the value, ~column), compacted when it fills
//
// A score is compared with a floor that only grows, so that the pass costs one comparison a score and a few entries: the
// first floor is one that k of the workgroup's threads reach with their first scores, and later ones come from a full list.
// Floors are found bit by bit from counts of the lanes that reach them, without sorting; only the last 64 keys are ranked.

__device__ inline auto order_of(float v) -> unsigned
{
  const unsigned b = __float_as_uint(v + 0.f);  // -0 and 0 are one value
  return b >> 31 ? ~b : b | 0x80000000u;
}

__device__ inline auto key_of(float v, int column) -> key64
{
  return key64{order_of(v)} << 32 | static_cast<unsigned>(~column);
}

__device__ inline auto value_of_order(unsigned o) -> float { return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ inline auto value_of(key64 k) -> float { return value_of_order(static_cast<unsigned>(k >> 32)); }
__device__ inline auto column_of(key64 k) -> int { return static_cast<int>(~static_cast<unsigned>(k)); }

/** A floor that at least k and, unless equal values forbid it, at most `most` of the wavefront's values reach, as orders
 * (0: none); 0 if there are not k. */
template <int N>
__device__ inline auto floor_of(const unsigned (&order)[N], int k, int most) -> unsigned
{
  unsigned p = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned q = p | 1u << bit;
    int c            = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      c += __popcll(__ballot(order[j] >= q));
    if (c >= k) {
      p = q;
      if (c <= most) break;
    }
  }
  return p;
}

/** The same for distinct keys, which leave at most `most`. */
template <int N>
__device__ inline auto floor_of(const key64 (&key)[N], int k, int most) -> key64
{
  unsigned order[N];
#pragma unroll
  for (int j = 0; j < N; ++j)
    order[j] = static_cast<unsigned>(key[j] >> 32);
  key64 p = key64{floor_of(order, k, most)} << 32;
  if (p == 0) return 0;
  int c = 0;
#pragma unroll
  for (int j = 0; j < N; ++j)
    c += __popcll(__ballot(key[j] >= p));
  for (int bit = 31; bit >= 0 && c > most; --bit) {  // equal values: by column
    const key64 q = p | key64{1} << bit;
    int d         = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      d += __popcll(__ballot(key[j] >= q));
    if (d >= k) p = q, c = d;
  }
  return p;
}

/** A score and its column, as they come. */
struct entry {
  unsigned column;
  float v;
};

__device__ inline auto lanes_below(key64 lanes) -> int
{
  return __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(lanes >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(lanes), 0));
}

struct top_list {
  entry* list;  // [kList] in LDS, this wavefront's
  int k;
  int n     = 0;
  float low = -FLT_MAX;  // no later score below it is among the k best

  /** The first floor: at least k of the workgroup's threads have a score cm that reaches it, and few more.  orders is LDS,
   * one a thread. */
  template <int NT>
  __device__ void start(float cm, unsigned* orders)
  {
    orders[threadIdx.x] = order_of(cm);
    lds_barrier();
    unsigned order[NT / 64];
#pragma unroll
    for (int j = 0; j < NT / 64; ++j)
      order[j] = orders[threadIdx.x % 64 + 64 * j];
    raise(floor_of(order, k, k + 8));
    lds_barrier();
  }

  /** The list's keys, 0 past its end. */
  __device__ void read(key64 (&key)[4]) const
  {
    const int lane = threadIdx.x % 64;
    wave_fence();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const entry e = list[lane + 64 * j];
      key[j]        = lane + 64 * j < n ? key_of(e.v, static_cast<int>(e.column)) : 0;
    }
    wave_fence();
  }

  /** Keeps the k best entries and at most 32 others.  Returns the order of a score that k of them reach (0: none). */
  __device__ auto compact() -> unsigned
  {
    key64 key[4];
    read(key);
    const key64 p = floor_of(key, k, k + 32);
    n             = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in  = key[j] != 0 && key[j] >= p;
      const key64 at = __ballot(in);
      if (in) list[n + lanes_below(at)] = {static_cast<unsigned>(column_of(key[j])), value_of(key[j])};
      n += __popcll(at);
    }
    return static_cast<unsigned>(p >> 32);
  }

  __device__ void raise(unsigned order)
  {
    // below: not a number's order; above: infinity's, in a row that has no alternatives anyway
    if (order >= 0x00800000u && order < 0xff800000u) low = fmaxf(low, value_of_order(order));
  }

  /** Scores v of columns at + i, above every column of earlier calls; cm is the lane's largest. */
  template <int N>
  __device__ void add(const float (&v)[N], float cm, int at)
  {
    if (__ballot(cm >= low) == 0) return;
    key64 reach[N];
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      reach[i] = __ballot(v[i] >= low);
      count += __popcll(reach[i]);
    }
    if (count <= kSparse && n + count <= kFull) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (reach[i] == 0) continue;
        if (v[i] >= low) list[n + lanes_below(reach[i])] = {static_cast<unsigned>(at + i), v[i]};
        n += __popcll(reach[i]);
      }
      return;
    }
    unsigned left = 0;  // of this lane's scores
#pragma unroll
    for (int i = 0; i < N; ++i)
      left |= v[i] >= low ? 1u << i : 0u;
    unsigned floor = 0;
    while (__ballot(left != 0) != 0) {  // every lane lists one
      const int i = __ffs(static_cast<int>(left)) - 1;
      float x     = v[0];
#pragma unroll
      for (int j = 1; j < N; ++j)
        x = i == j ? v[j] : x;
      // equal scores of lower columns may come in this very call, so a floor it raised lets them in
      const bool in     = left != 0 && x >= low;
      const key64 lanes = __ballot(in);
      if (in) list[n + lanes_below(lanes)] = {static_cast<unsigned>(at + i), x};
      n += __popcll(lanes);
      left &= left - 1;
      if (n > kFull) {
        floor = compact();
        raise(floor);
      }
    }
    if (floor != 0) raise(floor + 1);  // k scores of lower columns reach it: an equal one comes too late
  }
};

/** The wavefronts' keys (0: none; `mine` of them here) that may be among the k best to keys (LDS, [waves * 64]), dense.
 * Returns their number. */
template <int NT>
__device__ inline auto gather_keys(const key64 (&key)[4], int mine, int k, key64* keys, int* counts) -> int
{
  const int wave = threadIdx.x / 64;
  const key64 p  = mine <= 64 ? 1 : floor_of(key, k, 64);
  key64 in[4];
  mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    in[j] = __ballot(key[j] != 0 && key[j] >= p);
    mine += __popcll(in[j]);
  }
  if (threadIdx.x % 64 == 0) counts[wave] = mine;
  lds_barrier();
  int from = 0, n = 0;
  for (int w = 0; w < NT / 64; ++w) {
    from += w < wave ? counts[w] : 0;
    n += counts[w];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (key[j] != 0 && key[j] >= p) keys[from + lanes_below(in[j])] = key[j];
    from += __popcll(in[j]);
  }
  lds_barrier();
  return n;
}

/** Calls f(rank, key) for the k best of n (at most 64 * R) distinct keys in LDS, which it leaves in another order; a key's rank
 * is the number of greater ones.  One wavefront's work. */
template <int R, typename F>
__device__ inline void rank_keys(key64* keys, int n, int k, F f)
{
  const int lane = threadIdx.x % 64;
  if (n > 64) {
    key64 key[R];
#pragma unroll
    for (int j = 0; j < R; ++j)
      key[j] = lane + 64 * j < n ? keys[lane + 64 * j] : 0;
    wave_fence();
    const key64 p = floor_of(key, k, 64);
    n             = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool in  = key[j] != 0 && key[j] >= p;
      const key64 at = __ballot(in);
      if (in) keys[n + lanes_below(at)] = key[j];
      n += __popcll(at);
    }
    wave_fence();
  }
  const key64 mine = lane < n ? keys[lane] : 0;
  int rank         = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j)
    rank += keys[j] > mine;
  if (lane < n && rank < k) f(rank, mine);
}

/** The outputs of row r but its alternatives. */
template <typename T, int NT>
__device__ inline void write_log_probs(score_rows const& in, listed_ids const& ids, log_probs_out const& out, int64_t r,
                                       row_sums const& o)
{
  if (threadIdx.x == 0) {
    out.lse[r]     = o.lse;
    out.entropy[r] = o.entropy;
  }
  const T* row = static_cast<const T*>(in.x) + r * in.stride;
  for (int j = threadIdx.x; j < ids.k; j += NT) {
    const int64_t id        = id_at(ids, r, j);
    out.logp[r * ids.k + j] = id < 0 || id >= in.n ? 0.f : log_prob(static_cast<float>(row[id]), o, in.temperature);
  }
}

/** The alternatives of row r: the best of n keys in LDS.  The first wavefront's work. */
template <int R>
__device__ inline void write_top(score_rows const& in, log_probs_out const& out, int64_t r, row_sums const& o, key64* keys,
                                 int n)
{
  const int lane = static_cast<int>(threadIdx.x);
  if (lane >= 64) return;
  const bool bad = isnan(o.lse);
  const int have = bad ? 0 : min(n, out.top);
  rank_keys<R>(keys, bad ? 0 : n, out.top, [&](int rank, key64 key) {
    out.top_logp[r * out.top + rank] = log_prob(value_of(key), o, in.temperature);
    out.top_ids[r * out.top + rank]  = column_of(key);
  });
  if (lane >= have && lane < out.top) {
    out.top_logp[r * out.top + lane] = bad ? o.lse : -INFINITY;
    out.top_ids[r * out.top + lane]  = -1;
  }
}

/**
 * A workgroup a row, or with kSplit a workgroup a part of a row, which leaves its sums and its best keys (0: none) to
 * finish_log_probs_kernel.  One pass: a thread has 64 bytes on their way while it adds and lists 64 others.
 *
 * 4096 x 128,000 bfloat16: 186 us, 5.6 TB/s; with the 20 best 207 us, 5.1 TB/s, the first floors and the lists' ends being
 * what is not hidden (2048 rows: 95 and 115).  1 x 128,000, in two launches: 4.9 us, with the 20 best 11.2.
 */
template <typename T, int NT, bool kTop, bool kSplit>
__global__ __launch_bounds__(NT) void log_probs_kernel(score_rows in, listed_ids ids, log_probs_out out,
                                                             row_split split, part_sums* part, key64* best, int64_t row0)
{
  constexpr int kWavesHere = NT / 64;
  __shared__ run parts[kWavesHere];
  __shared__ entry lists[kTop ? kWavesHere * kList : 1];
  __shared__ key64 keys[kTop ? kWavesHere * 64 : 1];
  __shared__ int counts[kWavesHere];
  const int64_t b = row0 + blockIdx.x, r = kSplit ? b / split.parts : b;
  const int c0 = kSplit ? static_cast<int>(b - r * split.parts) * split.width : 0;
  const int c1 = kSplit ? min(c0 + split.width, in.n) : in.n;
  const T* row = static_cast<const T*>(in.x) + r * in.stride;
  const float c = kLog2e / in.temperature;
  auto sums     = nothing_long();
  top_list top{lists + (kTop ? threadIdx.x / 64 * kList : 0), out.top};
  for_scores<T, NT>(
    row, c0, c1,
    [&](float cm) {
      if constexpr (kTop) top.start<NT>(cm, reinterpret_cast<unsigned*>(keys));
    },
    [&](const auto& v, int at) {
      const float cm = add_scores<true>(sums, v, c);
      if constexpr (kTop) top.add(v, cm, at);
    },
    [&] { sums.fold<true>(c); });
  const run all = join_block<NT, true>(sums.whole(), c, parts);
  int n         = 0;
  if constexpr (kTop) {
    key64 key[4];
    top.read(key);
    n = gather_keys<NT>(key, top.n, out.top, keys, counts);
  }
  if constexpr (kSplit) {
    if (threadIdx.x == 0) part[b] = {all.m, all.s, all.t};
    if constexpr (kTop) {
      if (threadIdx.x < 64) {
        rank_keys<kWavesHere>(keys, n, out.top, [&](int rank, key64 key) { best[b * out.top + rank] = key; });
        if (static_cast<int>(threadIdx.x) >= n && static_cast<int>(threadIdx.x) < out.top) best[b * out.top + threadIdx.x] = 0;
      }
    }
  } else {
    const auto o = finish(all, in.temperature);
    write_log_probs<T, NT>(in, ids, out, r, o);
    if constexpr (kTop) write_top<kWavesHere>(in, out, r, o, keys, n);
  }
}

template <typename T, bool kTop>
__global__ __launch_bounds__(kThreads) void finish_log_probs_kernel(score_rows in, listed_ids ids, log_probs_out out,
                                                                    row_split split, const part_sums* part,
                                                                    const key64* best, int64_t row0)
{
  __shared__ key64 keys[kTop ? kWaves * 64 : 1];
  __shared__ int counts[kWaves];
  const int64_t r = row0 + blockIdx.x;
  key64 key[4];
  if constexpr (kTop) {
    const int all = split.parts * out.top;  // at most 4 * kThreads
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = static_cast<int>(threadIdx.x) + kThreads * j;
      key[j]      = i < all ? best[r * all + i] : 0;
    }
  }
  const auto o = finish(join_parts<true>(part, r, split.parts, kLog2e / in.temperature), in.temperature);
  write_log_probs<T, kThreads>(in, ids, out, r, o);
  if constexpr (kTop) write_top<kWaves>(in, out, r, o, keys, gather_keys<kThreads>(key, 256, out.top, keys, counts));
}

// ---- the teacher's distribution: entry e of a thread is the row's entry threadIdx.x + e * NT

/** Entries a thread: all of a list but for a single wavefront, which takes lists of up to kShortList. */
template <int NT>
constexpr int kEntries = (NT == 64 ? kShortList : kMaxListed) / NT;

/** A thread's entries of a row's list: ids (-1: not listed), the teacher's logits (-inf where not listed; differences of them
 * are divided by T, as a quotient of the lowest value may pass fp32) and the student's scores. */
template <int E>
struct listed_part {
  int id[E];
  float z[E], x[E];
};

template <int NT, int E>
__device__ inline void read_list(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, int64_t r,
                                 listed_part<E>& l)
{
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = static_cast<int>(threadIdx.x) + e * NT;
    l.id[e]     = -1;
    l.z[e]      = -INFINITY;
    if (j < ids.k) {
      const int64_t id = id_at(ids, r, j);
      const float z    = load_any(teacher.x, teacher.type, r * teacher.stride + j);
      const bool in_row = id >= 0 && id < in.n;
      l.id[e]          = in_row ? static_cast<int>(id) : -1;
      l.z[e]           = in_row ? z : -INFINITY;
    }
  }
}

template <typename T, int E>
__device__ inline void read_listed(const T* row, listed_part<E>& l)
{
#pragma unroll
  for (int e = 0; e < E; ++e)
    l.x[e] = l.id[e] >= 0 ? static_cast<float>(row[l.id[e]]) : 0.f;
}

/** The sums of the thread's entries: a NaN entry makes them NaN. */
template <int E>
__device__ inline auto teacher_run(listed_part<E> const& l, float temperature) -> run
{
  run t = nothing();
#pragma unroll
  for (int e = 0; e < E; ++e)
    t.m = fmaxf(t.m, l.z[e]);
  t.ref = t.m == -INFINITY ? 0.f : t.m;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (l.z[e] != -INFINITY) t.s += expf((l.z[e] - t.ref) / temperature);
  return t;
}

/** A list's sums, for the ln q of its entries. */
struct teacher_sums {
  float top, ln_w, temperature;
  bool some;  // whether an entry has a probability
};

__device__ inline auto teacher_of(run const& t, float temperature) -> teacher_sums
{
  return {t.m, logf(t.s), temperature, t.s != 0.f};
}

__device__ inline auto ln_q(float z, teacher_sums const& t) -> float { return (z - t.top) / t.temperature - t.ln_w; }

/** The thread's share of a row's loss. */
template <int E>
__device__ inline auto loss_of(score_rows const& in, listed_part<E> const& l, teacher_sums const& t, row_sums const& o) -> float
{
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (l.z[e] == -INFINITY) continue;
    const float lq = ln_q(l.z[e], t), p = expf(lq);
    if (p != 0.f) sum += p * (lq - log_prob(l.x[e], o, in.temperature));
  }
  return sum;
}

/** join_block of a row's sums and of its list's at one barrier; both is LDS, two a wavefront. */
template <int NT>
__device__ inline void join_both(run& sums, float c, run& t, run* both)
{
  sums = join_lanes<64, false>(sums, c);
  if (__ballot(t.s != 0.f) != 0) t = join_lanes<64, false>(t, c);
  if (threadIdx.x % 64 == 0) {
    both[threadIdx.x / 64 * 2]     = sums;
    both[threadIdx.x / 64 * 2 + 1] = t;
  }
  lds_barrier();
  const int w = threadIdx.x % (NT / 64);
  sums        = join_lanes<NT / 64, false>(both[2 * w], c);
  t           = both[2 * w + 1];
  if (__ballot(t.s != 0.f) != 0) t = join_lanes<NT / 64, false>(t, c);
}

/** A pass over rows, a workgroup each, or with kSplit a workgroup a part of a row, which leaves its sums to
 * finish_distill_kernel.  The list's q needs no pass of its own: its logits are a few registers of the threads, and its sums
 * are joined at the row's barrier.  4096 x 128,000 bfloat16 with 64 ids a row: 190 us, 5.5 TB/s. */
template <typename T, int NT, bool kSplit>
__global__ __launch_bounds__(NT) void distill_kernel(score_rows in, listed_ids ids, teacher_logits teacher,
                                                     float* loss, float* lse, row_split split, part_sums* part,
                                                     int64_t row0)
{
  constexpr int E = kEntries<NT>;
  __shared__ run both[2 * NT / 64];
  __shared__ float losses[NT / 64];
  const int64_t b = row0 + blockIdx.x, r = kSplit ? b / split.parts : b;
  const int c0  = kSplit ? static_cast<int>(b - r * split.parts) * split.width : 0;
  const int c1  = kSplit ? min(c0 + split.width, in.n) : in.n;
  const T* row  = static_cast<const T*>(in.x) + r * in.stride;
  const float c = kLog2e / in.temperature;
  listed_part<E> l;
  if constexpr (!kSplit) read_list<NT>(in, ids, teacher, r, l);
  auto added = nothing_long();
  for_scores<T, NT>(row, c0, c1, [](float) {}, [&](const auto& v, int) { add_scores<false>(added, v, c); },
                    [&] { added.fold<false>(c); });
  run sums = added.whole();
  if constexpr (kSplit) {
    sums = join_block<NT, false>(sums, c, both);
    if (threadIdx.x == 0) part[b] = {sums.m, sums.s, 0.f};
  } else {
    read_listed(row, l);
    run list = teacher_run(l, in.temperature);
    join_both<NT>(sums, c, list, both);
    const auto o      = finish(sums, in.temperature);
    const float share = sum_lanes(loss_of(in, l, teacher_of(list, in.temperature), o));
    if (threadIdx.x % 64 == 0) losses[threadIdx.x / 64] = share;
    lds_barrier();
    if (threadIdx.x == 0) {
      float sum = losses[0];
      for (int w = 1; w < NT / 64; ++w)
        sum += losses[w];
      loss[r] = sum;
      lse[r]  = o.lse;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(64) void finish_distill_kernel(score_rows in, listed_ids ids, teacher_logits teacher,
                                                            float* loss, float* lse, row_split split,
                                                            const part_sums* part, int64_t row0)
{
  constexpr int E = kMaxListed / 64;
  const int64_t r = row0 + blockIdx.x;
  listed_part<E> l;
  read_list<64>(in, ids, teacher, r, l);
  const auto o = finish(join_parts<false>(part, r, split.parts, kLog2e / in.temperature), in.temperature);
  read_listed(static_cast<const T*>(in.x) + r * in.stride, l);
  const run list  = join_lanes<64, false>(teacher_run(l, in.temperature), kLog2e / in.temperature);
  const float sum = sum_lanes(loss_of(in, l, teacher_of(list, in.temperature), o));
  if (threadIdx.x == 0) {
    loss[r] = sum;
    lse[r]  = o.lse;
  }
}

// ---- gradients

/** The shares -a q of the thread's entries. */
template <int NT, int E>
__device__ inline void write_shares(listed_part<E> const& l, teacher_sums const& t, float a, int k, listed_shares& s)
{
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = static_cast<int>(threadIdx.x) + e * NT;
    if (j >= k) continue;
    s.id[j] = l.id[e];
    s.w[j]  = l.z[e] != -INFINITY ? -a * expf(ln_q(l.z[e], t)) : 0.f;
  }
}

/** A workgroup a row or a part of one: A and B of the row from its list and its saved sums, then one pass.  4096 x 128,000
 * bfloat16: 418 us, 5.0 TB/s; 4096 x 32,000, its logits still in the last-level cache: 81 us, 6.5 TB/s. */
template <typename T, int NT>
__global__ __launch_bounds__(NT) void log_probs_backward_kernel(score_rows in, listed_ids ids, const float* grad_logp,
                                                                      const float* grad_entropy, const float* lse,
                                                                      const float* entropy, T* grad, int64_t gstride,
                                                                      bool by_cache, row_split split, int64_t row0)
{
  constexpr int E = kEntries<NT>;
  __shared__ listed_shares shares;
  __shared__ float totals[NT / 64];
  __shared__ run parts[NT / 64];
  const int64_t b = row0 + blockIdx.x, r = b / split.parts;
  const int c0 = static_cast<int>(b - r * split.parts) * split.width, c1 = min(c0 + split.width, in.n);
  const T* row = static_cast<const T*>(in.x) + r * in.stride;
  write_gradient<T, true, NT>(row, grad + r * gstride, by_cache, c0, c1, shares, ids.k, [&](bool&) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = static_cast<int>(threadIdx.x) + e * NT;
      if (j >= ids.k) continue;
      const int64_t id  = id_at(ids, r, j);
      const bool in_row = id >= 0 && id < in.n;
      const float gj    = in_row && grad_logp != nullptr ? grad_logp[r * ids.k + j] : 0.f;
      shares.id[j]      = in_row ? static_cast<int>(id) : -1;
      shares.w[j]       = gj / in.temperature;
      sum += gj;
    }
    sum = sum_lanes(sum);
    if (threadIdx.x % 64 == 0) totals[threadIdx.x / 64] = sum;
    lds_barrier();
    float total = totals[0];
    for (int w = 1; w < NT / 64; ++w)
      total += totals[w];
    const float h = grad_entropy != nullptr ? grad_entropy[r] : 0.f;
    auto g        = gradient_base<T, NT>(row, in.n, lse[r], in.temperature, parts);
    g.a           = -(total + (h != 0.f ? h * entropy[r] : 0.f)) / in.temperature;
    g.b           = -h / in.temperature;
    return g;
  });
}

/** The same for distill, whose q are made again from the teacher's logits: 4096 x 128,000 bfloat16 with 64 ids a row 418 us,
 * 5.0 TB/s. */
template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_backward_kernel(score_rows in, listed_ids ids, teacher_logits teacher,
                                                                    const float* grad_loss, const float* lse, T* grad,
                                                                    int64_t gstride, bool by_cache, row_split split,
                                                                    int64_t row0)
{
  constexpr int E = kEntries<NT>;
  __shared__ listed_shares shares;
  __shared__ run parts[NT / 64];
  const int64_t b = row0 + blockIdx.x, r = b / split.parts;
  const int c0 = static_cast<int>(b - r * split.parts) * split.width, c1 = min(c0 + split.width, in.n);
  const T* row  = static_cast<const T*>(in.x) + r * in.stride;
  const float a = grad_loss[r] / in.temperature;
  listed_part<E> l;
  read_list<NT>(in, ids, teacher, r, l);
  write_gradient<T, false, NT>(row, grad + r * gstride, by_cache, c0, c1, shares, ids.k, [&](bool& some) {
    const run list = join_block<NT, false>(teacher_run(l, in.temperature), kLog2e / in.temperature, parts);
    const auto t   = teacher_of(list, in.temperature);
    some           = t.some;
    write_shares<NT>(l, t, a, ids.k, shares);
    lds_barrier();  // parts has been read
    auto g = gradient_base<T, NT>(row, in.n, lse[r], in.temperature, parts);
    g.a    = a;
    return g;
  });
}

/**
 * Both directions of rows that a workgroup holds in registers, H pieces of 16 bytes a thread: each is read once and its
 * gradient written once.  A workgroup takes every gridDim-th row; as a piece of a row's gradient is stored, the same piece
 * of its next row is loaded in its place, and pieces that have arrived enter that row's sums, so that reads, writes and
 * arithmetic go on side by side.  The next row's list comes meanwhile, E entries a thread.
 *
 * 4096 x 128,000 bfloat16 with 64 ids a row: 450 us, 4.7 TB/s, against 609 by two passes; what it lacks to a copy's 440 is
 * the join between a row's last load and its gradient's first store, when this workgroup has nothing on its way.
 */
template <typename T, int NT, int H>
__global__ __launch_bounds__(NT) void distill_step_kernel(score_rows in, listed_ids ids, teacher_logits teacher,
                                                          const float* grad_loss, float* loss, float* lse, T* grad,
                                                          int64_t gstride, bool by_cache)
{
  constexpr int N = kPer16<T>, kStep = NT * N, kLag = 4;  // pieces on their way
  constexpr int E = NT > kMaxListed ? 1 : kEntries<NT>;
  __shared__ listed_shares shares;
  __shared__ run both[2 * NT / 64];
  __shared__ float losses[NT / 64];
  const int last = in.n - N, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 64 * N;
  int mine       = static_cast<int>(threadIdx.x) * N;
  const float c  = kLog2e / in.temperature;
  uint4 held[H];
  run sums = nothing();
  float v[N];
  listed_part<E> l, after;
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
    add_scores<false>(sums, v, c);
  };
  read_list<NT>(in, ids, teacher, blockIdx.x, l);
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (h * kStep < in.n) load(blockIdx.x, h);
  read_listed(row_at(blockIdx.x), l);
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (h * kStep < in.n) add(h);
  for (int64_t r = blockIdx.x; r < in.m; r += gridDim.x) {
    asm volatile("" : "+v"(mine));  // the pieces' places are made again for every row: kept, they would take H registers
    const int64_t next = r + gridDim.x;
    const bool more    = next < in.m;
    if (more) read_list<NT>(in, ids, teacher, next, after);
    run list = teacher_run(l, in.temperature);
    join_both<NT>(sums, c, list, both);
    const auto t  = teacher_of(list, in.temperature);
    const auto o  = finish(sums, in.temperature);
    const float a = grad_loss[r] / in.temperature;
    write_shares<NT>(l, t, a, ids.k, shares);
    const float share = sum_lanes(loss_of(in, l, t, o));
    if (threadIdx.x % 64 == 0) losses[threadIdx.x / 64] = share;
    lds_barrier();
    if (threadIdx.x == 0) {
      float sum = losses[0];
      for (int w = 1; w < NT / 64; ++w)
        sum += losses[w];
      loss[r] = sum;
      lse[r]  = o.lse;
    }
    const listed_share first = share_at(shares, static_cast<int>(threadIdx.x % 64), ids.k);
    const gradient_row g{sums.ref, c, sums.s > 0.f ? log2f(sums.s) : sums.s == 0.f ? INFINITY : sums.s, a, 0.f};
    T* out = grad + r * gstride;
    sums   = nothing();
#pragma unroll
    for (int h = 0; h < H + kLag; ++h) {
      if (h < H && h * kStep < in.n) {
        const int at = min(h * kStep + mine, last), w0 = h * kStep + wave;
        unpack16<T>(held[h], v);
#pragma unroll
        for (int i = 0; i < N; ++i)
          v[i] = t.some ? gradient<false>(v[i], g) : 0.f;
        if (t.some) add_shares<NT == 64>(v, at, w0, last, in.n, first, shares, ids.k);
        if (h * kStep + mine < in.n) {
          if (by_cache)
            store16(out + at, pack16<T>(v));
          else
            store16_nt(out + at, pack16<T>(v));
        }
        if (more) load(next, h);
      }
      if (h == H / 2 && more) read_listed(row_at(next), after);
      if (more && h >= kLag && (h - kLag) * kStep < in.n) add(h - kLag);
    }
    l = after;
  }
}

constexpr int kMidRows = 512;   // rows whose top entries take 512 threads (333 x 50,021 float32: 21.2 us, by 256 22.9)

}  // namespace

auto log_probs_workspace(int64_t m, int n, int top) -> int64_t
{
  const auto split = forward_split_of(m, n, top);
  return split.parts == 1 ? 0 : m * split.parts * static_cast<int64_t>(sizeof(key64) * top + sizeof(part_sums));
}

auto distill_workspace(int64_t m, int n) -> int64_t { return log_probs_workspace(m, n, 0); }

void launch_log_probs(score_rows const& in, listed_ids const& ids, log_probs_out const& out, void* workspace, hipStream_t s)
{
  const auto split = forward_split_of(in.m, in.n, out.top);
  auto* best       = static_cast<key64*>(workspace);
  auto* part       = reinterpret_cast<part_sums*>(best + (split.parts > 1 ? in.m * split.parts * out.top : 0));
  with_type(in.type, [&](auto e) {
    using T          = decltype(e);
    const auto launch = [&](auto kernel, int threads, int64_t total) {
      for_grids(total, threads, [&](int64_t first, unsigned count) {
        kernel<<<count, threads, 0, s>>>(in, ids, out, split, part, best, first);
        OCTEX_HIP(hipGetLastError());
      });
    };
    const bool top = out.top > 0;
    if (split.parts > 1) {
      launch(top ? log_probs_kernel<T, kThreads, true, true> : log_probs_kernel<T, kThreads, false, true>, kThreads,
             in.m * split.parts);
      launch(top ? finish_log_probs_kernel<T, true> : finish_log_probs_kernel<T, false>, kThreads, in.m);
    } else if (by_wavefront(in.m, in.n, 0)) {
      launch(top ? log_probs_kernel<T, 64, true, false> : log_probs_kernel<T, 64, false, false>, 64, in.m);
    } else if (top && in.m <= kMidRows) {
      launch(log_probs_kernel<T, 512, true, false>, 512, in.m);
    } else {
      launch(top ? log_probs_kernel<T, kThreads, true, false> : log_probs_kernel<T, kThreads, false, false>, kThreads, in.m);
    }
  });
}

void launch_log_probs_backward(score_rows const& in, listed_ids const& ids, const float* grad_logp,
                               const float* grad_entropy, const float* lse, const float* entropy, void* grad,
                               int64_t gstride, hipStream_t s)
{
  const auto split = split_of(in.m, in.n);
  with_type(in.type, [&](auto e) {
    using T           = decltype(e);
    const auto launch = [&](auto kernel, int threads) {
      for_grids(in.m * split.parts, threads, [&](int64_t first, unsigned count) {
        kernel<<<count, threads, 0, s>>>(in, ids, grad_logp, grad_entropy, lse, entropy, static_cast<T*>(grad), gstride,
                                         passes_cache(in), split, first);
        OCTEX_HIP(hipGetLastError());
      });
    };
    if (by_wavefront(in.m, in.n, ids.k))
      launch(log_probs_backward_kernel<T, 64>, 64);
    else
      launch(log_probs_backward_kernel<T, kThreads>, kThreads);
  });
}

void launch_distill(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, float* loss, float* lse,
                    void* workspace, hipStream_t s)
{
  const auto split = forward_split_of(in.m, in.n, 0);
  auto* part       = static_cast<part_sums*>(workspace);
  with_type(in.type, [&](auto e) {
    using T = decltype(e);
    const auto launch = [&](auto kernel, int threads, int64_t total) {
      for_grids(total, threads, [&](int64_t first, unsigned count) {
        kernel<<<count, threads, 0, s>>>(in, ids, teacher, loss, lse, split, part, first);
        OCTEX_HIP(hipGetLastError());
      });
    };
    if (split.parts > 1) {
      launch(distill_kernel<T, kThreads, true>, kThreads, in.m * split.parts);
      launch(finish_distill_kernel<T>, 64, in.m);
    } else if (by_wavefront(in.m, in.n, ids.k)) {
      launch(distill_kernel<T, 64, false>, 64, in.m);
    } else {
      launch(distill_kernel<T, kThreads, false>, kThreads, in.m);
    }
  });
}

void launch_distill_backward(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher,
                             const float* grad_loss, const float* lse, void* grad, int64_t gstride, hipStream_t s)
{
  const auto split = split_of(in.m, in.n);
  with_type(in.type, [&](auto e) {
    using T           = decltype(e);
    const auto launch = [&](auto kernel, int threads) {
      for_grids(in.m * split.parts, threads, [&](int64_t first, unsigned count) {
        kernel<<<count, threads, 0, s>>>(in, ids, teacher, grad_loss, lse, static_cast<T*>(grad), gstride, passes_cache(in),
                                         split, first);
        OCTEX_HIP(hipGetLastError());
      });
    };
    if (by_wavefront(in.m, in.n, ids.k))
      launch(distill_backward_kernel<T, 64>, 64);
    else
      launch(distill_backward_kernel<T, kThreads>, kThreads);
  });
}

constexpr int kHeldThreads = 1024, kHeldPieces = 16;  // of the widest row that a workgroup holds

/** Few wide rows are quicker in parts, by two passes: 1 x 128,000 bfloat16 in 9.7 us against 23, 300 x 100,003 float16 in 46
 * against 52 (but 16 x 32,000 float32 in 10.7 against 9.8, 768 x 128,000 bfloat16 in 112 against 93). */
auto distill_step_held(int64_t m, int n, elem type) -> bool
{
  const int per = 16 / elem_size(type), pieces = (n + per - 1) / per;
  if (n < per || pieces > kHeldThreads * kHeldPieces) return false;
  return pieces <= kHeldThreads * 8 || m >= 512;
}

void launch_distill_step(score_rows const& in, listed_ids const& ids, teacher_logits const& teacher, const float* grad_loss,
                         float* loss, float* lse, void* grad, int64_t gstride, void* workspace, hipStream_t s)
{
  if (!distill_step_held(in.m, in.n, in.type)) {
    launch_distill(in, ids, teacher, loss, lse, workspace, s);
    launch_distill_backward(in, ids, teacher, grad_loss, lse, grad, gstride, s);
    return;
  }
  with_type(in.type, [&](auto e) {
    using T           = decltype(e);
    const auto launch = [&](auto kernel, int threads, int64_t slots) {
      kernel<<<static_cast<unsigned>(std::min(in.m, slots)), threads, 0, s>>>(in, ids, teacher, grad_loss, loss, lse,
                                                                              static_cast<T*>(grad), gstride, passes_cache(in));
      OCTEX_HIP(hipGetLastError());
    };
    const int pieces = (in.n + kPer16<T> - 1) / kPer16<T>;
    if (pieces <= 256 && in.m >= 2048 && ids.k <= kShortList)
      launch(distill_step_kernel<T, 64, 4>, 64, 8192);
    else if (pieces <= 1024 && in.m >= 2048 && ids.k <= kShortList)
      launch(distill_step_kernel<T, 64, 16>, 64, 4096);
    else if (pieces <= 1024)
      launch(distill_step_kernel<T, 256, 4>, 256, 2048);
    else if (pieces <= 4096 && in.m > 256)
      launch(distill_step_kernel<T, 256, 16>, 256, 1024);
    else if (pieces <= 4096)
      launch(distill_step_kernel<T, 1024, 4>, 1024, 256);
    else if (pieces <= 8192)
      launch(distill_step_kernel<T, 1024, 8>, 1024, 256);
    else
      launch(distill_step_kernel<T, 1024, 16>, 1024, 256);
  });
}

}  // namespace cuvs::neighbors::octex::detail
