// Rows of a table by ids, and the table's gradient.
//
//   embed      out_i = scale r_v T_v,  v = ids_i  (r: the scales of int8 rows);  ids outside the table: 0
//   backward   G_v = scale (sum of g_i over i with ids_i = v)  [+ what G_v held]
//
// The gradient's tokens are sorted by id, equal ones by place (a stable sort, digit by digit), so that a row's gradients are
// added in a fixed order in fp32 and rounded once.  A sorted chunk is one team's; a row's tokens that reach into the chunk
// behind theirs are still their own team's, and longer runs (a common token's) leave a sum a chunk, which are joined after.
// Both are bound by the bytes of the rows; a large copy takes 5.06 TB/s of this GPU, writing alone 6.85.

#include "common.hpp"
#include "elems_device.hpp"
#include "table.hpp"

#include <algorithm>

namespace cuvs::neighbors::octex::detail {

namespace {

constexpr int kUnit    = 8;  // values that a lane takes at a time
constexpr int kThreads = 256;

/** kUnit values as they lie in memory. */
template <typename T>
struct unit {
  static constexpr int kWords = kUnit * static_cast<int>(sizeof(T)) / 4;
  unsigned w[kWords];
};

/** The values of a row from `from` on; of a row of d < kUnit all of them, and 0 behind its end. */
template <typename T>
__device__ inline auto load_unit(const T* row, int from, int d) -> unit<T>
{
  unit<T> u;
  if (d >= kUnit) {
    __builtin_memcpy(u.w, row + from, sizeof(u.w));
    return u;
  }
  T e[kUnit];
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    e[i] = i < d ? row[i] : T{};
  __builtin_memcpy(u.w, e, sizeof(u.w));
  return u;
}

template <typename T>
__device__ inline void unpack_unit(unit<T> const& u, float (&v)[kUnit])
{
  if constexpr (sizeof(T) == 1) {
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      v[i] = static_cast<float>(static_cast<int>(u.w[i / 4] << (24 - 8 * (i % 4))) >> 24);
  } else {
    constexpr int N = kPer16<T>;
#pragma unroll
    for (int j = 0; j < kUnit / N; ++j) {
      float e[N];
      unpack16<T>(uint4{u.w[4 * j], u.w[4 * j + 1], u.w[4 * j + 2], u.w[4 * j + 3]}, e);
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[j * N + i] = e[i];
    }
  }
}

/** The columns of the unit at `at` (a multiple of kUnit): where the row ends inside, the unit's values are those of the row's
 * last columns, of which the ones before `at` are another lane's. */
__device__ inline auto unit_start(int at, int d) -> int { return max(min(at, d - kUnit), 0); }

template <typename T>
__device__ inline void store_unit(T* row, const float (&v)[kUnit], int at, int d, bool by_cache)
{
  constexpr int N = kPer16<T>;
  if (at + kUnit > d) {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      const int column = unit_start(at, d) + i;
      if (column >= at && column < d) row[column] = static_cast<T>(v[i]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kUnit / N; ++j) {
    float e[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      e[i] = v[j * N + i];
    if (by_cache)
      store16(row + at + j * N, pack16<T>(e));
    else
      store16_nt(row + at + j * N, pack16<T>(e));
  }
}

__device__ inline auto id_of(row_ids const& ids, int64_t i) -> int64_t
{
  return ids.wide ? static_cast<const int64_t*>(ids.ids)[i * ids.stride] : static_cast<const int32_t*>(ids.ids)[i * ids.stride];
}

constexpr int kRowsAhead = 4;  // rows that a team has on their way

/**
 * Teams of W lanes take kRowsAhead rows each, a unit a lane (of the slice blockIdx.y of their columns): all ids first, then
 * all rows, then the results.
 */
template <typename T, typename O, int W>
__global__ __launch_bounds__(kThreads) void embed_kernel(table_rows table, row_ids ids, int d, float scale, O* out,
                                                         int64_t ostride, bool by_cache, int64_t block0)
{
  constexpr int kTeams = kThreads / W;
  const int at         = (static_cast<int>(blockIdx.y) * W + static_cast<int>(threadIdx.x) % W) * kUnit;
  const int64_t i0     = ((block0 + blockIdx.x) * kTeams + threadIdx.x / W) * kRowsAhead;
  if (at >= d) return;
  const int from = unit_start(at, d);
  int64_t id[kRowsAhead];
  float s[kRowsAhead];
  unit<T> u[kRowsAhead];
#pragma unroll
  for (int q = 0; q < kRowsAhead; ++q) {
    id[q] = i0 + q < ids.m ? id_of(ids, i0 + q) : -1;
    if (id[q] >= table.n) id[q] = -1;
  }
#pragma unroll
  for (int q = 0; q < kRowsAhead; ++q) {
    if (id[q] < 0) continue;
    u[q] = load_unit(static_cast<const T*>(table.x) + id[q] * table.stride, from, d);
    s[q] = sizeof(T) == 1 ? scale * table.scales[id[q]] : scale;
  }
#pragma unroll
  for (int q = 0; q < kRowsAhead; ++q) {
    if (i0 + q >= ids.m) break;
    float v[kUnit];
    if (id[q] >= 0) unpack_unit(u[q], v);
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      v[i] = id[q] >= 0 ? v[i] * s[q] : 0.f;
    store_unit(out + (i0 + q) * ostride, v, at, d, by_cache);
  }
}

// ---- tokens sorted by id

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortTile    = 4096;  // tokens of a workgroup
constexpr int kSortPer     = kSortTile / kSortThreads;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;

/** A token: its row of the table (n: padding) and its place. */
struct token {
  unsigned row;
  int place;
};

__device__ inline auto token_of(row_ids const& ids, int64_t n, int64_t i) -> token
{
  const int64_t id = id_of(ids, i);
  return {static_cast<unsigned>(id < 0 || id >= n ? n : id), static_cast<int>(i)};
}

/** Tokens [wave's first + 64 q + lane] of a tile, row ~0 past the end. */
template <typename F>
__device__ inline void read_tile(int64_t first, int64_t m, token (&t)[kSortPer], F read)
{
  const int64_t mine = first + threadIdx.x / 64 * (64 * kSortPer) + threadIdx.x % 64;
#pragma unroll
  for (int q = 0; q < kSortPer; ++q)
    t[q] = mine + 64 * q < m ? read(mine + 64 * q) : token{~0u, -1};
}

/** The lanes of the wavefront that have a token of the same digit. */
__device__ inline auto same_digit(unsigned digit, bool has) -> unsigned long long
{
  unsigned long long same = __ballot(has);
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const bool one                = digit >> b & 1;
    const unsigned long long ones = __ballot(one);
    same &= one ? ones : ~ones;
  }
  return same;
}

__device__ inline auto lanes_below(unsigned long long lanes) -> int
{
  return __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(lanes >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(lanes), 0));
}

/** The ranks of a tile's tokens among those of the same digit and wavefront, whose numbers they leave in counts (LDS, 0
 * before). */
__device__ inline void rank_tile(const token (&t)[kSortPer], int shift, int (*counts)[kDigits], int (&rank)[kSortPer])
{
  int* mine = counts[threadIdx.x / 64];
#pragma unroll
  for (int q = 0; q < kSortPer; ++q) {
    const unsigned digit = t[q].row >> shift & (kDigits - 1);
    const bool has       = t[q].place >= 0;
    const auto same      = same_digit(digit, has);
    const int below      = lanes_below(same);
    const int before     = has ? mine[digit] : 0;
    wave_fence();
    if (has && below == 0) mine[digit] = before + __popcll(same);
    wave_fence();
    rank[q] = before + below;
  }
}

__device__ inline void clear_counts(int (*counts)[kDigits])
{
  for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads)
    (&counts[0][0])[i] = 0;
}

/** The exclusive sums over kDigits values, one a thread of the first kDigits; sums is LDS, one a wavefront of them. */
__device__ inline auto scan_digits(int v, int* sums) -> int
{
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  int sum = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int other = __shfl_up(sum, d);
    if (lane >= d) sum += other;
  }
  if (lane == 63 && threadIdx.x < kDigits) sums[wave] = sum;
  lds_barrier();
  int before = 0;
  for (int w = 0; w < kDigits / 64; ++w)
    before += w < wave ? sums[w] : 0;
  lds_barrier();
  return before + sum - v;
}

/** Turns the wavefronts' counts into the places at which their tokens of a digit start; base: of the tile's, a thread's digit. */
__device__ inline void start_waves(int (*counts)[kDigits], int base)
{
  if (threadIdx.x < kDigits) {
    for (int w = 0; w < kSortWaves; ++w) {
      const int c            = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = base;
      base += c;
    }
  }
}

__device__ inline auto wave_total(int (*counts)[kDigits]) -> int
{
  int sum = 0;
  if (threadIdx.x < kDigits)
    for (int w = 0; w < kSortWaves; ++w)
      sum += counts[w][threadIdx.x];
  return sum;
}

/** Up to kSortTile tokens by one workgroup, all digits. */
__global__ __launch_bounds__(kSortThreads) void sort_alone_kernel(row_ids ids, int64_t n, int passes, token* out)
{
  __shared__ int counts[kSortWaves][kDigits];
  __shared__ token tokens[kSortTile];
  __shared__ int sums[kDigits / 64];
  token t[kSortPer];
  int rank[kSortPer];
  read_tile(0, ids.m, t, [&](int64_t i) { return token_of(ids, n, i); });
  for (int p = 0; p < passes; ++p) {
    const int shift = p * kDigitBits;
    clear_counts(counts);
    lds_barrier();
    rank_tile(t, shift, counts, rank);
    lds_barrier();
    start_waves(counts, scan_digits(wave_total(counts), sums));
    lds_barrier();
#pragma unroll
    for (int q = 0; q < kSortPer; ++q)
      if (t[q].place >= 0) tokens[counts[threadIdx.x / 64][t[q].row >> shift & (kDigits - 1)] + rank[q]] = t[q];
    lds_barrier();
    read_tile(0, ids.m, t, [&](int64_t i) { return tokens[i]; });
    lds_barrier();
  }
  const int64_t mine = threadIdx.x / 64 * (64 * kSortPer) + threadIdx.x % 64;
#pragma unroll
  for (int q = 0; q < kSortPer; ++q)
    if (t[q].place >= 0) out[mine + 64 * q] = t[q];
}

/** The numbers of a tile's tokens of each digit: tiles [gridDim, kDigits]. */
__global__ __launch_bounds__(kSortThreads) void count_digits_kernel(row_ids ids, int64_t n, const token* in, int shift,
                                                                    int* tiles)
{
  __shared__ int counts[kDigits];
  if (threadIdx.x < kDigits) counts[threadIdx.x] = 0;
  lds_barrier();
  token t[kSortPer];
  read_tile(int64_t{blockIdx.x} * kSortTile, ids.m, t,
            [&](int64_t i) { return in != nullptr ? in[i] : token_of(ids, n, i); });
#pragma unroll
  for (int q = 0; q < kSortPer; ++q)
    if (t[q].place >= 0) atomicAdd(counts + (t[q].row >> shift & (kDigits - 1)), 1);
  lds_barrier();
  if (threadIdx.x < kDigits) tiles[int64_t{blockIdx.x} * kDigits + threadIdx.x] = counts[threadIdx.x];
}

/** Moves a tile's tokens to their places by one digit; every workgroup adds up the tiles' counts itself. */
__global__ __launch_bounds__(kSortThreads) void move_tokens_kernel(row_ids ids, int64_t n, const token* in, int shift,
                                                                   const int* tiles, token* out)
{
  __shared__ int counts[kSortWaves][kDigits];
  __shared__ int sums[kDigits / 64];
  token t[kSortPer];
  int rank[kSortPer];
  read_tile(int64_t{blockIdx.x} * kSortTile, ids.m, t,
            [&](int64_t i) { return in != nullptr ? in[i] : token_of(ids, n, i); });
  clear_counts(counts);
  int before = 0, all = 0;
  if (threadIdx.x < kDigits) {
#pragma unroll 8
    for (unsigned b = 0; b < gridDim.x; ++b) {
      const int c = tiles[int64_t{b} * kDigits + threadIdx.x];
      all += c;
      before += b < blockIdx.x ? c : 0;
    }
  }
  const int base = scan_digits(all, sums) + before;
  rank_tile(t, shift, counts, rank);
  lds_barrier();
  start_waves(counts, base);
  lds_barrier();
#pragma unroll
  for (int q = 0; q < kSortPer; ++q)
    if (t[q].place >= 0) out[counts[threadIdx.x / 64][t[q].row >> shift & (kDigits - 1)] + rank[q]] = t[q];
}

// ---- the sums of sorted tokens

/** Sorted tokens [m] in chunks of `width`.  A run (the tokens of one row) that ends in the chunk behind its first token's, or
 * before, is that first chunk's; a longer one is cut at the borders, and its chunks leave their sums in cut [chunk][2][d]: of a
 * run that came from before at 0, of one that begins here at 1. */
struct sorted_tokens {
  const token* t;
  int64_t m, n;
  int width;
  float* cut;

  __device__ auto row(int64_t i) const -> int64_t { return t[i].row; }
  /** Whether the run at the last place before the border b goes on behind it. */
  __device__ auto crosses(int64_t b) const -> bool { return b < m && row(b) == row(b - 1); }
  /** Whether the run of `row`, which begins in the chunk before the border b and crosses it, is cut. */
  __device__ auto is_cut(int64_t b, int64_t of) const -> bool { return b + width < m && row(b + width) == of; }
};

constexpr int kTokensAhead = 8;  // whose gradients a team has on their way

template <typename O>
__device__ inline void write_sum(const float (&sum)[kUnit], float scale, bool add, O* row, int at, int d, bool by_cache)
{
  float v[kUnit];
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    v[i] = sum[i] * scale;
  if (add) {
    float old[kUnit];
    unpack_unit(load_unit(row, unit_start(at, d), d), old);
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      v[i] += old[i];
  }
  store_unit(row, v, at, d, by_cache);
}

/** Sets the rows [v0, v0 + rows) that have no token to 0; a thread looks for each. */
template <typename O>
__device__ inline void clear_rows(sorted_tokens const& s, int64_t v0, int rows, int d, O* out, int64_t ostride, bool by_cache)
{
  constexpr int N = kPer16<O>;
  __shared__ bool used[kThreads];
  if (static_cast<int>(threadIdx.x) < rows) {
    const int64_t v = v0 + threadIdx.x;
    int64_t lo = 0, hi = s.m;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (s.row(mid) < v)
        lo = mid + 1;
      else
        hi = mid;
    }
    used[threadIdx.x] = lo < s.m && s.row(lo) == v;
  }
  lds_barrier();
  const int pieces = (d + N - 1) / N;
  for (int i = threadIdx.x; i < rows * pieces; i += kThreads) {
    const int r = i / pieces, at = (i - r * pieces) * N;
    if (used[r]) continue;
    O* row = out + (v0 + r) * ostride;
    if (d < N) {
      for (int j = 0; j < d; ++j)
        row[j] = static_cast<O>(0.f);
    } else if (by_cache) {
      store16(row + min(at, d - N), uint4{0, 0, 0, 0});
    } else {
      store16_nt(row + min(at, d - N), uint4{0, 0, 0, 0});
    }
  }
}

/**
 * The sums of the runs of a chunk each, by teams of W lanes, a unit a lane (of one of `slices` slices of their columns), the
 * gradients of kTokensAhead tokens on their way at a time.  Workgroups from `sum_blocks` on clear `clear` rows each.
 */
template <typename T, typename O, int W>
__global__ __launch_bounds__(kThreads) void sum_runs_kernel(sorted_tokens s, const T* grad, int64_t gstride, int d, float scale,
                                                            bool add, O* out, int64_t ostride, bool by_cache,
                                                            unsigned slices, unsigned sum_blocks, int clear)
{
  if (blockIdx.x >= sum_blocks) {
    const int64_t v0 = int64_t{blockIdx.x - sum_blocks} * clear;
    return clear_rows(s, v0, static_cast<int>(min(s.n - v0, int64_t{clear})), d, out, ostride, by_cache);
  }
  constexpr int kTeams = kThreads / W;
  const int64_t chunk  = int64_t{blockIdx.x / slices} * kTeams + threadIdx.x / W;
  const int at         = (static_cast<int>(blockIdx.x % slices) * W + static_cast<int>(threadIdx.x) % W) * kUnit;
  const int64_t b = chunk * s.width, e = min(b + s.width, s.m);
  if (b >= s.m || at >= d) return;
  const int64_t first = s.row(b), last = s.row(e - 1);
  if (first >= s.n) return;  // padding, to the end
  const int from        = unit_start(at, d);
  const bool before     = b > 0 && s.row(b - 1) == first;
  const bool crosses    = last < s.n && s.crosses(e);
  const bool through    = before && crosses && first == last;  // the whole chunk is a cut run's
  const bool tail       = crosses && !through && s.is_cut(e, last);
  const bool goes_on    = crosses && !through && !tail;  // the last run ends in the next chunk
  bool head             = before && (through || (b > s.width && s.row(b - s.width - 1) == first));
  int64_t p             = b;
  if (before && !head)  // the chunk before has it
    while (p < e && s.row(p) == first)
      ++p;
  float* cut      = s.cut + chunk * 2 * d;
  int64_t current = -1;
  float sum[kUnit];
  // the place of the sum's run: what came from before, what is cut behind, or the row itself
  const auto flush = [&](bool at_end) {
    if (current < 0) return;
    if (head)
      write_sum(sum, 1.f, false, cut, at, d, true);
    else if (at_end && tail)
      write_sum(sum, 1.f, false, cut + d, at, d, true);
    else
      write_sum(sum, scale, add, out + current * ostride, at, d, by_cache);
    head = false;
  };
  const auto token_at = [&](int64_t i) {
    token t = i < s.m ? s.t[i] : token{~0u, 0};
    if (t.row >= s.n || (i >= e && !(goes_on && t.row == last))) t.row = ~0u;
    return t;
  };
  token next[kTokensAhead];
#pragma unroll
  for (int q = 0; q < kTokensAhead; ++q)
    next[q] = token_at(p + q);
  while (next[0].row != ~0u) {
    token t[kTokensAhead];
    unit<T> u[kTokensAhead];
#pragma unroll
    for (int q = 0; q < kTokensAhead; ++q) {
      t[q] = next[q];
      if (t[q].row != ~0u) u[q] = load_unit(grad + t[q].place * gstride, from, d);
    }
    p += kTokensAhead;
#pragma unroll
    for (int q = 0; q < kTokensAhead; ++q)
      next[q] = token_at(p + q);
#pragma unroll
    for (int q = 0; q < kTokensAhead; ++q) {
      if (t[q].row == ~0u) break;
      float v[kUnit];
      unpack_unit(u[q], v);
      if (t[q].row != current) {
        flush(false);
        current = t[q].row;
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] = v[i];
      } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] += v[i];
      }
    }
  }
  flush(true);
}

constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;

/** Joins the sums of the run that begins in a chunk and is cut, if one is; 64 units of its columns a workgroup. */
template <typename O>
__global__ __launch_bounds__(kJoinThreads) void join_runs_kernel(sorted_tokens s, int d, float scale, bool add, O* out,
                                                                 int64_t ostride, bool by_cache, int64_t chunk0)
{
  __shared__ float sums[kJoinWaves][64][kUnit];
  const int64_t chunk = chunk0 + blockIdx.x, b = chunk * s.width, e = b + s.width;
  if (e >= s.m) return;
  const int64_t last = s.row(e - 1);
  if (last >= s.n || !s.crosses(e) || !s.is_cut(e, last)) return;
  if (s.row(b) == last && b > 0 && s.row(b - 1) == last) return;  // it came from before
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int at = (static_cast<int>(blockIdx.y) * 64 + lane) * kUnit, from = unit_start(at, d);
  float sum[kUnit];
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    sum[i] = 0.f;
  const auto take = [&](const float* part) {
    float v[kUnit];
    unpack_unit(load_unit(part, from, d), v);
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      sum[i] += v[i];
  };
  if (at < d) {
    if (wave == 0) take(s.cut + (chunk * 2 + 1) * d);
    for (int64_t c = chunk + 1 + wave; c * s.width < s.m && s.row(c * s.width) == last; c += kJoinWaves)
      take(s.cut + c * 2 * d);
  }
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    sums[wave][lane][i] = sum[i];
  lds_barrier();
  if (wave > 0 || at >= d) return;
  for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      sum[i] += sums[w][lane][i];
  write_sum(sum, scale, add, out + last * ostride, at, d, by_cache);
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

/** Calls f with the lanes of a row's team: its units, or 64 of them a slice. */
template <typename F>
void with_team(int64_t d, F f)
{
  const int64_t units = (d + kUnit - 1) / kUnit;
  if (units <= 8)
    f(std::integral_constant<int, 8>{});
  else if (units <= 16)
    f(std::integral_constant<int, 16>{});
  else if (units <= 32)
    f(std::integral_constant<int, 32>{});
  else
    f(std::integral_constant<int, 64>{});
}

constexpr int64_t kMaxGrid = (int64_t{1} << 32) / kJoinThreads - 1;  // workgroups of a launch: less than 2^32 work-items

auto ceil_div(int64_t a, int64_t b) -> int64_t { return (a + b - 1) / b; }

/** Whether results are stored through the caches: up to half of the last-level cache's 256 MB, where their reader may find
 * them. */
auto passes_cache(int64_t rows, int64_t d, elem type) -> bool { return rows * d * elem_size(type) <= int64_t{128} << 20; }

/** Tokens of a chunk: as many as leave the GPU 4096 wavefronts, from 16 to 128. */
auto chunk_width(int64_t m, int64_t d) -> int
{
  const int64_t waves = m * ceil_div(d, 64 * kUnit) / 4096;
  int width           = 16;
  while (width < 128 && width < waves)
    width *= 2;
  return width;
}

/** How the workspace is laid out, from place to place in bytes. */
struct sort_layout {
  int passes;
  int64_t tiles, chunks, second, counts, cut, end;
};

auto layout_of(int64_t m, int64_t n, int64_t d) -> sort_layout
{
  const auto up = [](int64_t v) { return ceil_div(v, 256) * 256; };
  sort_layout l{};
  int bits = 1;
  while (n >> bits != 0)
    ++bits;
  l.passes        = static_cast<int>(ceil_div(bits, kDigitBits));
  l.tiles         = ceil_div(m, kSortTile);
  const int width = chunk_width(m, d);
  l.chunks        = ceil_div(m, width);
  l.second        = up(m * static_cast<int64_t>(sizeof(token)));
  l.counts        = l.tiles > 1 ? 2 * l.second : l.second;
  l.cut           = l.counts + (l.tiles > 1 ? up(l.tiles * kDigits * 4) : 0);
  l.end           = l.cut + (m > width ? l.chunks * 2 * d * 4 : 0);
  return l;
}

}  // namespace

void launch_embed(table_rows const& table, row_ids const& ids, int64_t d, float scale, value_rows const& out, hipStream_t s)
{
  const auto run = [&](auto t) {
    using T = decltype(t);
    with_type(out.type, [&](auto o) {
      using O = decltype(o);
      with_team(d, [&](auto lanes) {
        constexpr int W      = lanes();
        const int64_t blocks = ceil_div(ids.m, int64_t{kThreads / W} * kRowsAhead);
        const auto slices    = static_cast<unsigned>(ceil_div(d, W * kUnit));
        for (int64_t first = 0; first < blocks; first += kMaxGrid) {
          const dim3 grid(static_cast<unsigned>(std::min(kMaxGrid, blocks - first)), slices);
          embed_kernel<T, O, W><<<grid, kThreads, 0, s>>>(table, ids, static_cast<int>(d), scale, static_cast<O*>(out.x),
                                                          out.stride, passes_cache(ids.m, d, out.type), first);
          OCTEX_HIP(hipGetLastError());
        }
      });
    });
  };
  if (table.type == elem::i8)
    run(int8_t{});
  else
    with_type(table.type, run);
}

auto embed_backward_workspace(int64_t m, int64_t n, int64_t d) -> int64_t { return m == 0 ? 0 : layout_of(m, n, d).end; }

void launch_embed_backward(value_rows const& grad, row_ids const& ids, int64_t n, int64_t d, float scale, bool add,
                           value_rows const& out, void* workspace, hipStream_t s)
{
  const auto l    = layout_of(ids.m, n, d);
  auto* base      = static_cast<char*>(workspace);
  auto* tokens    = reinterpret_cast<token*>(base);
  auto* second    = reinterpret_cast<token*>(base + l.second);
  auto* counts    = reinterpret_cast<int*>(base + l.counts);
  if (l.tiles == 1) {
    sort_alone_kernel<<<1, kSortThreads, 0, s>>>(ids, n, l.passes, tokens);
    OCTEX_HIP(hipGetLastError());
  }
  for (int p = 0; l.tiles > 1 && p < l.passes; ++p) {
    const bool to_first = (l.passes - 1 - p) % 2 == 0;
    const token* in     = p == 0 ? nullptr : to_first ? second : tokens;
    const int shift     = p * kDigitBits;
    count_digits_kernel<<<static_cast<unsigned>(l.tiles), kSortThreads, 0, s>>>(ids, n, in, shift, counts);
    OCTEX_HIP(hipGetLastError());
    move_tokens_kernel<<<static_cast<unsigned>(l.tiles), kSortThreads, 0, s>>>(ids, n, in, shift, counts,
                                                                               to_first ? tokens : second);
    OCTEX_HIP(hipGetLastError());
  }
  const sorted_tokens sorted{tokens, ids.m, n, chunk_width(ids.m, d), reinterpret_cast<float*>(base + l.cut)};
  const bool by_cache = add || passes_cache(n, d, out.type);
  // rows that a workgroup clears: 256 KB of them, for each of which a thread looks
  const int clear = static_cast<int>(std::clamp<int64_t>((256 << 10) / (d * elem_size(out.type)), 16, kThreads));
  with_type(out.type, [&](auto o) {
    using O = decltype(o);
    with_type(grad.type, [&](auto t) {
      using T = decltype(t);
      with_team(d, [&](auto lanes) {
        constexpr int W   = lanes();
        const auto slices = static_cast<unsigned>(ceil_div(d, W * kUnit));
        const auto sums   = static_cast<unsigned>(ceil_div(l.chunks, kThreads / W)) * slices;
        const auto clears = add ? 0u : static_cast<unsigned>(ceil_div(n, clear));
        sum_runs_kernel<T, O, W><<<sums + clears, kThreads, 0, s>>>(sorted, static_cast<const T*>(grad.x), grad.stride,
                                                                    static_cast<int>(d), scale, add, static_cast<O*>(out.x),
                                                                    out.stride, by_cache, slices, sums, clear);
        OCTEX_HIP(hipGetLastError());
      });
    });
    // a cut run reaches into a third chunk
    for (int64_t first = 0; l.chunks > 2 && first < l.chunks; first += kMaxGrid) {
      const dim3 grid(static_cast<unsigned>(std::min(kMaxGrid, l.chunks - first)),
                      static_cast<unsigned>(ceil_div(d, 64 * kUnit)));
      join_runs_kernel<O><<<grid, kJoinThreads, 0, s>>>(sorted, static_cast<int>(d), scale, add, static_cast<O*>(out.x),
                                                        out.stride, by_cache, first);
      OCTEX_HIP(hipGetLastError());
    }
  });
}

}  // namespace cuvs::neighbors::octex::detail
