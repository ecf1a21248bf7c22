// Rows of a table by ids, and the table's gradient.
//
//   embed      out_i = scale r_v T_v,  v = ids_i  (r: the scales of int8 rows);  ids outside the table: 0
//   backward   G_v = scale (sum of g_i over i with ids_i = v)  [+ what G_v held]
//
// The gradient's tokens are sorted by id, equal ones by place (a stable sort, digit by digit; up to 1024 of them, and of short rows
// up to 4096, are looked through instead), so that a row's gradients are added in a fixed order in fp32 and rounded once.  A sorted
// chunk is one team's; a row's tokens that reach into the chunk behind theirs are still their own team's, and longer runs (a common
// token's) leave a sum a chunk, which are joined after.
// Both are bound by the bytes of the rows; a large copy takes 5.06 TB/s of this GPU, writing alone 6.85.  32,768 rows of 4096
// bfloat16 take 78 us (152 MB read, 268 written: 5.4 TB/s), the gradient of a table of 128,000 such rows 276 (1.3 GB: 4.8).

#include "common.hpp"
#include "elems_device.hpp"
#include "table.hpp"

#include <algorithm>

namespace cuvs::neighbors::octex::detail {

namespace {

constexpr int kUnit    = 8;  // values that a lane takes at a time
constexpr int kThreads = 256;

/** U values as they lie in memory. */
template <typename T, int U = kUnit>
struct unit {
  static constexpr int kWords = U * static_cast<int>(sizeof(T)) / 4;
  unsigned w[kWords];
};

/** The values of a row from `from` on; of a row of d < U (kShort) all of them, and 0 behind its end. */
template <bool kShort, int U = kUnit, typename T>
__device__ inline auto load_unit(const T* row, int from, int d) -> unit<T, U>
{
  unit<T, U> u;
  if constexpr (kShort) {
    T e[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      e[i] = i < d ? row[i] : T{};
    __builtin_memcpy(u.w, e, sizeof(u.w));
  } else {
    __builtin_memcpy(u.w, row + from, sizeof(u.w));
  }
  return u;
}

template <typename T, int U>
__device__ inline void unpack_unit(unit<T, U> const& u, float (&v)[U])
{
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if constexpr (sizeof(T) == 1)
      v[i] = static_cast<float>(static_cast<int>(u.w[i / 4] << (24 - 8 * (i % 4))) >> 24);
    else if constexpr (sizeof(T) == 4)
      v[i] = __uint_as_float(u.w[i]);
    else if constexpr (std::is_same_v<T, bf16>)
      v[i] = __uint_as_float(i % 2 == 0 ? u.w[i / 2] << 16 : u.w[i / 2] & 0xffff0000u);
    else
      v[i] = static_cast<float>(__builtin_bit_cast(f16, static_cast<unsigned short>(u.w[i / 2] >> 16 * (i % 2))));
  }
}

/** Where a lane finds its unit at the column `at` (a multiple of U): one that would pass the row's end is moved back to it, so
 * that columns before `at` are another lane's too. */
template <int U = kUnit>
__device__ inline auto unit_start(int at, int d) -> int
{
  return max(min(at, d - U), 0);
}

/** Stores a unit; lanes that have a column twice store it alike. */
template <bool kShort, typename T, int U>
__device__ inline void store_unit(T* row, const float (&v)[U], int from, int d, bool by_cache)
{
  constexpr int N = kPer16<T>;
  if constexpr (kShort) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (i < d) row[i] = static_cast<T>(v[i]);
  } else {
#pragma unroll
    for (int j = 0; j < U / N; ++j) {
      float e[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
        e[i] = v[j * N + i];
      if (by_cache)
        store16(row + from + j * N, pack16<T>(e));
      else
        store16_nt(row + from + j * N, pack16<T>(e));
    }
  }
}

/** The ids at places i0 + q * step, clamped to the last one: all of them on their way at once. */
template <int N>
__device__ inline void read_ids(row_ids const& ids, int64_t i0, int64_t step, int64_t (&id)[N])
{
  if (ids.wide) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      id[q] = static_cast<const int64_t*>(ids.ids)[min(i0 + q * step, ids.m - 1) * ids.stride];
  } else {
#pragma unroll
    for (int q = 0; q < N; ++q)
      id[q] = static_cast<const int32_t*>(ids.ids)[min(i0 + q * step, ids.m - 1) * ids.stride];
  }
}

constexpr int kRowsAhead = 4;  // rows that a team has on their way

/** Values of a result's 16 bytes, which a lane has: past the caches, pieces that do not lie side by side leave their lines in parts
 * (8 values of float32 a lane, in two pieces: 17,235 x 2752 of a table in 92 us). */
template <typename O>
constexpr int kResultUnit = kPer16<O>;

/**
 * Teams of W lanes (1: of rows shorter than a unit) take kRowsAhead rows each, kResultUnit values a lane (of one of `slices`
 * slices of their columns, side by side in a workgroup): all ids first, then all rows, then the results.  No load waits for a
 * condition: padding takes the table's first row and drops it.
 */
template <typename T, typename O, int W>
__global__ __launch_bounds__(kThreads) void embed_kernel(table_rows table, row_ids ids, int d, float scale, O* out,
                                                         int64_t ostride, bool by_cache, unsigned slices, int64_t block0)
{
  constexpr int kTeams = kThreads / W, U = kResultUnit<O>;
  const int64_t team   = (block0 + blockIdx.x) * kTeams + threadIdx.x / W;
  const int64_t i0     = team / slices * kRowsAhead;
  const int at         = (static_cast<int>(team % slices) * W + static_cast<int>(threadIdx.x) % W) * U;
  if (at >= d || i0 >= ids.m) return;
  const int from = unit_start<U>(at, d);
  int64_t id[kRowsAhead];
  float s[kRowsAhead];
  unit<T, U> u[kRowsAhead] = {};
  read_ids(ids, i0, 1, id);
  if (table.n > 0) {
#pragma unroll
    for (int q = 0; q < kRowsAhead; ++q) {
      const int64_t v = id[q] < 0 || id[q] >= table.n ? 0 : id[q];
      u[q]            = load_unit<W == 1, U>(static_cast<const T*>(table.x) + v * table.stride, from, d);
      s[q]            = sizeof(T) == 1 ? scale * table.scales[v] : scale;
    }
  }
#pragma unroll
  for (int q = 0; q < kRowsAhead; ++q) {
    if (i0 + q >= ids.m) break;
    const bool listed = id[q] >= 0 && id[q] < table.n;
    float v[U];
    unpack_unit(u[q], v);
#pragma unroll
    for (int i = 0; i < U; ++i)
      v[i] = listed ? v[i] * s[q] : 0.f;
    store_unit<W == 1>(out + (i0 + q) * ostride, v, from, d, by_cache);
  }
}

// ---- tokens sorted by id

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;

/** A token: its row of the table (n: padding) and its place. */
struct token {
  unsigned row;
  int place;
};

__device__ inline auto row_of(int64_t id, unsigned n) -> unsigned { return id < 0 || id >= n ? n : static_cast<unsigned>(id); }

/** A thread's tokens of the tile of kSortThreads * P places from `first` on: those at wave's first + 64 q + lane, so that ranks
 * by wavefront, q and lane are ranks by place.  Past the end their place is -1. */
template <int P>
__device__ inline auto my_place(int64_t first) -> int64_t
{
  return first + threadIdx.x / 64 * (64 * P) + threadIdx.x % 64;
}

template <int P>
__device__ inline void read_tile(row_ids const& ids, unsigned n, const token* in, int64_t first, token (&t)[P])
{
  const int64_t mine = my_place<P>(first);
  if (in != nullptr) {
#pragma unroll
    for (int q = 0; q < P; ++q)
      t[q] = in[min(mine + 64 * q, ids.m - 1)];
  } else {  // a first pass
    int64_t id[P];
    read_ids(ids, mine, 64, id);
#pragma unroll
    for (int q = 0; q < P; ++q)
      t[q] = {row_of(id[q], n), static_cast<int>(mine + 64 * q)};
  }
#pragma unroll
  for (int q = 0; q < P; ++q)
    if (mine + 64 * q >= ids.m) t[q].place = -1;
}

/** A digit of a token's row: `bits` (at most kDigitBits) from `shift` on. */
struct digit {
  int shift, bits;

  __device__ auto of(token const& t) const -> unsigned { return t.row >> shift & ((1u << bits) - 1); }
};

/** The lanes of the wavefront that have a token of the same digit. */
__device__ inline auto same_digit(unsigned value, int bits, bool has) -> unsigned long long
{
  unsigned long long same = __ballot(has);
  for (int b = 0; b < bits; ++b) {
    const bool one                = value >> b & 1;
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
template <int P>
__device__ inline void rank_tile(const token (&t)[P], digit d, int (*counts)[kDigits], int (&rank)[P])
{
  int* mine = counts[threadIdx.x / 64];
#pragma unroll
  for (int q = 0; q < P; ++q) {
    const bool has = t[q].place >= 0;
    if (__ballot(has) == 0) break;
    const unsigned value = d.of(t[q]);
    const auto same      = same_digit(value, d.bits, has);
    const int below      = lanes_below(same);
    const int before     = has ? mine[value] : 0;
    wave_fence();
    if (has && below == 0) mine[value] = before + __popcll(same);
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

/** The wavefronts' counts of a thread's digit, and their sum. */
__device__ inline auto wave_counts(int (*counts)[kDigits], int (&c)[kSortWaves]) -> int
{
  int sum = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w)
    sum += c[w] = threadIdx.x < kDigits ? counts[w][threadIdx.x] : 0;
  return sum;
}

/** Turns them into the places at which the wavefronts' tokens of the digit start. */
__device__ inline void start_waves(int (*counts)[kDigits], const int (&c)[kSortWaves], int base)
{
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    if (threadIdx.x < kDigits) counts[w][threadIdx.x] = base;
    base += c[w];
  }
}

/** A share of the table's gradient that is set to 0 beside a step of the sort, whichever rows have tokens: [first, first + bytes)
 * of dense rows, by `blocks` workgroups. */
struct fill_share {
  char* first;
  int64_t bytes;
  unsigned blocks;
};

constexpr int kFillBytes = 64 << 10;  // that a workgroup fills at a time

/** A workgroup's part of the share: whole 16-byte pieces but for the ends. */
__device__ inline void fill(fill_share const& f, unsigned block)
{
  const auto lead = static_cast<int64_t>(reinterpret_cast<uintptr_t>(f.first) % 16);
  for (int64_t base = int64_t{block} * kFillBytes - lead; base < f.bytes; base += int64_t{f.blocks} * kFillBytes) {
#pragma unroll
    for (int q = 0; q < kFillBytes / 16 / kSortThreads; ++q) {
      const int64_t at = base + (q * kSortThreads + static_cast<int>(threadIdx.x)) * 16;
      if (at >= 0 && at + 16 <= f.bytes) {
        store16(f.first + at, uint4{0, 0, 0, 0});
      } else {
        for (int64_t j = max(at, int64_t{0}); j < min(at + 16, f.bytes); j += 2)
          *reinterpret_cast<uint16_t*>(f.first + j) = 0;
      }
    }
  }
}

/** Up to kSortThreads * P tokens by the first workgroup, all of their `bits` in `passes`; the others fill. */
template <int P>
__global__ __launch_bounds__(kSortThreads) void sort_alone_kernel(row_ids ids, unsigned n, int passes, int bits, token* out,
                                                                  fill_share share)
{
  if (blockIdx.x > 0) return fill(share, blockIdx.x - 1);
  __shared__ int counts[kSortWaves][kDigits];
  __shared__ token tokens[kSortThreads * P];
  __shared__ int sums[kDigits / 64];
  token t[P];
  int rank[P], c[kSortWaves];
  read_tile<P>(ids, n, nullptr, 0, t);
  for (int p = 0; p < passes; ++p) {
    const digit d{p * bits, bits};
    clear_counts(counts);
    lds_barrier();
    rank_tile<P>(t, d, counts, rank);
    lds_barrier();
    start_waves(counts, c, scan_digits(wave_counts(counts, c), sums));
    lds_barrier();
    token* const to = p + 1 < passes ? tokens : out;
#pragma unroll
    for (int q = 0; q < P; ++q)
      if (t[q].place >= 0) to[counts[threadIdx.x / 64][d.of(t[q])] + rank[q]] = t[q];
    if (p + 1 == passes) return;
    lds_barrier();
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const int64_t mine = my_place<P>(0) + 64 * q;
      t[q]               = tokens[mine];
      if (mine >= ids.m) t[q].place = -1;
    }
    lds_barrier();
  }
}

/** The numbers of a tile's tokens of each digit: tiles [n_tiles, kDigits]; workgroups behind those fill. */
template <int P>
__global__ __launch_bounds__(kSortThreads) void count_digits_kernel(row_ids ids, unsigned n, const token* in, digit d,
                                                                    int* tiles, unsigned n_tiles, fill_share share)
{
  if (blockIdx.x >= n_tiles) return fill(share, blockIdx.x - n_tiles);
  __shared__ int counts[kDigits];
  if (threadIdx.x < kDigits) counts[threadIdx.x] = 0;
  lds_barrier();
  token t[P];
  read_tile<P>(ids, n, in, int64_t{blockIdx.x} * (kSortThreads * P), t);
#pragma unroll
  for (int q = 0; q < P; ++q)
    if (t[q].place >= 0) atomicAdd(counts + d.of(t[q]), 1);
  lds_barrier();
  if (threadIdx.x < kDigits) tiles[int64_t{blockIdx.x} * kDigits + threadIdx.x] = counts[threadIdx.x];
}

constexpr int kFewTiles = 64;  // whose counts every workgroup adds up itself
constexpr int kScanDigits = 16, kScanGroups = kSortThreads / kScanDigits;

/** Turns the counts of tiles into those of all tiles before each, and their sums into one more row; kScanDigits digits a
 * workgroup, a share of the tiles each of its groups of threads. */
__global__ __launch_bounds__(kSortThreads) void scan_tiles_kernel(int* tiles, unsigned n_tiles)
{
  __shared__ int sums[kScanGroups][kScanDigits];
  const int group = static_cast<int>(threadIdx.x) / kScanDigits, mine = static_cast<int>(threadIdx.x) % kScanDigits;
  int* const column   = tiles + blockIdx.x * kScanDigits + mine;
  const int64_t width = (int64_t{n_tiles} + kScanGroups - 1) / kScanGroups;
  const int64_t b0 = min(group * width, int64_t{n_tiles}), b1 = min(b0 + width, int64_t{n_tiles});
  int sum = 0;
#pragma unroll 8
  for (int64_t b = b0; b < b1; ++b)
    sum += column[b * kDigits];
  sums[group][mine] = sum;
  lds_barrier();
  int before = 0, all = 0;
  for (int g = 0; g < kScanGroups; ++g) {
    before += g < group ? sums[g][mine] : 0;
    all += sums[g][mine];
  }
#pragma unroll 8
  for (int64_t b = b0; b < b1; ++b) {
    const int count     = column[b * kDigits];
    column[b * kDigits] = before;
    before += count;
  }
  if (group == 0) column[int64_t{n_tiles} * kDigits] = all;
}

/** Moves a tile's tokens to their places by one digit; of up to kFewTiles tiles every workgroup adds up the counts itself, else
 * scan_tiles_kernel has. */
template <int P>
__global__ __launch_bounds__(kSortThreads) void move_tokens_kernel(row_ids ids, unsigned n, const token* in, digit d,
                                                                   const int* tiles, token* out, unsigned n_tiles,
                                                                   fill_share share)
{
  if (blockIdx.x >= n_tiles) return fill(share, blockIdx.x - n_tiles);
  __shared__ int counts[kSortWaves][kDigits];
  __shared__ int sums[kDigits / 64];
  token t[P];
  int rank[P], c[kSortWaves];
  read_tile<P>(ids, n, in, int64_t{blockIdx.x} * (kSortThreads * P), t);
  clear_counts(counts);
  int before = 0, all = 0;
  if (threadIdx.x < kDigits && n_tiles > kFewTiles) {
    before = tiles[int64_t{blockIdx.x} * kDigits + threadIdx.x];
    all    = tiles[int64_t{n_tiles} * kDigits + threadIdx.x];
  } else if (threadIdx.x < kDigits) {
#pragma unroll 16
    for (unsigned b = 0; b < n_tiles; ++b) {
      const int count = tiles[int64_t{b} * kDigits + threadIdx.x];
      all += count;
      before += b < blockIdx.x ? count : 0;
    }
  }
  const int base = scan_digits(all, sums) + before;
  rank_tile<P>(t, d, counts, rank);
  lds_barrier();
  (void)wave_counts(counts, c);
  start_waves(counts, c, base);
  lds_barrier();
#pragma unroll
  for (int q = 0; q < P; ++q)
    if (t[q].place >= 0) out[counts[threadIdx.x / 64][d.of(t[q])] + rank[q]] = t[q];
}

// ---- the sums of sorted tokens

/** Sorted tokens [m] in chunks of `width`.  A run (the tokens of one row) that ends in the chunk behind its first token's, or
 * before, is that first chunk's; a longer one is cut at the borders, and its chunks leave their sums in cut [chunk][2][d]: of a
 * run that came from before at 0, of one that begins here at 1. */
struct sorted_tokens {
  const token* t;
  int64_t m;
  unsigned n;
  int width;
  float* cut;

  /** The row of a token, of the first or last one for places that there are not. */
  __device__ auto row(int64_t i) const -> unsigned { return t[max(min(i, m - 1), int64_t{0})].row; }
};

/** What a chunk [b, e) has to do with the runs at its borders. */
struct chunk_runs {
  int64_t b, e;
  unsigned first, last;  // rows of its first and last token
  bool before;           // the first run came from the chunk before
  bool head;             // and is cut
  bool tail;             // the last run begins here and is cut
  bool goes_on;          // the last run begins here and ends in the next chunk

  __device__ chunk_runs(sorted_tokens const& s, int64_t chunk)
  {
    b = chunk * s.width, e = min(b + s.width, s.m);
    first = s.row(b), last = s.row(e - 1);
    const unsigned back = s.row(b - 1), far_back = s.row(b - s.width - 1), ahead = s.row(e), far_ahead = s.row(e + s.width);
    before             = b > 0 && back == first && first < s.n;
    const bool crosses = e < s.m && ahead == last && last < s.n;
    const bool through = before && crosses && first == last;  // the whole chunk is a cut run's
    head               = before && (through || (b > s.width && far_back == first));
    tail               = crosses && !through && e + s.width < s.m && far_ahead == last;
    goes_on            = crosses && !through && !tail;
  }
};

constexpr int kTokensAhead = 8;  // whose gradients a team has on their way

/** The same in every lane: of teams of 64 lanes, in a scalar register. */
template <int W, typename V>
__device__ inline auto of_team(V v) -> V
{
  if constexpr (W == 64) return static_cast<V>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
  return v;
}

/** Tokens [p, p + kTokensAhead), the last one again past the end. */
template <int W>
__device__ inline void read_tokens(sorted_tokens const& s, int64_t p, token (&t)[kTokensAhead])
{
#pragma unroll
  for (int q = 0; q < kTokensAhead; ++q)
    t[q] = s.t[min(p + q, s.m - 1)];
}

/** The end of the run of `row` that holds place p, or `end`; a team's lanes look side by side. */
template <int W>
__device__ inline auto run_end(sorted_tokens const& s, int64_t p, int64_t end, unsigned row) -> int64_t
{
  const int lane = threadIdx.x % 64, sub = lane % W;
  for (;; p += W) {
    const unsigned long long in = __ballot(p + sub < end && s.row(p + sub) == row) >> (lane - sub);
    const int n                 = __builtin_ctzll(~in | (W < 64 ? 1ull << (W % 64) : 0));
    if (W == 64 ? in != ~0ull : n < W) return p + n;
  }
}

/** Stores scale * sum, or what the row holds and that.  A column that two lanes have is added to by the one that has it first. */
template <bool kShort, typename O>
__device__ inline void write_sum(const float (&sum)[kUnit], float scale, bool add, O* row, int at, int d)
{
  if (at >= d) return;
  const int from = unit_start(at, d);
  float v[kUnit];
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    v[i] = sum[i] * scale;
  if (!add) return store_unit<kShort>(row, v, from, d, true);
  float old[kUnit];
  unpack_unit(load_unit<kShort>(row, from, d), old);
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    v[i] += old[i];
  if (from == at) return store_unit<kShort>(row, v, from, d, true);
  for (int i = 0; i < kUnit; ++i)
    if (from + i >= at) row[from + i] = static_cast<O>(v[i]);
}

/** Sets the elements [j0, j1) of d-wide dense rows to 0 whose row is not used; the first of them is in row r, at col. */
template <typename O>
__device__ inline void clear_elements(const bool* used, O* x, int j0, int j1, int r, int col, int d)
{
  for (int j = j0; j < j1; ++j) {
    for (; col >= d; col -= d)
      ++r;
    if (!used[r]) x[j] = static_cast<O>(0.f);
    ++col;
  }
}

/**
 * Sets the rows [v0, v0 + rows) that are not used (LDS, in v0's order) to 0.  Dense rows are one stretch of memory, in which a
 * wavefront's pieces of 16 bytes fill whole lines wherever rows begin; rows that lie apart are taken one by one.
 */
template <typename O>
__device__ inline void clear_rows(const bool* used, int64_t v0, int rows, int d, O* out, int64_t ostride)
{
  constexpr int N = kPer16<O>;
  O* const base   = out + v0 * ostride;
  if (ostride != d) {
    for (int r = 0; r < rows; ++r)
      for (int j = threadIdx.x; !used[r] && j < d; j += kThreads)
        base[r * ostride + j] = static_cast<O>(0.f);
    return;
  }
  const int total = rows * d, before = static_cast<int>(reinterpret_cast<uintptr_t>(base) % 1024 / sizeof(O));
  const int step_rows = kThreads * N / d, step_cols = kThreads * N - step_rows * d;
  int x = static_cast<int>(threadIdx.x) * N - before;
  if (x + N <= 0) x += kThreads * N;
  int r = max(x, 0) / d, col = x - r * d;  // below 0 where the first row begins inside the piece
  for (; x < total; x += kThreads * N) {
    const bool inside = x >= 0 && x + N <= total;
    if (inside && (col + N <= d ? !used[r] : N <= d && !used[r] && !used[r + 1])) {
      store16(base + x, uint4{0, 0, 0, 0});
    } else if (!inside || col + N > d) {
      const int j0 = max(-x, 0);
      clear_elements(used, base + x, j0, min(N, total - x), r, col + j0, d);
    }
    r += step_rows;
    col += step_cols;
    if (col >= d) col -= d, ++r;
    for (; col < 0; col += d)
      --r;
  }
}

/** Rows [first, n), `rows` a workgroup from `block0` on, that are set to 0 beside the sums where no token has them. */
struct clear_share {
  unsigned block0;
  int64_t first;
  int rows;
};

/** The first of the sorted tokens whose row is `row` or behind it; the lanes of a wavefront look at 64 places at a time. */
__device__ inline auto first_at_least(sorted_tokens const& s, int64_t row) -> int64_t
{
  int64_t lo = 0, hi = s.m;
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + threadIdx.x % 64 * step;
    const int before   = __popcll(__ballot(at < hi && s.t[min(at, s.m - 1)].row < row));
    if (before == 0) break;
    hi = min(lo + before * step, hi);
    lo += (before - 1) * step + 1;
  }
  return lo;
}

/** Whether one of the tokens [lo, hi) has the row. */
__device__ inline auto has_row(sorted_tokens const& s, int64_t lo, int64_t hi, unsigned row) -> bool
{
  const int64_t end = hi;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (s.t[mid].row < row)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo < end && s.t[lo].row == row;
}

/** Sets the rows of a workgroup's share that no token has to 0.  It marks its tokens' rows, or, where they are many more than its
 * rows (a common token's), looks for each row among them. */
template <typename O>
__device__ inline void clear_unlisted(sorted_tokens const& s, clear_share const& c, int d, O* out, int64_t ostride, bool* used,
                                      int64_t* range)
{
  const int64_t v0 = c.first + int64_t{blockIdx.x - c.block0} * c.rows;
  const int rows   = static_cast<int>(min(int64_t{s.n} - v0, int64_t{c.rows}));
  const int wave   = static_cast<int>(threadIdx.x) / 64;
  for (int r = threadIdx.x; r < rows; r += kThreads)
    used[r] = false;
  if (wave < 2) {
    const int64_t at = first_at_least(s, v0 + (wave == 0 ? 0 : rows));
    if (threadIdx.x % 64 == 0) range[wave] = at;
  }
  lds_barrier();
  const int64_t lo = range[0], hi = range[1];
  if (hi - lo <= int64_t{16} * kThreads * ((rows + kThreads - 1) / kThreads)) {
    for (int64_t p = lo + threadIdx.x; p < hi; p += kThreads)
      used[s.t[p].row - v0] = true;
  } else {
    for (int r = threadIdx.x; r < rows; r += kThreads)
      used[r] = has_row(s, lo, hi, static_cast<unsigned>(v0 + r));
  }
  lds_barrier();
  clear_rows(used, v0, rows, d, out, ostride);
}

/**
 * The sums of the runs of a chunk each, by teams of W lanes, a unit a lane (of one of `slices` slices of their columns), the
 * gradients of kTokensAhead tokens on their way at a time.  Workgroups behind those clear rows.
 */
template <typename T, typename O, int W>
__global__ __launch_bounds__(kThreads) void sum_runs_kernel(sorted_tokens s, const T* grad, int64_t gstride, int d, float scale,
                                                            bool add, O* out, int64_t ostride, unsigned slices, clear_share clear)
{
  constexpr int kTeams = kThreads / W;
  if (blockIdx.x >= clear.block0) {
    __shared__ bool used[kClearRows];
    __shared__ int64_t range[2];
    return clear_unlisted(s, clear, d, out, ostride, used, range);
  }
  const int64_t team   = int64_t{blockIdx.x} * kTeams + of_team<W>(static_cast<int>(threadIdx.x) / W);
  const int64_t chunk  = team / slices;  // a workgroup's teams take slices side by side
  const int at         = (static_cast<int>(team - chunk * slices) * W + static_cast<int>(threadIdx.x) % W) * kUnit;
  if (chunk * s.width >= s.m) return;  // a team's lanes without a column go along, and write nothing
  const chunk_runs c(s, chunk);
  if (c.first >= s.n) return;  // padding, to the end
  const int from = unit_start(at, d);
  float* cut     = s.cut + chunk * 2 * d;
  float sum[kUnit];
  unit<T> u[kTokensAhead];
  token t[kTokensAhead];
  // the gradients of the tokens in hand; of those that are not taken the first one's again
  const auto load = [&](const bool (&taken)[kTokensAhead]) {
#pragma unroll
    for (int q = 0; q < kTokensAhead; ++q)
      u[q] = load_unit<W == 1>(grad + of_team<W>(taken[q] ? t[q].place : t[0].place) * gstride, from, d);
  };
  // the part of a cut run that lies in this chunk from p on; returns its end
  const auto sum_part = [&](int64_t p, unsigned row, float* to) {
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      sum[i] = 0.f;
    for (bool more = true; more; p += kTokensAhead) {
      read_tokens<W>(s, p, t);
      bool taken[kTokensAhead];
#pragma unroll
      for (int q = 0; q < kTokensAhead; ++q)
        taken[q] = p + q < c.e && t[q].row == row;
      load(taken);
#pragma unroll
      for (int q = 0; q < kTokensAhead; ++q) {
        float v[kUnit];
        unpack_unit(u[q], v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] += taken[q] ? v[i] : 0.f;
      }
      more = taken[kTokensAhead - 1];
    }
    write_sum<W == 1>(sum, 1.f, false, to, at, d);
  };
  int64_t p = c.b;
  if (c.head) sum_part(p, c.first, cut);
  if (c.before) p = run_end<W>(s, p, c.e, c.first);  // of a run that is not cut the chunk before has all
  const auto taken_at = [&](int64_t i, unsigned row) {
    return row < s.n && (i < c.e ? !(c.tail && row == c.last) : i < s.m && c.goes_on && row == c.last);
  };
  token next[kTokensAhead];
  read_tokens<W>(s, p, next);
  unsigned current = ~0u;
  bool full         = true;  // so far
  while (full && taken_at(p, next[0].row)) {
    bool taken[kTokensAhead];
#pragma unroll
    for (int q = 0; q < kTokensAhead; ++q) {
      t[q]     = {of_team<W>(next[q].row), of_team<W>(next[q].place)};
      taken[q] = taken_at(p + q, t[q].row);
    }
    load(taken);
    read_tokens<W>(s, p + kTokensAhead, next);
#pragma unroll
    for (int q = 0; q < kTokensAhead; ++q) {
      if (!taken[q]) break;
      ++p;
      float v[kUnit];
      unpack_unit(u[q], v);
      const bool same = t[q].row == current;
      if (!same && current != ~0u) write_sum<W == 1>(sum, scale, add, out + current * ostride, at, d);
      current = t[q].row;
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
        sum[i] = same ? sum[i] + v[i] : v[i];
    }
    full = taken[kTokensAhead - 1];
  }
  if (current != ~0u) write_sum<W == 1>(sum, scale, add, out + current * ostride, at, d);
  if (c.tail) sum_part(p, c.last, cut + d);
}

constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;
constexpr int kJoinLanes = 32, kJoinTeams = kJoinThreads / kJoinLanes;
constexpr int kPartsAhead = 4;

/**
 * Joins the sums of the runs that begin in the chunks of a workgroup, one a wavefront to look at, and are cut; kJoinLanes units of
 * their columns (one of `slices` slices) a workgroup, whose teams take parts in turn, kPartsAhead of them on their way.  A common
 * token's run, or that of a batch's padding where it is a row of the table, has many: 65,536 tokens of 512 bfloat16 values, half of
 * them equal, take 67 us, and 222 where a workgroup of wavefronts for 512 columns each goes from part to part.
 */
template <typename O, bool kShort>
__global__ __launch_bounds__(kJoinThreads) void join_runs_kernel(sorted_tokens s, int d, float scale, bool add, O* out,
                                                                 int64_t ostride, int64_t chunks, unsigned slices, int64_t block0)
{
  __shared__ float sums[kJoinWaves][kUnit][kJoinLanes];
  __shared__ unsigned rows[kJoinWaves];
  __shared__ int64_t lasts[kJoinWaves];  // the chunks that the runs end in
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, sub = lane % kJoinLanes;
  const int64_t group = (block0 + blockIdx.x) / slices, chunk0 = group * kJoinWaves;
  const int at = (static_cast<int>(block0 + blockIdx.x - group * slices) * kJoinLanes + sub) * kUnit;
  unsigned mine = ~0u;
  if (chunk0 + wave < chunks) {
    const chunk_runs c(s, chunk0 + wave);
    if (c.tail) {
      mine               = c.last;
      const int64_t last = (first_at_least(s, int64_t{c.last} + 1) - 1) / s.width;
      if (lane == 0) lasts[wave] = last;
    }
  }
  if (lane == 0) rows[wave] = mine;
  lds_barrier();
  for (int j = 0; j < kJoinWaves; ++j) {
    const unsigned row = rows[j];
    if (row == ~0u) continue;
    const int64_t chunk = chunk0 + j, last = lasts[j];
    float sum[kUnit];
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      sum[i] = 0.f;
    for (int64_t p = chunk + threadIdx.x / kJoinLanes; p <= last; p += kJoinTeams * kPartsAhead) {
      unit<float> u[kPartsAhead];
#pragma unroll
      for (int q = 0; q < kPartsAhead; ++q) {
        const int64_t part = min(p + q * kJoinTeams, last);
        u[q] = load_unit<kShort>(s.cut + (part * 2 + (part == chunk ? 1 : 0)) * d, unit_start(at, d), d);
      }
#pragma unroll
      for (int q = 0; q < kPartsAhead; ++q) {
        float v[kUnit];
        unpack_unit(u[q], v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] += p + q * kJoinTeams <= last ? v[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      sum[i] += __shfl_xor(sum[i], kJoinLanes);
      if (lane < kJoinLanes) sums[wave][i][lane] = sum[i];
    }
    lds_barrier();
    if (threadIdx.x < kJoinLanes) {
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] += sums[w][i][lane];
      write_sum<kShort>(sum, scale, add, out + row * ostride, at, d);
    }
    lds_barrier();
  }
}

constexpr int kFewTokens = 1024, kSomeTokens = 4096;
constexpr int kLongRun = 4 * kTokensAhead;  // by one team 120 equal tokens of 1024 took 13.7 us, by all 9.4

/**
 * The same for up to M tokens without sorting them: a team a token looks through all of them, W at a time, and the first one of a
 * row lists the places of the others and adds up their gradients; those of more than kLongRun (a common token's) all teams of the
 * workgroup add up.  Workgroups from `sum_blocks` on clear rows, `clear` each, whose flags (a byte a row) fit in the words of
 * `rows`.
 */
template <typename T, typename O, int W, bool kShort, int M>
__global__ __launch_bounds__(kThreads) void sum_few_kernel(row_ids ids, unsigned n, const T* grad, int64_t gstride, int d,
                                                           float scale, bool add, O* out, int64_t ostride, unsigned slices,
                                                           unsigned sum_blocks, int clear)
{
  constexpr int kTeams = kThreads / W, kPer = M / kThreads, kLooks = M / kFewTokens;
  __shared__ unsigned rows[std::max(M, kUnit * kThreads)];
  __shared__ unsigned short places[kTeams][M];
  __shared__ int counts[kTeams];
  const int m = static_cast<int>(ids.m);
  int64_t id[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q)
    id[q] = -1;
  if (m > 0) read_ids(ids, threadIdx.x, kThreads, id);
  if (blockIdx.x >= sum_blocks) {
    bool* used       = reinterpret_cast<bool*>(rows);
    const int64_t v0 = int64_t{blockIdx.x - sum_blocks} * clear;
    const int mine   = static_cast<int>(min(int64_t{n} - v0, int64_t{clear}));
    for (int r = threadIdx.x; r < mine; r += kThreads)
      used[r] = false;
    lds_barrier();
#pragma unroll
    for (int q = 0; q < kPer; ++q)
      if (id[q] >= v0 && id[q] < v0 + mine) used[id[q] - v0] = true;
    lds_barrier();
    return clear_rows(used, v0, mine, d, out, ostride);
  }
#pragma unroll
  for (int q = 0; q < kPer; ++q)
    rows[threadIdx.x + q * kThreads] = static_cast<int>(threadIdx.x) + q * kThreads < m ? row_of(id[q], n) : ~0u;
  lds_barrier();
  const int team = static_cast<int>(threadIdx.x) / W, lane = threadIdx.x % 64, sub = lane % W;
  // a workgroup's teams have one slice, so that a long run's slices are different workgroups'
  const int token    = static_cast<int>(blockIdx.x / slices) * kTeams + team;
  const int at       = (static_cast<int>(blockIdx.x % slices) * W + sub) * kUnit;
  const unsigned row = token < m ? rows[token] : n;
  const auto above = [&](unsigned long long lanes) { return W == 64 ? lanes : lanes >> (lane - sub) & ((1ull << (W % 64)) - 1); };
  int count = 0;
  for (int i = 0; i < m && row < n; i += W * kLooks) {
    bool in[kLooks], earlier = false;
#pragma unroll
    for (int q = 0; q < kLooks; ++q)
      in[q] = rows[i + q * W + sub] == row;
#pragma unroll
    for (int q = 0; q < kLooks; ++q) {
      const auto same = above(__ballot(in[q]));
      if (same == 0) continue;
      earlier = earlier || i + q * W + __builtin_ctzll(same) < token;
      if (in[q]) places[team][count + __popcll(same & ((1ull << sub) - 1))] = static_cast<unsigned short>(i + q * W + sub);
      count += __popcll(same);
    }
    if (earlier) {  // that token's team has the row
      count = 0;
      break;
    }
  }
  if (sub == 0) counts[team] = count;
  float sum[kUnit];
  // the gradients of kTokensAhead of every `step` listed places, from `first` on
  const auto add_up = [&](const unsigned short* list, int length, int first, int step, int from) {
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      sum[i] = 0.f;
    for (int j = first; j < length; j += step) {
      unit<T> u[kTokensAhead];
#pragma unroll
      for (int q = 0; q < kTokensAhead; ++q)
        u[q] = load_unit<kShort>(grad + of_team<W>(static_cast<int>(list[min(j + q, length - 1)])) * gstride, from, d);
#pragma unroll
      for (int q = 0; q < kTokensAhead; ++q) {
        float v[kUnit];
        unpack_unit(u[q], v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] += j + q < length ? v[i] : 0.f;
      }
    }
  };
  wave_fence();
  if (count > 0 && count <= kLongRun) {
    add_up(places[team], count, 0, kTokensAhead, unit_start(at, d));
    write_sum<kShort>(sum, scale, add, out + row * ostride, at, d);
  }
  lds_barrier();
  auto* const parts = reinterpret_cast<float(*)[kThreads]>(rows);  // the rows of tokens make room
  for (int t = 0; t < kTeams; ++t) {
    if (counts[t] <= kLongRun) continue;
    add_up(places[t], counts[t], team * kTokensAhead, kTeams * kTokensAhead, unit_start(at, d));
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      parts[i][threadIdx.x] = sum[i];
    lds_barrier();
    if (team == t) {
      for (int other = 0; other < kTeams; ++other)
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
          sum[i] = (other == 0 ? 0.f : sum[i]) + parts[i][other * W + sub];
      write_sum<kShort>(sum, scale, add, out + row * ostride, at, d);
    }
    lds_barrier();
  }
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

/** Calls f with the lanes of a row's team: its units, or 64 of them a slice; one for rows shorter than a unit. */
template <int U = kUnit, typename F>
void with_team(int64_t d, F f)
{
  const int64_t units = (d + U - 1) / U;
  if (d < U)
    f(std::integral_constant<int, 1>{});
  else if (units <= 8)
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

/** Whether a gradient's tokens are looked through, by every slice of every token, and not sorted: one launch in place of three to
 * six.  Of even ids, of those of text (the i-th commonest as 1 / i), and with half or all of them equal (a padded batch's), sorted
 * in brackets: 32,000 x 512 bfloat16 from 3000 tokens 16, 16, 48, 83 us (27, 33, 30, 26), 8000 x 512 from 4096 15, 19, 55, 101 (25,
 * 31, 30, 25), 8000 x 2000 from 2896, near the bound, 30, 29, 47, 83 (27, 32, 32, 26).  Which ids they are is not known here:
 * batches of one token pay for the others, and still take less than torch's additions by atomics (126, 134, 127 where all are
 * equal). */
auto takes_few(int64_t m, int64_t d) -> bool
{
  return m <= kFewTokens || (m <= kSomeTokens && m * m * ceil_div(d, 64 * kUnit) <= int64_t{1} << 25);
}

/** How the workspace is laid out, from place to place in bytes. */
struct sort_layout {
  int passes, bits, per;  // of a digit; tokens of a thread
  int64_t tiles, chunks, second, counts, cut, end;
};

auto layout_of(int64_t m, int64_t n, int64_t d) -> sort_layout
{
  const auto up = [](int64_t v) { return ceil_div(v, 256) * 256; };
  sort_layout l{};
  if (takes_few(m, d)) return l;
  int bits = 1;
  while (n >> bits != 0)
    ++bits;
  l.passes        = static_cast<int>(ceil_div(bits, kDigitBits));
  l.bits          = static_cast<int>(ceil_div(bits, l.passes));
  l.per           = m <= 2 * kSortThreads ? 2 : m <= 4 * kSortThreads ? 4 : m <= 8 * kSortThreads ? 8 : m <= 65536 ? 2 : 8;
  l.tiles         = ceil_div(m, l.per * kSortThreads);
  const int width = chunk_width(m, d);
  l.chunks        = ceil_div(m, width);
  l.second        = up(m * static_cast<int64_t>(sizeof(token)));
  l.counts        = l.tiles > 1 ? 2 * l.second : l.second;
  l.cut           = l.counts + (l.tiles > 1 ? up((l.tiles + 1) * kDigits * 4) : 0);
  l.end           = l.cut + l.chunks * 2 * d * 4;
  return l;
}

/** Sorts the tokens, and fills [out, out + bytes) meanwhile. */
template <int P>
void sort_tiles(row_ids const& ids, unsigned n, sort_layout const& l, token* tokens, token* second, int* counts, char* out,
                int64_t bytes, hipStream_t s)
{
  const auto tiles = static_cast<unsigned>(l.tiles);
  const int steps  = tiles == 1 ? 1 : 2 * l.passes;
  const int64_t per_step = ceil_div(ceil_div(bytes, steps), kFillBytes) * kFillBytes;
  const auto share = [&](int step) {
    const int64_t first = std::min(step * per_step, bytes), own = std::min(per_step, bytes - first);
    // where a share begins inside a piece it takes one more
    return fill_share{out + first, own,
                      own > 0 ? static_cast<unsigned>(std::min<int64_t>(ceil_div(own + 16, kFillBytes), 1 << 20)) : 0u};
  };
  if (tiles == 1) {
    const auto f = share(0);
    sort_alone_kernel<P><<<1 + f.blocks, kSortThreads, 0, s>>>(ids, n, l.passes, l.bits, tokens, f);
    OCTEX_HIP(hipGetLastError());
    return;
  }
  for (int p = 0; p < l.passes; ++p) {
    const bool to_first = (l.passes - 1 - p) % 2 == 0;
    const token* in     = p == 0 ? nullptr : to_first ? second : tokens;
    const digit of{p * l.bits, l.bits};
    const auto f = share(2 * p), g = share(2 * p + 1);
    count_digits_kernel<P><<<tiles + f.blocks, kSortThreads, 0, s>>>(ids, n, in, of, counts, tiles, f);
    OCTEX_HIP(hipGetLastError());
    if (tiles > kFewTiles) {
      scan_tiles_kernel<<<kDigits / kScanDigits, kSortThreads, 0, s>>>(counts, tiles);
      OCTEX_HIP(hipGetLastError());
    }
    move_tokens_kernel<P><<<tiles + g.blocks, kSortThreads, 0, s>>>(ids, n, in, of, counts, to_first ? tokens : second, tiles, g);
    OCTEX_HIP(hipGetLastError());
  }
}

/** The bytes that are filled while the tokens are sorted, in about the time that this takes on few CUs: 4.6 us and 6.7 to count and
 * to move tiles of 2048 tokens that all run at once (more tiles take longer, and fill the same), 8 to 18 for 2 to 8 tokens a thread
 * of a single workgroup.  128,000 x 4096 bfloat16 from 32,768 tokens: 276 us, 303 if all of the table is filled there, and the
 * tokens' rows are written twice (64 MB a pass: 278, 160 MB: 278). */
auto fill_bytes(sort_layout const& l) -> int64_t
{
  return l.tiles == 1 ? (int64_t{l.per} + 4) * (14 << 20) : int64_t{l.passes} * (96 << 20);
}

}  // namespace

void launch_embed(table_rows const& table, row_ids const& ids, int64_t d, float scale, value_rows const& out, hipStream_t s)
{
  const auto run = [&](auto t) {
    using T = decltype(t);
    with_type(out.type, [&](auto o) {
      using O = decltype(o);
      with_team<kResultUnit<O>>(d, [&](auto lanes) {
        constexpr int W      = lanes();
        const auto slices    = static_cast<unsigned>(ceil_div(d, W * kResultUnit<O>));
        const int64_t blocks = ceil_div(ceil_div(ids.m, kRowsAhead) * slices, kThreads / W);
        for (int64_t first = 0; first < blocks; first += kMaxGrid) {
          embed_kernel<T, O, W><<<static_cast<unsigned>(std::min(kMaxGrid, blocks - first)), kThreads, 0, s>>>(
            table, ids, static_cast<int>(d), scale, static_cast<O*>(out.x), out.stride, passes_cache(ids.m, d, out.type), slices,
            first);
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

auto embed_backward_workspace(int64_t m, int64_t n, int64_t d) -> int64_t { return layout_of(m, n, d).end; }

void launch_embed_backward(value_rows const& grad, row_ids const& ids, int64_t n, int64_t d, float scale, bool add,
                           value_rows const& out, void* workspace, hipStream_t s)
{
  const auto rows  = static_cast<unsigned>(n);
  const auto width = static_cast<int>(d);
  const bool few = takes_few(ids.m, d), fewer = ids.m <= kFewTokens;
  // of few tokens: rows that a workgroup clears, 16 KB of them, or 64 KB where it reads more ids for that
  const int64_t least = (fewer ? 16 << 10 : 64 << 10) / (d * elem_size(out.type));
  const int clear     = static_cast<int>(
    std::clamp<int64_t>(std::max(least, ceil_div(n, 1 << 22)), 1, fewer ? kFewTokens : kSomeTokens));
  const auto clears = add || !few ? 0u : static_cast<unsigned>(ceil_div(n, clear));
  const auto l      = layout_of(ids.m, n, d);
  auto* base        = static_cast<char*>(workspace);
  const sorted_tokens sorted{reinterpret_cast<token*>(base), ids.m, rows, chunk_width(ids.m, d),
                             reinterpret_cast<float*>(base + l.cut)};
  // of many: rows that are filled beside the sort, wherever tokens are, and those that are cleared after it
  const int64_t row_bytes = d * elem_size(out.type);
  const int64_t filled    = add || few || out.stride != d ? 0 : std::min(n, fill_bytes(l) / row_bytes);
  const int64_t left      = add || few ? 0 : n - filled;
  const int64_t per_group = rows_to_clear(left, row_bytes);
  with_type(out.type, [&](auto o) {
    using O = decltype(o);
    O* to   = static_cast<O*>(out.x);
    if (!few) {
      const auto sort = l.per == 2 ? sort_tiles<2> : l.per == 4 ? sort_tiles<4> : sort_tiles<8>;
      sort(ids, rows, l, reinterpret_cast<token*>(base), reinterpret_cast<token*>(base + l.second),
           reinterpret_cast<int*>(base + l.counts), static_cast<char*>(out.x),
           filled * row_bytes, s);
    }
    with_type(grad.type, [&](auto t) {
      using T       = decltype(t);
      const T* from = static_cast<const T*>(grad.x);
      with_team(d, [&](auto lanes) {
        constexpr int W   = lanes();
        constexpr int F   = std::max(W, 8);
        const auto slices = static_cast<unsigned>(ceil_div(d, W == 1 ? kUnit : W * kUnit));
        const int team    = !few ? W : fewer ? F : 64;
        const int teams   = kThreads / team;
        const auto sums   = static_cast<unsigned>(few ? ceil_div(ids.m, teams) * slices : ceil_div(l.chunks * slices, teams));
        const auto launch_few = [&](auto kernel) {
          kernel<<<sums + clears, kThreads, 0, s>>>(ids, rows, from, grad.stride, width, scale, add, to, out.stride, slices, sums,
                                                    clear);
        };
        if (fewer)
          launch_few(sum_few_kernel<T, O, F, W == 1, kFewTokens>);
        else if (few && ids.m <= kSomeTokens / 2)
          launch_few(sum_few_kernel<T, O, 64, W == 1, kSomeTokens / 2>);
        else if (few)
          launch_few(sum_few_kernel<T, O, 64, W == 1, kSomeTokens>);
        else
          sum_runs_kernel<T, O, W><<<sums + static_cast<unsigned>(ceil_div(left, per_group)), kThreads, 0, s>>>(
            sorted, from, grad.stride, width, scale, add, to, out.stride, slices, {sums, filled, static_cast<int>(per_group)});
        OCTEX_HIP(hipGetLastError());
      });
    });
    const auto slices   = static_cast<unsigned>(ceil_div(d, kJoinLanes * kUnit));
    const int64_t joins = ceil_div(l.chunks, kJoinWaves) * slices;
    for (int64_t first = 0; first < joins; first += kMaxGrid) {
      const auto join = d < kUnit ? join_runs_kernel<O, true> : join_runs_kernel<O, false>;
      join<<<static_cast<unsigned>(std::min(kMaxGrid, joins - first)), kJoinThreads, 0, s>>>(sorted, width, scale, add, to,
                                                                                             out.stride, l.chunks, slices, first);
      OCTEX_HIP(hipGetLastError());
    }
  });
}

}  // namespace cuvs::neighbors::octex::detail
