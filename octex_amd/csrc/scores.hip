// Scores in 8-bit integers: out[i][j] = qs[i] rs[j] sum_d q[i][d] r[j][d] + bias[j], the sums exact in int32.

#include "common.hpp"
#include "elems_device.hpp"
#include "scores.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace cuvs::neighbors::octex::detail {

namespace {

using i32x4  = int __attribute__((ext_vector_type(4)));
using i32x16 = int __attribute__((ext_vector_type(16)));

// ---- quantization of rows

constexpr int kQuantThreads = 256;

/** A magnitude's bits, which order as it does, with infinity and NaN above every finite one. */
__device__ inline auto magnitude(float v) -> unsigned { return __float_as_uint(v) & 0x7fffffffu; }

/** The 127th part of a magnitude, as the product with 1 / 127 in fp32: what torch's division by a number makes on the GPU, so
 * that its plain expression there has the same codes.  A quotient (torch's on the CPU, numpy's) is another scale by one unit in
 * 4 to 5 % of rows, and then another code for one value in 9 million of float32, 200,000 of float16 and 57,000 of bfloat16,
 * whose quotients more often lie at the middle of two whole numbers; with either, codes are nearest to x / scale. */
__device__ inline auto scale_of(unsigned top) -> float
{
  return top < 0x7f800000u ? __uint_as_float(top) * (1.f / 127.f) : NAN;
}

/**
 * The codes of v: v / scale, rounded to fp32, then to a whole number.  The product with 1 / scale is at most 3 units in the
 * last place from the quotient, 2.3e-5 where it is below 128, and rounds alike unless it lies as near to the middle of two
 * whole numbers: then, or if 1 / scale is no finite number, the divisions are made.  8192 x 4096 bfloat16: 23.5 us, with all
 * divided 29.
 */
template <int N>
__device__ inline void codes_of(const float (&v)[N], float scale, float inverse, int8_t (&c)[N])
{
  float code[N], far = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float q = v[i] * inverse;
    code[i]       = rintf(q);
    far           = fmaxf(far, fabsf(q - code[i]));
  }
  if (!(inverse < INFINITY && far < 0.5f - 3e-5f)) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      code[i] = scale > 0.f ? fminf(fmaxf(rintf(v[i] / scale), -127.f), 127.f) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    c[i] = static_cast<int8_t>(static_cast<int>(code[i]));
}

template <int W>
__device__ inline auto max_lanes(unsigned top) -> unsigned
{
#pragma unroll
  for (int mask = W / 2; mask > 0; mask >>= 1)
    top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), mask)));
  return top;
}

__device__ inline auto block_max(unsigned top, unsigned* parts) -> unsigned
{
  top = max_lanes<64>(top);
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = top;
  lds_barrier();
  for (int w = 0; w < static_cast<int>(blockDim.x) / 64; ++w)
    top = max(top, parts[w]);
  return top;
}

struct product {
  int8_rows q, r;
  int64_t m, n;
  int k;
  const float* bias;
  void* out;
  int64_t ostride;
};

__device__ inline auto score_of(int sum, float qs, product const& p, int64_t j) -> float
{
  return fmaf(static_cast<float>(sum) * qs, p.r.scales[j], p.bias != nullptr ? p.bias[j] : -0.f);
}

/** 16 values of a row at column at, those from k on 0. */
__device__ inline auto load_codes(const int8_t* row, int at, int k) -> i32x4
{
  i32x4 v = {0, 0, 0, 0};
  if (at + 16 <= k)
    __builtin_memcpy(&v, row + at, 16);
  else if (at < k) {
    int8_t e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
      e[i] = at + i < k ? row[at + i] : int8_t{0};
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

// ---- rows laid out anew: 16-byte chunks at aligned places, zeros after the last value

/** Rows x [n, k] that a kernel lays out at out, `pitch` apart; n = 0: none. */
struct pack_job {
  const int8_t* x;
  int64_t stride, n;
  int k;
  int8_t* out;
  int64_t pitch;
};

constexpr int kPackRows = 4;  // of a workgroup, a wavefront each

__device__ inline void pack_rows(pack_job const& p, int64_t first)
{
  const int64_t i = first + threadIdx.x / 64;
  if (i >= p.n) return;
  for (int at = static_cast<int>(threadIdx.x % 64) * 16; at < p.k; at += 64 * 16)
    *reinterpret_cast<i32x4*>(p.out + i * p.pitch + at) = load_codes(p.x + i * p.stride, at, p.k);
}

__global__ __launch_bounds__(64 * kPackRows) void pack_kernel(pack_job p, int64_t first)
{
  pack_rows(p, first + int64_t{blockIdx.x} * kPackRows);
}

/**
 * scale = max |x| / 127 (see scale_of); code = the whole number nearest to x / scale (ties to even), the quotient rounded to
 * fp32 first.
 * A row of zeros has scale 0 and codes 0; one with a NaN or an infinity has scale NaN and codes 0.
 *
 * kLanes threads hold a row of up to kHeld * kLanes 16-byte pieces in registers between the maximum and the codes, so that it
 * is read once; longer rows are read again.  Columns k .. pad are written as 0.  Workgroups past the rows' lay out `job`.
 * Bound by the rows' bytes: 100,000 x 960 float32 takes 86 us, 5.6 TB/s.
 */
template <typename T, int kLanes, int kHeld>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(const T* x, int64_t stride, int k, int pad, int8_t* codes,
                                                                 int64_t cstride, float* scales, int64_t row0, int64_t rows,
                                                                 unsigned blocks, pack_job job)
{
  constexpr int N = kPer16<T>, kStep = kLanes * N;
  static_assert(kQuantThreads == 64 * kPackRows);
  __shared__ unsigned parts[kQuantThreads / 64];
  if (blockIdx.x >= blocks) {
    pack_rows(job, int64_t{blockIdx.x - blocks} * kPackRows);
    return;
  }
  const int64_t r = row0 + int64_t{blockIdx.x} * (kQuantThreads / kLanes) + threadIdx.x / kLanes;
  const int lane  = threadIdx.x % kLanes, mine = lane * N;
  if (kLanes <= 64 && r >= row0 + rows) return;
  const T* row = x + r * stride;
  int8_t* out  = codes + r * cstride;
  uint4 held[kHeld];
  float v[N];
  unsigned top = 0;
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * kStep + mine < k) held[u] = load_row16(row, u * kStep + mine, k);
  const auto take = [&](uint4 raw) {  // 0 past the row
    unpack16<T>(raw, v);
#pragma unroll
    for (int i = 0; i < N; ++i)
      top = max(top, magnitude(v[i]));
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * kStep + mine < k) take(held[u]);
  for (int at = kHeld * kStep + mine; at < k; at += kStep)
    take(load_row16(row, at, k));
  if constexpr (kLanes <= 64)
    top = max_lanes<kLanes>(top);
  else
    top = block_max(top, parts);
  const float scale = scale_of(top), inverse = 1.f / scale;
  if (lane == 0) scales[r] = scale;
  const auto give = [&](uint4 raw, int at) {
    unpack16<T>(raw, v);
    int8_t c[N];
    codes_of(v, scale, inverse, c);
    if (at + N <= k) {
      __builtin_memcpy(out + at, c, N);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i < k) out[at + i] = c[i];
    }
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u * kStep + mine < k) give(held[u], u * kStep + mine);
  for (int at = kHeld * kStep + mine; at < k; at += kStep)
    give(load_row16(row, at, k), at);
  if (lane < pad - k) out[k + lane] = 0;
}

// ---- the product

constexpr int64_t kMaxInt8Stride = int64_t{1} << 22;  // a tile's 256 rows within 32-bit offsets

// ---- the product of few queries: every row's bytes are read once, by one wavefront

constexpr int kPiece = 256;  // bytes of a row that a wavefront multiplies at a time

/**
 * A workgroup scores RT * 16 rows for up to 16 queries; its KW wavefronts share the columns out and their sums meet in
 * LDS.  A matrix instruction takes 64 columns of 16 rows and 16 queries, so a lane loads 16 bytes of a row, and four such
 * loads cover whole 128-byte lines.  With kFused the queries are floats: the workgroup quantizes them into LDS first.
 *
 * Bound by the rows' bytes: 1 x 1024 x 32,000 (queries, values, rows), quantized on the way, takes 9.1 us, 3.6 TB/s; 16 x 4097 x
 * 100,000, whose rows lie at odd places, 275 us, 1.5 TB/s.
 */
template <int RT, int KW, bool kFused, typename Q, typename O>
__global__ __launch_bounds__(64 * KW) void few_scores_kernel(product p, const Q* floats, int64_t fstride, int pitch)
{
  extern __shared__ __align__(16) char few_lds[];
  __shared__ float qscales[16];
  __shared__ unsigned parts[KW];
  constexpr int kThreadsHere = 64 * KW;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, m = static_cast<int>(p.m);
  const int64_t j0 = int64_t{blockIdx.x} * RT * 16;
  int k0           = wave * kPiece;
  const int8_t* rows[RT];
  i32x4 acc[RT] = {}, b[RT][4];
#pragma unroll
  for (int y = 0; y < RT; ++y)
    rows[y] = p.r.x + min(j0 + 16 * y + lane % 16, p.n - 1) * p.r.stride;
  const auto load_rows = [&](int from) {
    if (from + kPiece <= p.k) {
#pragma unroll
      for (int y = 0; y < RT; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_memcpy(&b[y][i], rows[y] + from + 64 * i + 16 * (lane / 16), 16);
    } else if (from < p.k) {
#pragma unroll
      for (int y = 0; y < RT; ++y)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          b[y][i] = load_codes(rows[y], from + 64 * i + 16 * (lane / 16), p.k);
    }
  };
  load_rows(k0);  // they are on their way while the queries are quantized
  const auto load_query = [&](int at) {
    const int i = min(lane % 16, m - 1);
    if constexpr (!kFused) return load_codes(p.q.x + i * p.q.stride, at, p.k);
    // the codes in LDS end with zeros
    return at < pitch ? *reinterpret_cast<const i32x4*>(few_lds + i * pitch + at) : i32x4{0, 0, 0, 0};
  };
  if constexpr (kFused) {
    for (int i = 0; i < m; ++i) {
      const Q* row = floats + i * fstride;
      unsigned top = 0;
      for (int at = threadIdx.x; at < p.k; at += kThreadsHere)
        top = max(top, magnitude(static_cast<float>(row[at])));
      const float scale = scale_of(block_max(top, parts)), inverse = 1.f / scale;
      if (threadIdx.x == 0) qscales[i] = scale;
      for (int at = threadIdx.x; at < pitch; at += kThreadsHere) {
        const float v[1] = {at < p.k ? static_cast<float>(row[at]) : 0.f};
        int8_t c[1];
        codes_of(v, scale, inverse, c);
        few_lds[i * pitch + at] = static_cast<char>(c[0]);
      }
      lds_barrier();
    }
  } else {
    for (int i = threadIdx.x; i < m; i += kThreadsHere)
      qscales[i] = p.q.scales[i];
  }
  for (; k0 < p.k; k0 += KW * kPiece) {
    i32x4 a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      a[i] = load_query(k0 + 64 * i + 16 * (lane / 16));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int y = 0; y < RT; ++y)
        acc[y] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[y][i], acc[y], 0, 0, 0);
    load_rows(k0 + KW * kPiece);
  }
  auto* sums = reinterpret_cast<int*>(few_lds);  // [KW][16][RT * 16]
  constexpr int kWide = RT * 16, kAll = 16 * kWide;
  lds_barrier();
#pragma unroll
  for (int y = 0; y < RT; ++y)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      sums[wave * kAll + (4 * (lane / 16) + e) * kWide + 16 * y + lane % 16] = acc[y][e];
  lds_barrier();
  for (int e = threadIdx.x; e < m * kWide; e += kThreadsHere) {
    const int i = e / kWide;
    const int64_t j = j0 + e % kWide;
    if (j >= p.n) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < KW; ++w)
      sum += sums[w * kAll + e];
    static_cast<O*>(p.out)[i * p.ostride + j] = static_cast<O>(score_of(sum, qscales[i], p, j));
  }
}

// ---- the product of many rows: tiles of BM queries x BN rows, both operands' next 128 bytes loaded into LDS while the
// matrix cores work on these

constexpr unsigned kXcds = 8;

/** A grid of tiles in the order its workgroups take them. */
struct tile_order {
  unsigned tm, tn;  // tiles of queries and of rows
};

/** The tile of a workgroup.  Workgroups go round the 8 XCDs in turn; each XCD takes a run of consecutive tiles, and a run
 * goes through kBand tiles of queries before the next tile of rows, so that the tiles an XCD works on at a time share
 * operands in its L2. */
__device__ inline auto tile_of(unsigned b, tile_order o) -> uint2
{
  constexpr unsigned kBand = 4;
  const unsigned tiles = o.tm * o.tn, xcd = b % kXcds, each = tiles / kXcds, more = tiles % kXcds;
  const unsigned t     = xcd * each + min(xcd, more) + b / kXcds;
  const unsigned band = t / (kBand * o.tn), in = t % (kBand * o.tn), high = min(kBand, o.tm - band * kBand);
  return {band * kBand + in % high, in / high};
}

using rsrc_t = __amdgpu_buffer_rsrc_t;

/** Waits until at most N of the wavefront's loads are in flight, and with kLds until its LDS reads are back. */
template <int N, bool kLds = false>
__device__ inline void wait_loads()
{
  static_assert(N < 64);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (kLds ? 0 : 15) << 8 | (N >> 4) << 14);
  asm volatile("" ::: "memory");
}

/**
 * WM x WN wavefronts score TM x TN parts of 32 x 32 each, kStep values of the rows at a time, with kAhead steps on their way
 * from memory to LDS, which the loads fill without passing by registers.  Of a step, the next 32 values' operands are read
 * from LDS while the matrix cores multiply these; the loads are spread over the step, one or two a matrix instruction, and
 * are waited for by count, at the step's one barrier.
 *
 * Bound by power, as far as it is by one thing: 8192 x 4096 x 16,384 takes 500 us, 2200 TOP/s, with scales, rounding and all
 * (a library's bare product 498 us), the clock falls to 1.7 GHz and the matrix cores are busy for 62 % of its cycles; matrix
 * instructions alone reach 3000 to 3300 TOP/s.  A part of 4 x 2 reads 3/4 of what two of 2 x 2 read from LDS, and 256 x 256
 * tiles load 2/3 of what 256 x 128 ones do.  Where few values are summed the results' bytes count as much: 1000 x 960 x
 * 100,000 takes 141 us, 1360 TOP/s and 2.1 TB/s.  Few queries are bound by the rows: 24 x 2048 x 50,000 20.3 us, 5.2 TB/s.
 */
template <int WM, int WN, int TM, int TN, int kStep, int kAhead, typename O>
__global__ __launch_bounds__(64 * WM * WN, (160 << 10) / ((kAhead + 1) * (WM * TM + WN * TN) * 32 * kStep) * WM * WN / 4)
void tiled_scores_kernel(product p, tile_order order)  // registers for as many workgroups as LDS has place for
{
  constexpr int kWavesHere = WM * WN, BM = WM * TM * 32, BN = WN * TN * 32;
  constexpr int kChunks    = kStep / 16, kRows = 64 / kChunks;        // of a row; rows that a load of a wavefront covers
  constexpr int kLoads     = (BM + BN) / kRows / kWavesHere;          // a wavefront's loads of a step
  constexpr int kParts     = kStep / 32;                              // of a step, a matrix instruction deep
  constexpr int kBuffer    = (BM + BN) * kStep;
  static_assert((BM + BN) % (kRows * kWavesHere) == 0, "every wavefront loads as much, so that the waits count alike");
  extern __shared__ __align__(1024) char lds[];  // kAhead + 1 buffers: queries, then rows
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const uint2 tile = tile_of(blockIdx.x, order);
  const int64_t i0 = int64_t{tile.x} * BM, j0 = int64_t{tile.y} * BN;
  const int mi = static_cast<int>(min(int64_t{BM}, p.m - i0)), nj = static_cast<int>(min(int64_t{BN}, p.n - j0));
  // rows past the end lie past the buffer's: they load as 0
  const auto qr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.q.x + i0 * p.q.stride), 0,
                                                    static_cast<int>((mi - 1) * p.q.stride + p.k), 0x00020000);
  const auto rr = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(p.r.x + j0 * p.r.stride), 0,
                                                    static_cast<int>((nj - 1) * p.r.stride + p.k), 0x00020000);
  // chunk c of row i lies at c ^ swizzle(i): any 16 rows' chunks c then cover all banks once
  const auto swizzle = [](int i) { return i / (16 / kChunks) % kChunks; };
  const int qrow = (lane / kChunks) * static_cast<int>(p.q.stride), rrow = (lane / kChunks) * static_cast<int>(p.r.stride);
  const auto load = [&](int k0, int buffer, int u) {
    const int g     = wave * kLoads + u;
    const bool q    = g < BM / kRows;
    const int chunk = 16 * ((lane % kChunks) ^ swizzle(g * kRows + lane / kChunks));
    const int base  = (q ? g : g - BM / kRows) * kRows * static_cast<int>(q ? p.q.stride : p.r.stride);
    // k is a multiple of 16; what lies past it loads as 0, and so do steps past the last, that the waits count alike
    __builtin_amdgcn_raw_ptr_buffer_load_lds(q ? qr : rr,
                                             (__attribute__((address_space(3))) void*)(lds + buffer * kBuffer + g * 1024), 16,
                                             k0 + chunk < p.k ? base + (q ? qrow : rrow) + chunk + k0 : 0x7fffff00, 0, 0, 0);
  };
  const int wi = wave / WN * TM * 32, wj = wave % WN * TN * 32;
  i32x16 acc[TM][TN] = {};
  i32x4 a[2][TM], b[2][TN];
  const auto read = [&](int buffer, int part, i32x4(&fa)[TM], i32x4(&fb)[TN]) {
    const char* qa = lds + buffer * kBuffer;
    const int at   = ((2 * part + lane / 32) ^ swizzle(lane % 32)) * 16 + (lane % 32) * kStep;
#pragma unroll
    for (int y = 0; y < TN; ++y)
      fb[y] = *reinterpret_cast<const i32x4*>(qa + (BM + wj + 32 * y) * kStep + at);
#pragma unroll
    for (int x = 0; x < TM; ++x)
      fa[x] = *reinterpret_cast<const i32x4*>(qa + (wi + 32 * x) * kStep + at);
  };
#pragma unroll
  for (int t = 0; t < kAhead; ++t)
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      load(t * kStep, t, u);
  const int steps = (p.k + kStep - 1) / kStep;
  wait_loads<(kAhead - 1) * kLoads>();
  __builtin_amdgcn_s_barrier();
  read(0, 0, a[0], b[0]);
  int buffer = 0;
  for (int t = 0; t < steps; ++t) {
    const int before = buffer == 0 ? kAhead : buffer - 1, after = buffer == kAhead ? 0 : buffer + 1;
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int now = part & 1;
      if (part + 1 < kParts) {
        read(buffer, part + 1, a[1 - now], b[1 - now]);
      } else {
        // the next step's loads have landed in every wavefront, and this step's buffer has been read
        wait_loads<(kAhead - 1) * kLoads, true>();
        __builtin_amdgcn_s_barrier();
        read(after, 0, a[1 - now], b[1 - now]);
      }
      constexpr int kMfma = TM * TN, kReads = TM + TN;
      constexpr int kEach = (kLoads + kParts - 2) / (kParts - 1);  // the last part loads none
      constexpr int kLoadsEach = (kEach + kMfma - 1) / kMfma, kReadsEach = (kReads + kMfma - 1) / kMfma;
#pragma unroll
      for (int x = 0; x < TM; ++x)
#pragma unroll
        for (int y = 0; y < TN; ++y) {
          acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[now][y], a[now][x], acc[x][y], 0, 0, 0);
#pragma unroll
          for (int e = 0; e < kLoadsEach; ++e) {
            const int i = (x * TN + y) * kLoadsEach + e, u = part * kEach + i;
            if (part + 1 < kParts && i < kEach && u < kLoads) load((t + kAhead) * kStep, before, u);
          }
        }
      // a matrix instruction, then the LDS reads and the loads that go beside it
#pragma unroll
      for (int i = 0; i < kMfma; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kReadsEach, 0);
        if (part + 1 < kParts) __builtin_amdgcn_sched_group_barrier(0x020, kLoadsEach, 0);
      }
    }
    buffer = after;
  }
  // a lane holds, of query lane % 32, rows 8 * (e / 4) + 4 * (lane / 32) + e % 4 of each 32 x 32 part: they go through LDS,
  // 32 queries of the wavefront's at a time, so that a row of the output is stored in 16-byte pieces side by side
  constexpr int kThreadsHere = 64 * kWavesHere, kWide = TN * 32, N = kPer16<O>;
  constexpr int kPitch       = kWide * static_cast<int>(sizeof(O)) + 16;
  constexpr int kPieces = kWide / N, kAtOnce = 64 / kPieces;  // of a row; rows that a store of the wavefront covers
  auto* scales = reinterpret_cast<float*>(lds);  // of the tile's rows, then their biases
  auto* biases = scales + BN;
  // results of whole 64-byte pieces pass by the caches: the 200 MB of 1,000 x 960 x 100,000 in float16 then take 138 us in
  // place of 153, where pieces at odd places lose (2048 x 512 x 50,000: 114 us against 102)
  const bool by_cache = (reinterpret_cast<uintptr_t>(p.out) | p.ostride * sizeof(O)) % 64 != 0;
  char* mine          = lds + 2 * BN * sizeof(float) + wave * 32 * kPitch;
  wait_loads<0, true>();  // the steps past the last, which load zeros
  __syncthreads();
  for (int j = threadIdx.x; j < BN; j += kThreadsHere) {
    scales[j] = j < nj ? p.r.scales[j0 + j] : 0.f;
    biases[j] = j < nj && p.bias != nullptr ? p.bias[j0 + j] : -0.f;
  }
  float qs[TM];
#pragma unroll
  for (int x = 0; x < TM; ++x)
    qs[x] = p.q.scales[i0 + min(wi + 32 * x + lane % 32, mi - 1)];
  __syncthreads();
  const auto of_rows = [&](const float* from, int y, int e4) {
    return *reinterpret_cast<const float4*>(from + wj + 32 * y + 8 * e4 + 4 * (lane / 32));
  };
  constexpr bool kHeld = TM > 2;  // where registers are left for them
  float4 rs[TN][4], bs[TN][4];
#pragma unroll
  for (int y = 0; y < TN; ++y)
#pragma unroll
    for (int e4 = 0; kHeld && e4 < 4; ++e4)
      rs[y][e4] = of_rows(scales, y, e4), bs[y][e4] = of_rows(biases, y, e4);
  const int io = wi + lane / kPieces, jo = wj + lane % kPieces * N, left = nj - jo;
  O* to        = static_cast<O*>(p.out) + (i0 + io) * p.ostride + j0 + jo;
#pragma unroll
  for (int x = 0; x < TM; ++x) {
#pragma unroll
    for (int y = 0; y < TN; ++y)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const float4 r = kHeld ? rs[y][e4] : of_rows(scales, y, e4), d = kHeld ? bs[y][e4] : of_rows(biases, y, e4);
        const auto sum = [&](int e) { return static_cast<float>(acc[x][y][4 * e4 + e]) * qs[x]; };
        const O v[4]   = {static_cast<O>(fmaf(sum(0), r.x, d.x)), static_cast<O>(fmaf(sum(1), r.y, d.y)),
                          static_cast<O>(fmaf(sum(2), r.z, d.z)), static_cast<O>(fmaf(sum(3), r.w, d.w))};
        char* at       = mine + (lane % 32) * kPitch + (32 * y + 8 * e4 + 4 * (lane / 32)) * static_cast<int>(sizeof(O));
        __builtin_memcpy(__builtin_assume_aligned(at, 8), v, sizeof(v));
      }
    wave_fence();
#pragma unroll
    for (int u = 0; u < 32 / kAtOnce; ++u) {
      const uint4 raw = *reinterpret_cast<const uint4*>(mine + (u * kAtOnce + lane / kPieces) * kPitch + lane % kPieces * 16);
      if (io + 32 * x + u * kAtOnce >= mi || left <= 0) continue;
      O* at = to + (32 * x + u * kAtOnce) * p.ostride;
      if (left >= N) {
        if (by_cache)
          store16(at, raw);
        else
          store16_nt(at, raw);
      } else {
        O part[N];
        __builtin_memcpy(part, &raw, 16);
#pragma unroll
        for (int q = 0; q < N - 1; ++q)
          if (q < left) at[q] = part[q];
      }
    }
    wave_fence();
  }
}

template <typename F>
void with_float(elem type, F f)
{
  if (type == elem::f32)
    f(float{});
  else if (type == elem::f16)
    f(f16{});
  else
    f(bf16{});
}

}  // namespace

namespace {

/** launch_quantize_rows that also lays out `job` beside its first rows. */
void launch_quantize(const void* x, elem type, int64_t m, int k, int pad, int64_t stride, int8_t* codes, int64_t cstride,
                     float* scales, pack_job const& job, hipStream_t s)
{
  constexpr int64_t kRows = int64_t{1} << 23;  // with a job's, less than 2^32 work-items a grid
  with_float(type, [&](auto e) {
    using T = decltype(e);
    for (int64_t row0 = 0; row0 < m; row0 += kRows) {
      const auto rows     = std::min(kRows, m - row0);
      const pack_job part = row0 == 0 ? job : pack_job{};
      constexpr int N     = kPer16<T>;
      const auto launch   = [&](auto kernel, int lanes) {
        const int64_t blocks = (rows * lanes + kQuantThreads - 1) / kQuantThreads;
        kernel<<<static_cast<unsigned>(blocks + (part.n + kPackRows - 1) / kPackRows), kQuantThreads, 0, s>>>(
          static_cast<const T*>(x), stride, k, pad, codes, cstride, scales, row0, rows, static_cast<unsigned>(blocks), part);
      };
      if (k <= 2 * 16 * N)  // 100,000 x 128 float32: 14.5 us, by 256 threads a row 82
        launch(quantize_kernel<T, 16, 2>, 16);
      else if (k <= 4 * 64 * N)  // 100,000 x 960 float32: 89 us, by 256 threads a row 134
        launch(quantize_kernel<T, 64, 4>, 64);
      else if (k <= 2 * kQuantThreads * N)
        launch(quantize_kernel<T, kQuantThreads, 2>, kQuantThreads);
      else
        launch(quantize_kernel<T, kQuantThreads, 8>, kQuantThreads);
      OCTEX_HIP(hipGetLastError());
    }
  });
}

}  // namespace

void launch_quantize_rows(const void* x, elem type, int64_t m, int k, int64_t stride, int8_t* codes, int64_t cstride,
                          float* scales, hipStream_t s)
{
  launch_quantize(x, type, m, k, k, stride, codes, cstride, scales, {}, s);
}

namespace {

constexpr int64_t kMaxItems = (int64_t{1} << 32) - 1;  // work-items of a grid

template <int WM, int WN, int TM, int TN, int kStep, int kAhead, typename O>
void launch_tiled(product const& p, hipStream_t s)
{
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, kThreadsHere = 64 * WM * WN;
  constexpr int kOut   = 8 * BN + WM * WN * 32 * (TN * 32 * static_cast<int>(sizeof(O)) + 16);
  constexpr size_t lds = std::max((kAhead + 1) * (BM + BN) * kStep, kOut);
  const auto kernel    = tiled_scores_kernel<WM, WN, TM, TN, kStep, kAhead, O>;
  allow_lds(reinterpret_cast<const void*>(kernel), lds);
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  OCTEX_EXPECTS(tm * tn <= kMaxItems / kThreadsHere, "octex: too many scores at once");
  const tile_order o{static_cast<unsigned>(tm), static_cast<unsigned>(tn)};
  kernel<<<o.tm * o.tn, kThreadsHere, lds, s>>>(p, o);
  OCTEX_HIP(hipGetLastError());
}

template <typename Q, bool kFused, typename O>
void launch_few(product const& p, const Q* floats, int64_t fstride, hipStream_t s)
{
  const int chunks = (p.k + 15) / 16, pitch = 16 * (chunks | 1);  // an odd number of chunks: rows on other banks
  const auto launch = [&](auto rt, auto kw) {
    constexpr int RT = decltype(rt)::value, KW = decltype(kw)::value;
    const auto kernel = few_scores_kernel<RT, KW, kFused, Q, O>;
    const size_t lds  = std::max<size_t>(KW * RT * 1024, kFused ? p.m * pitch : 0);
    allow_lds(reinterpret_cast<const void*>(kernel), lds);
    const int64_t blocks = (p.n + RT * 16 - 1) / (RT * 16);
    OCTEX_EXPECTS(blocks * 64 * KW <= kMaxItems, "octex: too many rows to score at once");
    kernel<<<static_cast<unsigned>(blocks), 64 * KW, lds, s>>>(p, floats, fstride, pitch);
    OCTEX_HIP(hipGetLastError());
  };
  if (p.n >= 8192)
    launch(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
  else
    launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
}

/**
 * The tilings, and what each takes: `a` us a column and c us for one tile by itself; with all of its slots (workgroups on the
 * GPU at a time) busy, `rate` operations a us and e us to store a round's results.  Larger tiles load each operand fewer
 * times and smaller ones fill the GPU with less, so a product takes the tiling whose estimate is least.  The numbers were
 * fitted to the times of 21 products whose rows come from memory; of these six they now choose the best tiling for all but the
 * second, which takes 256 x 128 (us, of 256 x 256, 256 x 128, 128 x 128 and 64 x 64):
 *   1000 x 960 x 100,000: 141, 166, 212, 282;  512 x 512 x 200,000: 95, 103, 126, 191;  4096 x 4096 x 4096: 62, 76, 84, 110;
 *   2048 x 2048 x 2048: 24, 19, 14, 19;  333 x 1008 x 5003: 18, 13, 10, 8.8;  128 x 4096 x 8192: 39, 27, 20, 12.7.
 * No bytes are in the estimate, so it is blind among tilings of a product that is bound by its rows.  256 x 256 tiles have two
 * steps of 64 on their way: with one of 128 the first of these products took 8 % longer, 8192 x 4096 x 16,384 3 % (but 4096 x
 * 4096 x 4096 4 % less); with three of 64 all three took 1 % longer.
 */
struct tiling {
  int bm, bn, slots;
  double c, a, rate, e;
};
constexpr tiling kTilings[] = {{256, 256, 256, 8.0, 0.0100, 2.24e9, 10.5},
                               {256, 128, 512, 5.8, 0.0068, 1.48e9, 5.4},
                               {128, 128, 512, 6.2, 0.0044, 1.50e9, 5.7},
                               {64, 64, 768, 4.5, 0.0023, 1.07e9, 2.6}};

/** Queries that take tiles of 32 x 128, which hold fewer zeros: 24 x 2048 x 50,000 20.3 us, by 64 x 64 26.9 (but 32 x 4096 x
 * 100,000 89 against 87). */
constexpr int64_t kThinQueries = 32;

auto estimate(tiling const& t, product const& p) -> double
{
  const double tiles  = static_cast<double>((p.m + t.bm - 1) / t.bm) * static_cast<double>((p.n + t.bn - 1) / t.bn);
  const double rounds = std::ceil(tiles / t.slots), left = tiles - (rounds - 1) * t.slots;
  const double tile   = 2.0 * t.bm * t.bn * p.k / t.rate;
  return t.c + (rounds - 1) * (t.slots * tile + t.e) + std::max(t.a * p.k, left * tile);
}

template <typename O>
void launch_best(product const& p, hipStream_t s)
{
  if (p.m <= kThinQueries) return launch_tiled<1, 4, 1, 1, 128, 2, O>(p, s);
  int best = 0;
  for (int i = 1; i < 4; ++i)
    if (estimate(kTilings[i], p) < estimate(kTilings[best], p)) best = i;
  if (best == 0)
    launch_tiled<2, 4, 4, 2, 64, 2, O>(p, s);
  else if (best == 1)
    launch_tiled<4, 2, 2, 2, 64, 2, O>(p, s);
  else if (best == 2)
    launch_tiled<2, 2, 2, 2, 64, 3, O>(p, s);
  else
    launch_tiled<2, 2, 1, 1, 128, 2, O>(p, s);
}

/** Whether whole 16-byte chunks reach all of an operand, a tile's rows within 32-bit offsets. */
auto chunked(int8_rows const& r, int k) -> bool
{
  return k % 16 == 0 && r.stride % 16 == 0 && reinterpret_cast<uintptr_t>(r.x) % 16 == 0 && r.stride <= kMaxInt8Stride;
}

void launch_pack(pack_job const& job, hipStream_t s)
{
  constexpr int64_t kRows = kMaxItems / (64 * kPackRows) * kPackRows;
  for (int64_t first = 0; first < job.n; first += kRows) {
    const int64_t rows = std::min(kRows, job.n - first);
    pack_kernel<<<static_cast<unsigned>((rows + kPackRows - 1) / kPackRows), 64 * kPackRows, 0, s>>>(job, first);
    OCTEX_HIP(hipGetLastError());
  }
}

constexpr int kFewQueries      = 16;                  // a matrix instruction's
constexpr int64_t kFewRows     = 8192;                // tiles leave half of the GPU idle (1 x 4096 x 5000: 12.8 us, not 7.9)
constexpr int kFewFused        = 8192;                // values up to which each workgroup quantizes all queries itself
constexpr int64_t kPackedBytes = int64_t{128} << 20;  // of rows laid out anew at a time: they stay in the last-level cache

/** How a product is made, and where its workspace lies. */
struct scores_plan {
  bool few;                          // by few_scores_kernel, from operands as they are (floats: quantized on the way)
  bool pack_q, pack_r;               // operands laid out anew
  int64_t pitch, part;               // of such rows; how many of them at a time
  int64_t codes, scales, rows, end;  // offsets: the queries' codes and scales, the rows
};

auto plan_of(int8_query const& q, int64_t m, int8_rows const& r, int64_t n, int k) -> scores_plan
{
  constexpr int64_t kAlign = 256;
  const auto up            = [](int64_t v) { return (v + kAlign - 1) / kAlign * kAlign; };
  const bool floats = q.type != elem::i8, fused = floats && m <= kFewQueries && m * k <= kFewFused;
  scores_plan p{};
  // quantized queries end with zeros, so that their rows' chunks may be whole
  const bool q_fits = floats || chunked({static_cast<const int8_t*>(q.x), q.stride, nullptr}, k), r_fits = chunked(r, k);
  p.few    = fused || (m <= kFewQueries && (!r_fits || !q_fits || n < kFewRows));
  p.pitch  = int8_pitch(k);
  p.pack_q = !floats && !p.few && !(q_fits && r_fits);
  p.pack_r = !p.few && !r_fits;
  p.part   = p.pack_r ? std::min(n, std::max<int64_t>(kPackedBytes / p.pitch, 1)) : n;
  if ((floats && !fused) || p.pack_q) p.scales = up(m * p.pitch);
  if (floats && !fused) p.rows = p.scales + up(m * 4);
  if (p.pack_q) p.rows = p.scales;
  p.end = p.rows + (p.pack_r ? up(p.part * p.pitch) : 0);
  return p;
}

}  // namespace

auto int8_scores_workspace(int8_query const& q, int64_t m, int8_rows const& r, int64_t n, int k) -> int64_t
{
  return plan_of(q, m, r, n, k).end;
}

void launch_int8_scores(int8_query const& q, int64_t m, int8_rows const& r, int64_t n, int k, const float* bias, void* out,
                        elem type, int64_t ostride, void* workspace, hipStream_t s)
{
  const auto plan   = plan_of(q, m, r, n, k);
  auto* w           = static_cast<int8_t*>(workspace);
  const bool floats = q.type != elem::i8;
  product p{{static_cast<const int8_t*>(q.x), q.stride, q.scales}, r, m, n, k, bias, out, ostride};
  with_float(type, [&](auto e) {
    using O = decltype(e);
    if (floats && plan.end == 0) {
      with_float(q.type, [&](auto f) {
        using Q = decltype(f);
        launch_few<Q, true, O>(p, static_cast<const Q*>(q.x), q.stride, s);
      });
      return;
    }
    const int chunks = (k + 15) / 16 * 16;
    const auto pack  = [&](int64_t j0) {  // of the part of the rows that begins at j0
      return plan.pack_r ? pack_job{r.x + j0 * r.stride, r.stride, std::min(plan.part, n - j0), k, w + plan.rows, plan.pitch}
                         : pack_job{};
    };
    if (floats) {
      auto* scales = reinterpret_cast<float*>(w + plan.scales);
      launch_quantize(q.x, q.type, m, k, chunks, q.stride, w, plan.pitch, scales, pack(0), s);
      p.q = {w, plan.pitch, scales};
    } else if (plan.pack_q) {
      launch_pack({p.q.x, p.q.stride, m, k, w, plan.pitch}, s);
      p.q = {w, plan.pitch, q.scales};
    }
    if (plan.few) {
      launch_few<float, false, O>(p, nullptr, 0, s);
      return;
    }
    p.k = chunks;
    for (int64_t j0 = 0; j0 < n; j0 += plan.part) {
      p.n = std::min(plan.part, n - j0);
      p.r = {r.x + j0 * r.stride, r.stride, r.scales + j0};
      if (plan.pack_r) {
        if (j0 > 0 || !floats) launch_pack(pack(j0), s);
        p.r.x = w + plan.rows, p.r.stride = plan.pitch;
      }
      p.bias = bias != nullptr ? bias + j0 : nullptr;
      p.out  = static_cast<O*>(out) + j0;
      launch_best<O>(p, s);
    }
  });
}

}  // namespace cuvs::neighbors::octex::detail
