// Scores in 8-bit integers: out[i][j] = qs[i] rs[j] sum_d q[i][d] r[j][d] + bias[j], the sums exact in int32.

#include "common.hpp"
#include "elems_device.hpp"
#include "scores.hpp"

#include <algorithm>

namespace cuvs::neighbors::octex::detail {

namespace {

using i32x4  = int __attribute__((ext_vector_type(4)));
using i32x16 = int __attribute__((ext_vector_type(16)));

// ---- quantization of rows

constexpr int kQuantThreads = 256;

__device__ inline auto code_of(float v, float scale) -> int
{
  return static_cast<int>(fminf(fmaxf(rintf(v / scale), -127.f), 127.f));
}

/** scale = max |x| / 127; code = the whole number nearest to x / scale (ties to even), the quotient rounded to fp32 first.
 * A row of zeros has scale 0 and codes 0; one with a NaN or an infinity has scale NaN and codes 0. */
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(const T* x, int64_t stride, int k, int8_t* codes,
                                                                 int64_t cstride, float* scales, int64_t row0)
{
  __shared__ unsigned tops[kQuantThreads / 64];
  const int64_t r = row0 + blockIdx.x;
  const T* row    = x + r * stride;
  // a magnitude's bits order as it does, with infinity and NaN above every finite one
  unsigned top = 0;
  for (int i = threadIdx.x; i < k; i += kQuantThreads)
    top = max(top, __float_as_uint(static_cast<float>(row[i])) & 0x7fffffffu);
#pragma unroll
  for (int mask = 32; mask > 0; mask >>= 1)
    top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), mask)));
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
  for (int w = 0; w < kQuantThreads / 64; ++w)
    top = max(top, tops[w]);
  const bool finite = top < 0x7f800000u;
  const float scale = finite ? __uint_as_float(top) / 127.f : NAN;
  if (threadIdx.x == 0) scales[r] = scale;
  for (int i = threadIdx.x; i < k; i += kQuantThreads)
    codes[r * cstride + i] = scale > 0.f ? static_cast<int8_t>(code_of(static_cast<float>(row[i]), scale)) : 0;
}

// ---- the product: tiles of 64 x 64, 128 bytes of both operands in LDS at a time

constexpr int kBK = 128;  // bytes of a row in LDS

struct product {
  int8_rows q, r;
  int64_t m, n;
  int k;
  const float* bias;
  void* out;
  int64_t ostride;
};

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

template <typename O>
__global__ __launch_bounds__(256) void scores_kernel(product p, unsigned tiles_n)
{
  // a row's eight 16-byte chunks, chunk c of row i at c ^ (i % 8): a fragment's 32 rows then fall on different banks
  __shared__ i32x4 qa[64 * 8], ra[64 * 8];
  const int64_t i0 = int64_t{blockIdx.x / tiles_n} * 64, j0 = int64_t{blockIdx.x % tiles_n} * 64;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int wi = wave / 2 * 32, wj = wave % 2 * 32;
  i32x16 acc = {};
  for (int k0 = 0; k0 < p.k; k0 += kBK) {
    i32x4 a[2], b[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = threadIdx.x + 256 * u, i = e / 8, c = e % 8;
      a[u] = i0 + i < p.m ? load_codes(p.q.x + (i0 + i) * p.q.stride, k0 + 16 * c, p.k) : i32x4{0, 0, 0, 0};
      b[u] = j0 + i < p.n ? load_codes(p.r.x + (j0 + i) * p.r.stride, k0 + 16 * c, p.k) : i32x4{0, 0, 0, 0};
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = threadIdx.x + 256 * u, i = e / 8, c = e % 8;
      qa[i * 8 + (c ^ (i & 7))] = a[u];
      ra[i * 8 + (c ^ (i & 7))] = b[u];
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const int c = 2 * kk + lane / 32, i = lane % 32;
      const i32x4 fa = qa[(wi + i) * 8 + (c ^ (i & 7))], fb = ra[(wj + i) * 8 + (c ^ (i & 7))];
      acc            = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa, fb, acc, 0, 0, 0);
    }
  }
  const int64_t j = j0 + wj + lane % 32;
  if (j >= p.n) return;
  const float rs = p.r.scales[j], b = p.bias != nullptr ? p.bias[j] : 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int64_t i = i0 + wi + 8 * (e / 4) + 4 * (lane / 32) + e % 4;
    if (i >= p.m) continue;
    float v = static_cast<float>(acc[e]) * p.q.scales[i] * rs;
    if (p.bias != nullptr) v += b;
    static_cast<O*>(p.out)[i * p.ostride + j] = static_cast<O>(v);
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

void launch_quantize_rows(const void* x, elem type, int64_t m, int k, int64_t stride, int8_t* codes, int64_t cstride,
                          float* scales, hipStream_t s)
{
  constexpr int64_t kRows = (int64_t{1} << 32) / kQuantThreads - 1;  // less than 2^32 work-items a grid
  with_float(type, [&](auto e) {
    using T = decltype(e);
    for (int64_t row0 = 0; row0 < m; row0 += kRows) {
      quantize_kernel<T><<<static_cast<unsigned>(std::min(kRows, m - row0)), kQuantThreads, 0, s>>>(
        static_cast<const T*>(x), stride, k, codes, cstride, scales, row0);
      OCTEX_HIP(hipGetLastError());
    }
  });
}

void launch_int8_scores(int8_rows const& q, int64_t m, int8_rows const& r, int64_t n, int k, const float* bias, void* out,
                        elem type, int64_t ostride, hipStream_t s)
{
  constexpr int64_t kTiles = (int64_t{1} << 32) / 256 - 1;  // less than 2^32 work-items a grid
  const int64_t tiles_n    = (n + 63) / 64;
  OCTEX_EXPECTS(tiles_n <= kTiles, "octex: too many rows to score at once");
  const int64_t step = kTiles / tiles_n * 64;  // queries of a grid
  with_float(type, [&](auto e) {
    using O = decltype(e);
    for (int64_t i0 = 0; i0 < m; i0 += step) {
      product p{q, r, std::min(step, m - i0), n, k, bias, static_cast<O*>(out) + i0 * ostride, ostride};
      p.q.x += i0 * q.stride;
      p.q.scales += i0;
      const int64_t tiles = (p.m + 63) / 64 * tiles_n;
      scores_kernel<O><<<static_cast<unsigned>(tiles), 256, 0, s>>>(p, static_cast<unsigned>(tiles_n));
      OCTEX_HIP(hipGetLastError());
    }
  });
}

}  // namespace cuvs::neighbors::octex::detail
