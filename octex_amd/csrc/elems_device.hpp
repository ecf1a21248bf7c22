// Element access of the operators' kernels: 16 bytes of a row at a time as floats, and back with one rounding.
#pragma once

#include "rows.hpp"

#include <hip/hip_runtime.h>

#include <cmath>

namespace cuvs::neighbors::octex::detail {

using bf16 = __bf16;
using f16  = _Float16;

__device__ inline void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

/** A barrier for what lies in LDS: the workgroup's loads and stores of other memory stay on their way. */
__device__ inline void lds_barrier()
{
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

/** Elements of 16 bytes. */
template <typename T>
constexpr int kPer16 = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ inline void unpack16(uint4 raw, float (&v)[kPer16<T>])
{
  const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __uint_as_float(w[i]);
  } else if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i]     = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i]     = static_cast<float>(__builtin_bit_cast(f16, static_cast<unsigned short>(w[i])));
      v[2 * i + 1] = static_cast<float>(__builtin_bit_cast(f16, static_cast<unsigned short>(w[i] >> 16)));
    }
  }
}

template <typename T>
__device__ inline auto pack16(const float (&v)[kPer16<T>]) -> uint4
{
  T e[kPer16<T>];
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i)
    e[i] = static_cast<T>(v[i]);
  uint4 raw;
  __builtin_memcpy(&raw, e, 16);
  return raw;
}

/** 16 bytes at any alignment of their elements: the hardware takes an unaligned 16-byte load. */
template <typename T>
__device__ inline auto load16(const T* p) -> uint4
{
  uint4 raw;
  __builtin_memcpy(&raw, p, 16);
  return raw;
}

template <typename T>
__device__ inline void store16(T* p, uint4 raw)
{
  __builtin_memcpy(p, &raw, 16);
}

/** The same for results that no kernel reads soon: they pass by the caches. */
template <typename T>
__device__ inline void store16_nt(T* p, uint4 raw)
{
  using words = unsigned __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  __builtin_nontemporal_store(words{raw.x, raw.y, raw.z, raw.w}, reinterpret_cast<words*>(p));
}

/** Elements [at, at + kPer16) of a row as they lie in memory, those from `end` on 0. */
template <typename T>
__device__ inline auto load_row16(const T* row, int at, int end) -> uint4
{
  if (at + kPer16<T> <= end) return load16(row + at);
  T e[kPer16<T>];
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i)
    e[i] = at + i < end ? row[at + i] : static_cast<T>(0.f);
  uint4 raw;
  __builtin_memcpy(&raw, e, 16);
  return raw;
}

/** One element of a small array whose type is known at run time. */
__device__ inline auto load_any(const void* p, elem type, int64_t i) -> float
{
  if (type == elem::f32) return static_cast<const float*>(p)[i];
  if (type == elem::f16) return static_cast<float>(static_cast<const f16*>(p)[i]);
  return static_cast<float>(static_cast<const bf16*>(p)[i]);
}

}  // namespace cuvs::neighbors::octex::detail
