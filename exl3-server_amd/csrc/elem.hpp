// Element types of the token mixer's and the sampler's operands (f16, bf16, f32): loads and
// stores of single values and of 8 adjacent ones, always computed on in f32.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "exl3_device.hpp"
#include "exl3_moe.h"

typedef __bf16 bf16;

namespace exl3e {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// One value as f32 (exact) and back (one rounding to nearest even).
template <typename E>
__device__ __forceinline__ float to_f32(E v) {
  return (float)v;
}
template <typename E>
__device__ __forceinline__ E from_f32(float v) {
  return (E)v;
}

// Eight adjacent 16-bit values: one 16-byte load or store.
template <typename E>
__device__ __forceinline__ void load8(const E *p, float (&v)[8]) {
  typedef E vec __attribute__((ext_vector_type(8)));
  const vec x = *reinterpret_cast<const vec *>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
}
template <bool kPast = false, typename E>
__device__ __forceinline__ void store8(E *p, const float (&v)[8]) {
  typedef E vec __attribute__((ext_vector_type(8)));
  vec x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (E)v[i];
  if constexpr (kPast) __builtin_nontemporal_store(x, reinterpret_cast<vec *>(p));  // past the caches
  else *reinterpret_cast<vec *>(p) = x;
}

// Whether the bytes [p, p + n) and [q, q + m) meet.
inline bool spans_meet(uintptr_t p, size_t n, uintptr_t q, size_t m) { return n && m && p < q + m && q < p + n; }
inline bool spans_meet(const void *p, size_t n, const void *q, size_t m) {
  return spans_meet(reinterpret_cast<uintptr_t>(p), n, reinterpret_cast<uintptr_t>(q), m);
}

// f(E{}) for a 16-bit element type (EXL3_ST_F16 or EXL3_ST_BF16).
template <typename F>
void with_elem16(int32_t dtype, F &&f) {
  if (dtype == EXL3_ST_BF16) f(bf16{});
  else f(f16{});
}

}  // namespace exl3e
