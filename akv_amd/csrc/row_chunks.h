// Rows as lanes hold them: chunks of eight elements, of any storage type, and
// single elements (gfx950).
#pragma once

#include "common.h"

namespace akv {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) u32x4 global_u32x4;

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }

// Eight consecutive elements as stored: one or two 16-byte words.
template <typename T>
struct Chunk {
  static constexpr int kWords = sizeof(T) / 2;
  u32x4 w[kWords];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = *((const global_u32x4*)p + i);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) *((global_u32x4*)p + i) = w[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    typedef T T8 __attribute__((ext_vector_type(8)));
    const T8 v = __builtin_bit_cast(T8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[i]);
    __builtin_memcpy(w, &v, sizeof(w));
  }
};

// Eight values of a vector of any storage type (uniform branch).
__device__ __forceinline__ void load8(const void* p, int32_t dtype, int64_t at, float (&x)[8]) {
  if (dtype == AKV_F32) {
    Chunk<float> c;
    c.load(static_cast<const float*>(p) + at);
    c.get(x);
  } else if (dtype == AKV_F16) {
    Chunk<_Float16> c;
    c.load(static_cast<const _Float16*>(p) + at);
    c.get(x);
  } else {
    Chunk<__bf16> c;
    c.load(static_cast<const __bf16*>(p) + at);
    c.get(x);
  }
}

__device__ __forceinline__ float load1(const void* p, int32_t dtype, int64_t at) {
  if (dtype == AKV_F32) return static_cast<const float*>(p)[at];
  if (dtype == AKV_F16) return to_f32(static_cast<const _Float16*>(p)[at]);
  return to_f32(static_cast<const __bf16*>(p)[at]);
}

}  // namespace
}  // namespace akv
