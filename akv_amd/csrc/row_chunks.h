// Rows as lanes hold them: chunks of eight elements, of any storage type, and
// single elements (gfx950).
#pragma once

#include "common.h"

namespace akv {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) u32x4 global_u32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) u32x2 global_u32x2;

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
  // Two quads, the second `mid` elements behind the first.
  __device__ __forceinline__ void load_quads(const T* p, int mid) {
    if constexpr (kWords == 1) {
      const u32x2 a = *(const global_u32x2*)p, b = *(const global_u32x2*)(p + mid);
      w[0] = u32x4{a[0], a[1], b[0], b[1]};
    } else {
      w[0] = *(const global_u32x4*)p;
      w[1] = *(const global_u32x4*)(p + mid);
    }
  }
  __device__ __forceinline__ void store_quads(T* p, int mid) const {
    if constexpr (kWords == 1) {
      *(global_u32x2*)p = u32x2{w[0][0], w[0][1]};
      *(global_u32x2*)(p + mid) = u32x2{w[0][2], w[0][3]};
    } else {
      *(global_u32x4*)p = w[0];
      *(global_u32x4*)(p + mid) = w[1];
    }
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

// Eight values of a vector of any storage type (uniform branch); of two quads, the second
// `mid` elements behind the first, where that is not 4.
template <bool QUADS = false>
__device__ __forceinline__ void load8(const void* p, int32_t dtype, int64_t at, float (&x)[8], int mid = 4) {
  auto take = [&](auto c, auto* from) __attribute__((always_inline)) {
    if constexpr (QUADS)
      c.load_quads(from + at, mid);
    else
      c.load(from + at);
    c.get(x);
  };
  if (dtype == AKV_F32) {
    take(Chunk<float>(), static_cast<const float*>(p));
  } else if (dtype == AKV_F16) {
    take(Chunk<_Float16>(), static_cast<const _Float16*>(p));
  } else {
    take(Chunk<__bf16>(), static_cast<const __bf16*>(p));
  }
}

__device__ __forceinline__ float load1(const void* p, int32_t dtype, int64_t at) {
  if (dtype == AKV_F32) return static_cast<const float*>(p)[at];
  if (dtype == AKV_F16) return to_f32(static_cast<const _Float16*>(p)[at]);
  return to_f32(static_cast<const __bf16*>(p)[at]);
}

}  // namespace
}  // namespace akv
