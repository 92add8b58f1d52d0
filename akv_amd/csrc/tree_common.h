// What the attentions of new tokens over a cache share (tree_attention.hip,
// kv8_attention.hip): their arguments, a lane's operations, and the second launch
// that merges the pieces of rows whose keys were cut (gfx950).
#pragma once

#include <algorithm>
#include <cmath>

#include "common.h"

extern "C" __device__ long long __ockl_wfred_add_i64(long long);
extern "C" __device__ int __ockl_wfred_max_i32(int);
extern "C" __device__ int __ockl_wfred_min_i32(int);
extern "C" __device__ long long __ockl_wfscan_add_i64(long long, bool);

namespace akv {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) u32x4 global_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kLog2e = 1.4426950408889634f;
// A weight sum above 2^32 takes exact maxima (the keys alone add up to 2^30).  Values
// up to 2^94 stay finite in a wave's products; waves and pieces are joined by shares
// of their sums, which stay between the values.
constexpr float kHuge = 4294967296.f;

// Workgroups of a launch that shares the keys out: two per CU.
constexpr int kGroupsShift = 9, kGroups = 1 << kGroupsShift;
constexpr int64_t kMostKeys = 1 << 30;  // of a request: ranks and tiles stay far inside 32 bits

constexpr int kWordsKept = 2;  // mask words of a row in LDS: trees of up to 128 tokens

struct TreeArgs {
  const void* q;
  int64_t q_st, q_sh;
  const char* k;
  const char* v;
  int64_t k_ss, k_sh, v_ss, v_sh;  // bytes
  int64_t pool_slots;
  const void* qo_indptr;
  const void* kv_indptr;
  const int32_t* kv_indices;
  int64_t table_stride, table_width;  // a block table's row stride and pages; a flat list: stride 0, its length
  const uint64_t* mask;
  int64_t mask_stride;
  const int32_t* key_starts;
  const float* sinks;
  const int32_t* gate;
  float scale_log2;
  void* out;
  int64_t o_st, o_sh;
  float* part_o;   // [2 kGroups][rows of a block][D], each divided by its piece's sum
  float* part_ml;  // [2 kGroups][rows of a block][2]
  int32_t* owner;  // [tokens][q heads][4]: the workgroups with the row's first (-1: all) and last keys, its row
  int64_t n_tokens, max_len;
  int32_t n_requests, q_heads, kv_heads, group, head_dim, mask_words, page_size;
  int32_t row_blocks;  // whole launch: workgroups that share a request's rows
  bool indptr64, out_f32, out_vectors, paged, whole;
};

static __device__ __attribute__((aligned(16))) const uint32_t zero_row[64] = {};

__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = uniform(static_cast<uint32_t>(v)), hi = uniform(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

template <typename T>
struct Vec {
  typedef T x4 __attribute__((ext_vector_type(4)));
  typedef T x8 __attribute__((ext_vector_type(8)));
};

__device__ __forceinline__ f32x4 product(Vec<__bf16>::x8 a, Vec<__bf16>::x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product(Vec<_Float16>::x8 a, Vec<_Float16>::x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Whether the 16 bits are an infinity or NaN of type T.
template <typename T>
__device__ __forceinline__ bool not_finite(short bits) {
  constexpr short e = __is_same(T, __bf16) ? 0x7f80 : 0x7c00;
  return (bits & e) == e;
}

// Four dims of an output row.
template <typename T>
__device__ __forceinline__ void store_four(const TreeArgs& a, int64_t at, f32x4 x) {
  if (a.out_f32) {
    float* to = static_cast<float*>(a.out) + at;
    if (a.out_vectors) {
      *reinterpret_cast<f32x4*>(to) = x;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = x[i];
  } else {
    T* to = static_cast<T*>(a.out) + at;
    const typename Vec<T>::x4 y = __builtin_convertvector(x, typename Vec<T>::x4);
    if (a.out_vectors) {
      *reinterpret_cast<typename Vec<T>::x4*>(to) = y;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = y[i];
  }
}

// 1 / l; a weight sum of 0 (nothing was seen) gives rows of 0.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// v_max3_f32 / v_max_f32 without the canonicalising moves around fmaxf of
// matrix-core results; a NaN score still reaches the output through exp2.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// Maximum over the lanes col, col + 16, col + 32, col + 48 of a column.
__device__ __forceinline__ float column_max(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto r16 = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  const uint32_t a0 = r16[0], a1 = r16[1];
  x = max2(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  const uint32_t c = __builtin_bit_cast(uint32_t, x);
  const auto r32 = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  const uint32_t c0 = r32[0], c1 = r32[1];
  return max2(__builtin_bit_cast(float, c0), __builtin_bit_cast(float, c1));
}

// The same value, of which the compiler knows nothing: what is derived from it
// is not computed ahead of the loops before it, and holds no register there.
__device__ __forceinline__ int32_t here_only(int32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Loads straight into LDS: lane l's bytes go to `to` + 16 l (4 l).  In asm, since
// the compiler takes every later LDS read for one that may meet them and waits
// for all of them; arrive() does the waiting.
__device__ __forceinline__ void load_16(const void* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to)
               : "memory", "m0");
}
__device__ __forceinline__ void load_4(const void* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(to)
               : "memory", "m0");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

// Waits for this wave's loads and LDS accesses, then for the other waves.
__device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Merges the pieces of rows that a cut went through, and the sink: WAYS x D / 4
// lanes per (token, head), each way every WAYS-th piece, AHEAD of them in flight.
template <typename T, int D, int WAYS, int AHEAD>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeArgs a, const int block_rows, const int64_t row0) {
  constexpr int kLanes = D / 4;
  const int64_t row = row0 + static_cast<int64_t>(blockIdx.x) * (256 / (kLanes * WAYS)) + threadIdx.x / (kLanes * WAYS);
  const int d = 4 * (threadIdx.x % kLanes), way = threadIdx.x / kLanes % WAYS;
  const int64_t token = row / a.q_heads;
  const int head = static_cast<int>(row - token * a.q_heads);
  if (token >= a.n_tokens) return;
  // one round of loads: whether the row is a token's, and who has its pieces
  const int64_t begin = load_index(a.qo_indptr, a.indptr64, 0), end = load_index(a.qo_indptr, a.indptr64, a.n_requests);
  const int32_t* owner = a.owner + 4 * row;
  const int first = owner[0], last = owner[1], r = owner[2];
  const float sink = a.sinks ? a.sinks[head] * kLog2e : -INFINITY;
  if (gated(a.gate) || token < begin || token >= end) return;
  // (indptrs that descend leave rows without owners)
  if (first < 0 || last < first || last >= kGroups || r < 0 || r >= block_rows) return;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};  // of the pieces so far, divided by l
  for (int w = first + way; w <= last; w += AHEAD * WAYS) {
    f32x2 ml[AHEAD];
    f32x4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int at = w + i * WAYS <= last ? w + i * WAYS : last;
      const int64_t place = (2ll * at + (at == first ? 1 : 0)) * block_rows + r;
      ml[i] = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * place);
      x[i] = *reinterpret_cast<const f32x4*>(a.part_o + place * D + d);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
    const float base = top == -INFINITY ? 0.f : top;
    // a piece without a key carries m = -inf, l = 0 and O = 0
    const float kept = l * __builtin_amdgcn_exp2f(m - base);
    l = kept;
    m = top;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      ml[i].y = w + i * WAYS <= last ? ml[i].y * __builtin_amdgcn_exp2f(ml[i].x - base) : 0.f;
      l += ml[i].y;
    }
    const float inv = inverse(l);
    o *= kept * inv;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (w + i * WAYS <= last) o += x[i] * (ml[i].y * inv);
  }
  float top = fmaxf(m, sink);
#pragma unroll
  for (int off = kLanes; off < kLanes * WAYS; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float base = top == -INFINITY ? 0.f : top;
  const float mine = l * __builtin_amdgcn_exp2f(m - base);
  l = mine;
#pragma unroll
  for (int off = kLanes; off < kLanes * WAYS; off <<= 1) l += __shfl_xor(l, off);
  if (a.sinks) l += __builtin_amdgcn_exp2f(sink - base);
  o *= mine * inverse(l);
#pragma unroll
  for (int off = kLanes; off < kLanes * WAYS; off <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], off);
  }
  if (way == 0 && d < a.head_dim) store_four<T>(a, token * a.o_st + head * a.o_sh + d, o);
}

// Workgroups of 256 threads in a launch: a grid has fewer than 2^32 threads, and
// what is beyond is left out without an error.
constexpr int64_t kMostBlocks = 1 << 23;

// Rows of a KV head that a request may have.
int64_t most_rows(int64_t n_tokens, int64_t q_heads, int64_t kv_heads, int64_t max_new) {
  return std::max<int64_t>(1, std::min(max_new, n_tokens)) * (q_heads / kv_heads);
}

int64_t owner_bytes(int64_t n_tokens, int64_t q_heads) { return 16 * n_tokens * q_heads; }

int64_t cut_bytes(int d, int sub, int64_t n_tokens, int64_t q_heads) {
  return owner_bytes(n_tokens, q_heads) + 2ll * kGroups * (16 * kWaves * sub) * (d + 2) * 4;
}

// Few rows are cut into many pieces each, and many rows fill the chip: a wave per
// row up to kFewRows, D / 4 lanes beyond (both launches, us by the wave and by the
// lanes: 512 rows of one request of 8192 keys 22.6, 31.5; 4096 rows 42.8, 44.8; 16384
// rows of 16 requests of 4096 49.7, 46.8).  Up to kFewestRows all of a row's pieces
// are on their way at once, 16 per way, 4 beyond (128 rows of 128 dims over 4096 keys
// 16.8, 18.3; 512 rows over 8192 21.1, 22.1; 4096 rows 44.2, 41.2).
constexpr int64_t kFewRows = 4096, kFewestRows = 512;

template <typename T, int D, int WAYS, int AHEAD>
void merge_by(const TreeArgs& a, int block_rows, hipStream_t st) {
  constexpr int kRows = 256 / (D / 4 * WAYS);
  const int64_t rows = a.n_tokens * a.q_heads;
  for (int64_t row0 = 0; row0 < rows; row0 += kMostBlocks * kRows) {
    const dim3 grid(static_cast<unsigned>(std::min(kMostBlocks, (rows - row0 + kRows - 1) / kRows)));
    hipLaunchKernelGGL((tree_combine_kernel<T, D, WAYS, AHEAD>), grid, dim3(256), 0, st, a, block_rows, row0);
  }
}

template <typename T, int D>
void merge(const TreeArgs& a, int block_rows, hipStream_t st) {
  constexpr int kWays = 64 / (D / 4);
  const int64_t rows = a.n_tokens * a.q_heads;
  if (rows <= kFewestRows)
    merge_by<T, D, kWays, 16>(a, block_rows, st);
  else if (rows <= kFewRows)
    merge_by<T, D, kWays, 4>(a, block_rows, st);
  else
    merge_by<T, D, 1, 4>(a, block_rows, st);
}

}  // namespace
}  // namespace akv
