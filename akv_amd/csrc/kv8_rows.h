// Rows into a cache held in 8 bits, with a scale for each block of slots and
// head: what the calls that write them share (kv8_append.hip, kv8_move.hip; gfx950).
//
// A value is code * scale, the code an 8-bit float (e4m3: largest F = 448; e5m2:
// F = 57344), the scale that of the slot's block (slots s with the same s / B) and
// head.  The rows that a call brings to a block, A their largest finite magnitude:
//   from the block's first slot on   s = the smallest power of two >= 2^-100 with A <= F s
//   behind rows it holds             s = s0 2^k, s0 its scale, k >= 0 the least with A <= F s;
//                                    for k > 0 those rows become round(code s0 / s)
// and each value y the code round(y / s), to nearest, ties to even.  Powers of two:
// codes are floats, so a finer scale would not make them more exact, and a scale
// that grows leaves the codes' digits as they are (but for those that fall below the
// smallest normal one); y / s is y (1 / s) with no further rounding.  F = 1.75 2^n in both
// types, so s is read off the bits of A.
//
// A wave takes the rows of one block and head (of several heads where a block has
// fewer rows than a wave holds): 16 values a lane, the chunks of a rotation pair in
// one lane, the block's maximum by lane permutations.  Values stay in fp32 registers
// from their load to their one rounding.
#pragma once

#include <algorithm>
#include <cstdlib>

#include "row_chunks.h"

namespace akv {
namespace {

#define KV8_INLINE __attribute__((always_inline))

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMostBlock = 64;      // slots of a scale block
constexpr int kMostHeadDim = 128;
constexpr uint32_t kLeastScale = (127 - 100) << 23;  // 2^-100

// Workgroups of a launch: a grid has fewer than 2^32 threads.
constexpr int64_t kMostBlocks = 1 << 23;

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Strides in bytes (codes) and elements (scales).
struct Cache {
  int64_t k_ss, k_sh, v_ss, v_sh;
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
  int64_t slots;
  int32_t heads, head_dim, log2_block;
};

struct Rope {
  const void* table;
  int64_t stride, rows;
  int32_t dim, dtype;  // dim 0: no rotation
  bool neox;
};

template <bool E5>
__device__ __forceinline__ float largest() { return E5 ? 57344.f : 448.f; }

// The smallest power of two s >= 2^-100 with top <= F s.
template <bool E5>
__device__ __forceinline__ float fitting(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  const int32_t e = static_cast<int32_t>(bits >> 23) - (E5 ? 15 : 8) + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  const int32_t s = e << 23;
  return __builtin_bit_cast(float, s > static_cast<int32_t>(kLeastScale) ? s : static_cast<int32_t>(kLeastScale));
}

// A block's scale once values up to `top` join those that `before` scales.  One
// that is no positive number scales nothing.
template <bool E5>
__device__ __forceinline__ float grown(float top, float before) {
  if (!(before > 0.f && before < INFINITY)) return fitting<E5>(top);
  const float holds = largest<E5>() * before;
  if (top <= holds) return before;
  if (before < __builtin_bit_cast(float, kLeastScale)) return fitting<E5>(top);
  const uint32_t x = __builtin_bit_cast(uint32_t, top), y = __builtin_bit_cast(uint32_t, holds);
  const int k = static_cast<int>(x >> 23) - static_cast<int>(y >> 23) + ((x & 0x7fffff) > (y & 0x7fffff) ? 1 : 0);
  return __builtin_ldexpf(before, k);
}

template <bool E5>
__device__ __forceinline__ void decode8(u32x2 w, float* x) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 lo = E5 ? __builtin_amdgcn_cvt_pk_f32_bf8(w[i], false) : __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
    const f32x2 hi = E5 ? __builtin_amdgcn_cvt_pk_f32_bf8(w[i], true) : __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
    x[4 * i] = lo.x, x[4 * i + 1] = lo.y, x[4 * i + 2] = hi.x, x[4 * i + 3] = hi.y;
  }
}

template <bool E5>
__device__ __forceinline__ u32x2 encode8(const float* x) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* y = x + 4 * i;
    uint32_t r;
    if (E5) {
      r = __builtin_amdgcn_cvt_pk_bf8_f32(y[0], y[1], 0, false);
      r = __builtin_amdgcn_cvt_pk_bf8_f32(y[2], y[3], r, true);
    } else {
      r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
    }
    w[i] = r;
  }
  return w;
}

// Eight codes at any address (the compiler knows that the target's global accesses
// need no alignment).
typedef u32x2 any_u32x2 __attribute__((aligned(1)));
typedef __attribute__((address_space(1))) any_u32x2 global_any_u32x2;

typedef uint32_t any_u32 __attribute__((aligned(1)));
typedef __attribute__((address_space(1))) any_u32 global_any_u32;

__device__ __forceinline__ u32x2 load_codes(const uint8_t* p) { return *((const global_any_u32x2*)p); }
__device__ __forceinline__ void store_codes(uint8_t* p, u32x2 w) { *((global_any_u32x2*)p) = w; }

// How a lane takes its 16 values of a row: element by element, in two chunks of
// eight, or in two chunks of two quads (a rotation that ends inside a chunk).
enum Mode { kByElement, kByChunk, kByQuad };

template <int MODE>
__device__ __forceinline__ u32x2 load_chunk(const uint8_t* p, int mid) {
  if constexpr (MODE == kByQuad) return u32x2{*((const global_any_u32*)p), *((const global_any_u32*)(p + mid))};
  return load_codes(p);
}
template <int MODE>
__device__ __forceinline__ void store_chunk(uint8_t* p, int mid, u32x2 w) {
  if constexpr (MODE == kByQuad) {
    *((global_any_u32*)p) = w[0];
    *((global_any_u32*)(p + mid)) = w[1];
  } else {
    store_codes(p, w);
  }
}

// Scales by address: named as global, since flat accesses wait for everything.
typedef __attribute__((address_space(1))) float global_float;
typedef __attribute__((address_space(1))) uint8_t global_byte;
__device__ __forceinline__ float load_scale(const float* p) { return *((const global_float*)p); }
__device__ __forceinline__ void store_scale(float* p, float s) { *((global_float*)p) = s; }

// A lane's 16 values of a row: 8 from at0 and 8 from at1 on, each in two quads, the
// second mid0 (mid1) elements behind the first.
struct Place {
  int at0, at1, mid0, mid1;
  bool turned;  // pairs of the rotation, coefficients 8 u + i
  bool all;     // all eight pairs, or the first four
};

template <int MODE>
__device__ __forceinline__ Place place_of(int u, bool rotates, const Rope& rope) {
  const bool turned = MODE != kByElement && rotates && 16 * u < rope.dim;
  const bool apart = turned && rope.neox;  // the halves of a neox pair lie R / 2 apart
  Place p{apart ? 8 * u : 16 * u, apart ? 8 * u + rope.dim / 2 : 16 * u + 8, 4, 4, turned, true};
  if (MODE == kByQuad && turned && 16 * u + 8 == rope.dim) {
    // the last four pairs, and the eight dims behind the rotation
    p.all = false;
    if (rope.neox) p.mid0 = rope.dim - p.at0, p.mid1 = rope.dim + 4 - p.at1;
  }
  return p;
}

// Turns a lane's eight pairs: (x, y) -> (x c - y s, y c + x s).
__device__ __forceinline__ void turn(float (&y)[16], const float (&c)[8], const float (&s)[8], bool neox) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int one = neox ? i : 2 * i, two = neox ? 8 + i : 2 * i + 1;
    const float p = y[one], r = y[two];
    y[one] = p * c[i] - r * s[i];
    y[two] = r * c[i] + p * s[i];
  }
}

// The same, with the form a uniform branch around register-only code.
__device__ __forceinline__ void turn_either(float (&y)[16], const float (&c)[8], const float (&s)[8], bool neox) {
  if (neox)
    turn(y, c, s, true);
  else
    turn(y, c, s, false);
}

// The same of the first four pairs, where those are all; the others' values stay.
template <int MODE>
__device__ __forceinline__ void turn_place(float (&y)[16], const float (&c)[8], const float (&s)[8], bool neox, bool all) {
  float kept[8];
  if constexpr (MODE == kByQuad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) kept[i] = neox && i < 4 ? y[4 + i] : y[8 + i];
  }
  turn_either(y, c, s, neox);
  if constexpr (MODE == kByQuad) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float& x = y[8 + i];
      x = all || (neox && i < 4) ? x : kept[i];
      if (i < 4) y[4 + i] = all || !neox ? y[4 + i] : kept[i];
    }
  }
}

// Element i < R of a row, element by element: its pair's number, whether it is the
// second of it, and the other one.
struct Pair {
  int number, other;
  bool second;
};
__device__ __forceinline__ Pair pair_of(int i, const Rope& rope) {
  const int half = rope.dim / 2;
  if (rope.neox) return {i < half ? i : i - half, i < half ? i + half : i - half, i >= half};
  return {i / 2, i ^ 1, (i & 1) != 0};
}

__device__ __forceinline__ float nan32() { return __builtin_nanf(""); }

// Where a lane stands in its wave: 16-element part u of row r (of `rows`) of the
// wave's sub-th head.
template <int LANES>
struct Stand {
  int u, r, sub, rows, span;
  __device__ __forceinline__ explicit Stand(int log2_block) {
    const int lane = threadIdx.x & 63;
    rows = 1 << log2_block < 64 / LANES ? 1 << log2_block : 64 / LANES;
    span = rows * LANES;
    u = lane % LANES;
    r = lane / LANES & (rows - 1);
    sub = lane / span;
  }
};

// Maximum over groups of `span` lanes (a power of two, uniform).  Lanes of a group
// of four, eight and sixteen by the lane permutations of a row of 16; then the rows.
template <int CTRL>
__device__ __forceinline__ float max_with(float x) {
  const int other = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true);
  return __builtin_fmaxf(x, __builtin_bit_cast(float, other));
}
__device__ __forceinline__ float max_across(float x, int half) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  uint32_t lo, hi;
  if (half == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    lo = r[0], hi = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    lo = r[0], hi = r[1];
  }
  return __builtin_fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
// (selects, no branches: loads and stores in flight around them stay counted)
template <int LANES>
__device__ __forceinline__ float group_max(float x, int span) {
  static_assert(LANES == 4 || LANES == 8, "a row is 4 or 8 lanes");
  x = max_with<0xb1>(x);  // quad_perm [1, 0, 3, 2]
  x = max_with<0x4e>(x);  // quad_perm [2, 3, 0, 1]
  const float by8 = max_with<0x141>(x);  // row_half_mirror
  x = LANES == 8 || span >= 8 ? by8 : x;
  const float by16 = max_with<0x140>(x);  // row_mirror
  x = span >= 16 ? by16 : x;
  const float by32 = max_across(x, 16);
  x = span >= 32 ? by32 : x;
  const float by64 = max_across(x, 32);
  return span >= 64 ? by64 : x;
}

// Largest magnitude of a lane's values in units of `by`, NaN left out (infinities too,
// where the first maximum is one).
__device__ __forceinline__ float largest_of(const float (&x)[16], float by, bool finite_only) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    float p = __builtin_fabsf(x[e]), q = __builtin_fabsf(x[e + 1]);
    if (finite_only) {
      p = __builtin_fabsf(x[e] * by) == INFINITY ? 0.f : p;
      q = __builtin_fabsf(x[e + 1] * by) == INFINITY ? 0.f : q;
    }
    m = __builtin_fmaxf(__builtin_fmaxf(m, p), q);
  }
  m *= __builtin_fabsf(by);
  return finite_only && m == INFINITY ? 0.f : m;
}

// The rows that a block holds below its offset `first`, from units of `before` to
// units of s.
template <bool E5, int LANES>
__device__ __forceinline__ void rescale(const Stand<LANES>& at, int first, uint8_t* block, int64_t stride, float before,
                                        float s) {
  const float ratio = before > 0.f && before < INFINITY ? before / s : 0.f;
  for (int o = at.r; o < first; o += at.rows) {
    uint8_t* row = block + o * stride + 16 * at.u;
    float x[16];
    decode8<E5>(load_codes(row), x);
    decode8<E5>(load_codes(row + 8), x + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= ratio;
    store_codes(row, encode8<E5>(x));
    store_codes(row + 8, encode8<E5>(x + 8));
  }
}

// One run: the rows that the call brings to one block of a head, from its offset
// `first` on (uniform).  value(it, i, z, unit) loads the lane's part of the run's row
// i = it * rows + r, z in units of `unit`, and says whether it is to be written (the same for
// all lanes of a row; where no row of a head is, neither is its scale); `block` is
// the block's first row at this lane's head, off[it] how far behind it the lane's part of
// the round's row lies (place: its chunks).  ITERS: rounds of rows that stay
// in registers (0: any number of rounds, loaded twice).  UNITS: units other than 1.
template <bool E5, int LANES, int ITERS, int MODE, bool UNITS, typename F>
__device__ __forceinline__ void write_run(const Stand<LANES>& at, bool in, int len, int first, uint8_t* block,
                                          int64_t stride, const int64_t* off, Place place, float* scale, F value) {
  constexpr int N = ITERS ? ITERS : 1;
  float z[N][16], unit[N];
  bool live[N];
  const float before = in && first ? load_scale(scale) : 0.f;
  float top = -1.f;  // below 0: no row is written (one of a unit that is no number counts as 0)
  auto settle = [&](bool finite_only) KV8_INLINE {
    top = -1.f;
    if constexpr (ITERS > 0) {
#pragma unroll
      for (int it = 0; it < N; ++it)
        if (live[it]) top = __builtin_fmaxf(__builtin_fmaxf(top, 0.f), largest_of(z[it], unit[it], finite_only));
    } else {
      for (int it = 0; it * at.rows < len; ++it) {
        const int i = it * at.rows + at.r;
        if (in && i < len && value(it, i, z[0], unit[0]))
          top = __builtin_fmaxf(__builtin_fmaxf(top, 0.f), largest_of(z[0], unit[0], finite_only));
      }
    }
    top = group_max<LANES>(top, at.span);
  };
#pragma unroll
  for (int it = 0; it < N; ++it) unit[it] = 1.f;
  if constexpr (ITERS > 0) {
#pragma unroll
    for (int it = 0; it < N; ++it) {
      const int i = it * at.rows + at.r;
      live[it] = in && i < len;
      if (live[it]) live[it] = value(it, i, z[it], unit[it]);
    }
  }
  settle(false);
  if (__builtin_amdgcn_ballot_w64(!(top < INFINITY))) settle(true);
  const float s = first ? grown<E5>(top, before) : fitting<E5>(top);
  // 1 / s: of a power of two by its bits; behind other rows s may be any number, also one
  // whose inverse is past fp32's range: then 2^-24 / s, of values times 2^24
  float inverse = __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, s));
  bool tiny = false;
  if (first) {
    tiny = s < 0x1p-126f;
    inverse = 1.f / (tiny ? s * 0x1p24f : s);
  }
  auto write = [&](float (&x)[16], float by, uint8_t* row) KV8_INLINE {
    if (tiny) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= 0x1p24f;
    }
    float f = inverse;
    if (UNITS) {
      f *= by;
      if (f == INFINITY && by < INFINITY) f = 0x1.fffffep127f;  // (a row of zeros)
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] *= f;
    store_chunk<MODE>(row, place.mid0, encode8<E5>(x));
    store_chunk<MODE>(row + (place.at1 - place.at0), place.mid1, encode8<E5>(x + 8));
  };
  if constexpr (ITERS > 0) {
#pragma unroll
    for (int it = 0; it < N; ++it)
      if (live[it]) write(z[it], unit[it], block + off[it]);
  } else {
    for (int it = 0; it * at.rows < len; ++it) {
      const int i = it * at.rows + at.r;
      if (in && i < len && value(it, i, z[0], unit[0])) write(z[0], unit[0], block + off[0] + it * at.rows * stride);
    }
  }
  if (!in || top < 0.f) return;  // (what the block holds keeps its scale)
  if (first && s != before) rescale<E5>(at, first, block, stride, before, s);
  if (at.u == 0 && at.r == 0) store_scale(scale, s);
}

// A lane's 64-bit value at lane `at` (uniform).
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int at) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), at);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), at);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// The run that begins at entry t of a list of slots: its length, 0 where it began
// earlier or the entry has no slot (skip: entries to pass over).  slot_at(i): entry
// i, -1 where it has none; before: entry t - 1.
struct Run {
  int64_t slot;
  int len, skip;
};
template <typename F>
__device__ __forceinline__ Run run_at(F slot_at, int64_t t, int64_t n, int32_t log2_block, int64_t before) {
  const int lane = threadIdx.x & 63, B = 1 << log2_block;
  const int64_t mine = slot_at(t + lane < n ? t + lane : n - 1);
  const int64_t cur = static_cast<int64_t>(lane_value(static_cast<uint64_t>(mine), 0));
  const int64_t last = static_cast<int64_t>(lane_value(static_cast<uint64_t>(before), 0));
  if (cur < 0) return {cur, 0, 1};
  const int off = static_cast<int>(cur & (B - 1));
  const bool follows = t + lane < n && off + lane < B && mine == cur + lane;
  const uint64_t other = ~__builtin_amdgcn_ballot_w64(follows);
  const int len = other ? __builtin_ctzll(other) : 64;
  return {cur, off && last == cur - 1 ? 0 : len, len};
}

// Lanes of a row.
int lanes_of(int32_t head_dim) { return head_dim <= 64 ? 4 : 8; }

// A constant as an argument.
template <int N>
struct Number {
  static constexpr int value = N;
};
// What both calls ask of the cache; 0 or a failure with `who` in its message.
int check_cache(const char* who, int32_t format, int32_t heads, int32_t head_dim, int32_t rotary_dim,
                int32_t scale_block, int64_t slots) {
  if (format != AKV_E4M3 && format != AKV_E5M2)
    return fail(AKV_EINVAL, "%s: the cache must be e4m3 or e5m2", who);
  if (heads <= 0 || heads > 32767) return fail(AKV_EINVAL, "%s: %d KV heads", who, heads);
  if (head_dim < 16 || head_dim > kMostHeadDim || head_dim % 16)
    return fail(AKV_EINVAL, "%s: head_dim %d (multiples of 16 up to %d)", who, head_dim, kMostHeadDim);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(AKV_EINVAL, "%s: rotary_dim %d of %d", who, rotary_dim, head_dim);
  if (scale_block < 1 || scale_block > kMostBlock || (scale_block & (scale_block - 1)))
    return fail(AKV_EINVAL, "%s: scale_block %d (powers of two up to %d)", who, scale_block, kMostBlock);
  if (slots < 0) return fail(AKV_EINVAL, "%s: negative size", who);
  return AKV_OK;
}

// Rows and scales that a call writes lie apart: two waves write any two of them.
int check_apart(const char* who, const Cache& c) {
  const bool heads = c.slots > 0 && c.heads > 1, slots = c.slots > 1, blocks = c.slots > 1ll << c.log2_block;
  auto close = [](int64_t one, int64_t two, int64_t to) { return std::abs(one) < to || std::abs(two) < to; };
  if ((heads && close(c.k_sh, c.v_sh, c.head_dim)) || (slots && close(c.k_ss, c.v_ss, c.head_dim)) ||
      (heads && close(c.ks_sh, c.vs_sh, 1)) || (blocks && close(c.ks_sb, c.vs_sb, 1)))
    return fail(AKV_EINVAL, "%s: rows or scales of the cache overlap", who);
  return AKV_OK;
}

int log2_of(int32_t x) { return __builtin_ctz(static_cast<uint32_t>(x)); }

bool float_dtype(int32_t d) { return d == AKV_F32 || d == AKV_F16 || d == AKV_BF16; }

bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace
}  // namespace akv
