// Rows into a cache held in 8 bits, with a scale for each block of slots and
// head: new ones with the rotation on the way, and kept ones moved to fresh
// slots and new positions (gfx950).
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
// smallest normal one).  F = 1.75 2^n in both types, so s is read off the bits of A.
//
// A wave takes the rows of one block and head (of several heads where a block has
// fewer rows than a wave holds): 16 values a lane, the chunks of a rotation pair in
// one lane, the block's maximum by lane swaps.  Values stay in fp32 registers from
// their load to their one rounding.
#include <algorithm>

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

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) u32x2 global_u32x2;

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

struct AppendArgs {
  Cache c;
  Rope rope;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh;
  uint8_t* k_pool;
  uint8_t* v_pool;
  float* k_scales;
  float* v_scales;
  const void* slots;
  const void* positions;
  int64_t n_tokens;
  int64_t kv_units, q_units, q_parts;  // waves for the cache, for q, for a token's q rows
  int32_t window, head_groups;
  int32_t q_heads;
  bool slots64, pos64, whole;  // whole: codes on multiples of 8
};

struct MoveArgs {
  Cache c;
  Rope rope;
  const uint64_t* k_ptrs;
  const uint64_t* v_ptrs;
  const uint64_t* k_scale_ptrs;
  const uint64_t* v_scale_ptrs;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* pairs;
  const int32_t* gate;
  int64_t pair_stride, n_tokens, units, windows;
  int32_t window, head_groups, n_layers, layers;  // layers: of a wave
  bool skip_zero, whole;
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

// Eight codes at any address; `whole` (uniform): a multiple of 8.
__device__ __forceinline__ u32x2 load_codes(const uint8_t* p, bool whole) {
  if (whole) return *((const global_u32x2*)p);
  u32x2 w = {0u, 0u};
  for (int i = 0; i < 8; ++i) w[i / 4] |= static_cast<uint32_t>(p[i]) << 8 * (i % 4);
  return w;
}

__device__ __forceinline__ void store_codes(uint8_t* p, u32x2 w, bool whole) {
  if (whole) {
    *((global_u32x2*)p) = w;
    return;
  }
  for (int i = 0; i < 8; ++i) p[i] = static_cast<uint8_t>(w[i / 4] >> 8 * (i % 4));
}

// A lane's 16 values of a row, 8 from at0 and 8 from at1 on.
struct Place {
  int at0, at1;
  bool turned;  // pairs of the rotation, coefficients 8 u + i (vector kernels)
};

template <bool VEC>
__device__ __forceinline__ Place place_of(int u, bool rotates, const Rope& rope) {
  const bool turned = VEC && rotates && 16 * u < rope.dim;
  const bool apart = turned && rope.neox;  // the halves of a neox pair lie R / 2 apart
  return {apart ? 8 * u : 16 * u, apart ? 8 * u + rope.dim / 2 : 16 * u + 8, turned};
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

// One run: the rows that the call brings to one block of a head, from its offset
// `first` on.  value(it, i, y) loads the lane's part of the run's row i = it * rows +
// r and says whether it is to be written; `block` is the block's first row at this
// lane's head.  ITERS: rounds of rows that stay in registers (0: any number of
// rounds, loaded twice).
template <bool E5, int LANES, int ITERS, typename F>
__device__ __forceinline__ void write_run(const Stand<LANES>& at, bool in, int len, int first, uint8_t* block,
                                          int64_t stride, float* scale, Place place, bool whole, F value) {
  constexpr int N = ITERS ? ITERS : 1;
  float y[N][16];
  bool live[N];
  const float before = in && first ? *scale : 0.f;
  float top = 0.f;
  auto largest_of = [&](const float (&x)[16], bool finite_only) KV8_INLINE {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float m = __builtin_fabsf(x[e]);
      top = __builtin_fmaxf(top, finite_only && m == INFINITY ? 0.f : m);  // (NaN is left out)
    }
  };
  auto settle = [&](bool finite_only) KV8_INLINE {
    top = 0.f;
    if constexpr (ITERS > 0) {
#pragma unroll
      for (int it = 0; it < N; ++it)
        if (live[it]) largest_of(y[it], finite_only);
    } else {
      for (int it = 0; it * at.rows < len; ++it) {
        const int i = it * at.rows + at.r;
        if (in && i < len && value(it, i, y[0])) largest_of(y[0], finite_only);
      }
    }
    for (int off = 1; off < at.span; off <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off));
  };
  if constexpr (ITERS > 0) {
#pragma unroll
    for (int it = 0; it < N; ++it) {
      const int i = it * at.rows + at.r;
      live[it] = in && i < len;
      if (live[it]) live[it] = value(it, i, y[it]);
    }
  }
  settle(false);
  if (__builtin_amdgcn_ballot_w64(top == INFINITY)) settle(true);
  const float s = first ? grown<E5>(top, before) : fitting<E5>(top);
  const bool simple = (__builtin_bit_cast(uint32_t, s) & 0x7fffff) == 0;  // a power of two: y / s = y (1 / s)
  const float inv = 1.f / s;
  const bool all_simple = __builtin_amdgcn_ballot_w64(in && !simple) == 0;
  auto write = [&](float (&x)[16], int i) KV8_INLINE {
    uint8_t* row = block + (first + i) * stride;
    if (all_simple) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= inv;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] /= s;
    }
    store_codes(row + place.at0, encode8<E5>(x), whole);
    store_codes(row + place.at1, encode8<E5>(x + 8), whole);
  };
  if constexpr (ITERS > 0) {
#pragma unroll
    for (int it = 0; it < N; ++it)
      if (live[it]) write(y[it], it * at.rows + at.r);
  } else {
    for (int it = 0; it * at.rows < len; ++it) {
      const int i = it * at.rows + at.r;
      if (in && i < len && value(it, i, y[0])) write(y[0], i);
    }
  }
  if (!in) return;
  if (first && s != before) {
    // the rows that the block holds, in units of its new scale
    const float ratio = before > 0.f && before < INFINITY ? before / s : 0.f;
    for (int o = at.r; o < first; o += at.rows) {
      uint8_t* row = block + o * stride + 16 * at.u;
      float x[16];
      decode8<E5>(load_codes(row, whole), x);
      decode8<E5>(load_codes(row + 8, whole), x + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] *= ratio;
      store_codes(row, encode8<E5>(x), whole);
      store_codes(row + 8, encode8<E5>(x + 8), whole);
    }
  }
  if (at.u == 0 && at.r == 0) *scale = s;
}

// The run that begins at entry t of a list of slots: its length, 0 where it began
// earlier or the entry has no slot (skip: entries to pass over).  slot_at(i): entry
// i, -1 where it has none.
struct Run {
  int64_t slot;
  int len, skip;
};
template <typename F>
__device__ __forceinline__ Run run_at(F slot_at, int64_t t, int64_t n, int32_t log2_block) {
  const int lane = threadIdx.x & 63, B = 1 << log2_block;
  const int64_t before = t > 0 ? slot_at(t - 1) : -1;
  const int64_t mine = slot_at(t + lane < n ? t + lane : n - 1), cur = slot_at(t);
  if (cur < 0) return {cur, 0, 1};
  const int off = static_cast<int>(cur & (B - 1));
  const bool follows = t + lane < n && off + lane < B && mine == cur + lane;
  const uint64_t other = ~__builtin_amdgcn_ballot_w64(follows);
  const int len = other ? __builtin_ctzll(other) : 64;
  return {cur, off && before == cur - 1 ? 0 : len, len};
}

// VEC: whole chunks of 8, pairs of the rotation within a lane; else element by
// element.
template <typename T, bool E5, int LANES, int ITERS, bool VEC>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendArgs a) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rope& rope = a.rope;
  auto position = [&](int64_t t) -> int64_t {
    const int64_t p = load_index(a.positions, a.pos64, t);
    return p >= 0 && p < rope.rows ? p : -1;
  };
  // cos and sin of a lane's eight pairs
  auto coefficients = [&](int64_t p, int u, float (&c)[8], float (&s)[8]) KV8_INLINE {
    load8(rope.table, rope.dtype, p * rope.stride + 8 * u, c);
    load8(rope.table, rope.dtype, p * rope.stride + rope.dim / 2 + 8 * u, s);
  };
  // part u of a row, element by element; rotates: by the row p of the table
  auto by_element = [&](const T* from, int u, bool rotates, int64_t p, float (&y)[16]) KV8_INLINE {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      __builtin_amdgcn_sched_barrier(0);  // (few elements in flight: registers)
      const int i = 16 * u + e;
      float x = to_f32(from[i]);
      if (rotates && i < rope.dim && p >= 0) {
        const Pair w = pair_of(i, rope);
        const float c = load1(rope.table, rope.dtype, p * rope.stride + w.number);
        const float s = load1(rope.table, rope.dtype, p * rope.stride + rope.dim / 2 + w.number);
        const float o = to_f32(from[w.other]);
        x = w.second ? x * c + o * s : x * c - o * s;
      }
      y[e] = x;
    }
  };
  auto part = [&](const T* from, Place place, float (&y)[16]) KV8_INLINE {
    Chunk<T> x0, x1;
    x0.load(from + place.at0);
    x1.load(from + place.at1);
    float (&lo)[8] = *reinterpret_cast<float (*)[8]>(y), (&hi)[8] = *reinterpret_cast<float (*)[8]>(y + 8);
    x0.get(lo);
    x1.get(hi);
  };

  if (unit >= a.kv_units) {
    // q rows: 64 / LANES heads at a time, the token's cos and sin kept
    const int64_t mine = unit - a.kv_units;
    if (mine >= a.q_units) return;
    const int64_t t = mine / a.q_parts;
    const int first = static_cast<int>(mine - t * a.q_parts);
    const int u = threadIdx.x % LANES, sub = (threadIdx.x & 63) / LANES;
    const Place place = place_of<VEC>(u, true, rope);
    const int64_t p = position(t);
    float c[8], s[8];
    if (place.turned && p >= 0) coefficients(p, u, c, s);
    for (int head = first * (64 / LANES) + sub; head < a.q_heads; head += static_cast<int>(a.q_parts) * (64 / LANES)) {
      if (16 * u >= a.c.head_dim) break;
      const T* from = static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh;
      T* to = static_cast<T*>(a.q_out) + t * a.qo_st + head * a.qo_sh;
      float y[16];
      if constexpr (!VEC) {
        // (q_out may be q: all of a row is read before any of it is written)
        by_element(from, u, true, p, y);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 16; ++e) to[16 * u + e] = static_cast<T>(p < 0 ? nan32() : y[e]);
      } else {
        part(from, place, y);
        if (place.turned && p >= 0) turn_either(y, c, s, rope.neox);
        if (p < 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = nan32();
        }
        Chunk<T> x0, x1;
        x0.set(*reinterpret_cast<float (*)[8]>(y));
        x1.set(*reinterpret_cast<float (*)[8]>(y + 8));
        x0.store(to + place.at0);
        x1.store(to + place.at1);
      }
    }
    return;
  }

  const Stand<LANES> at(a.c.log2_block);
  const int64_t w = unit / a.head_groups;
  const int row = static_cast<int>(unit - w * a.head_groups) * (64 / at.span) + at.sub;  // K heads, then V heads
  const bool in = row < 2 * a.c.heads && 16 * at.u < a.c.head_dim;
  const bool is_v = row >= a.c.heads;
  const int head = is_v ? row - a.c.heads : row;
  const bool rotates = !is_v && rope.dim > 0;
  const Place place = place_of<VEC>(at.u, rotates, rope);
  const T* rows = is_v ? static_cast<const T*>(a.v) + head * a.v_sh : static_cast<const T*>(a.k) + head * a.k_sh;
  const int64_t row_stride = is_v ? a.v_st : a.k_st;
  uint8_t* pool = is_v ? a.v_pool + head * a.c.v_sh : a.k_pool + head * a.c.k_sh;
  const int64_t slot_stride = is_v ? a.c.v_ss : a.c.k_ss;
  float* scales = is_v ? a.v_scales + head * a.c.vs_sh : a.k_scales + head * a.c.ks_sh;
  const int64_t block_stride = is_v ? a.c.vs_sb : a.c.ks_sb;
  auto slot_at = [&](int64_t t) -> int64_t {
    const int64_t s = load_index(a.slots, a.slots64, t);
    return s >= 0 && s < a.c.slots ? s : -1;
  };
  const int64_t end = std::min<int64_t>(a.n_tokens, (w + 1) * a.window);
  for (int64_t t = w * a.window; t < end;) {
    const Run run = run_at(slot_at, t, a.n_tokens, a.c.log2_block);
    if (run.len) {
      const int64_t block = run.slot >> a.c.log2_block;
      const int first = static_cast<int>(run.slot - (block << a.c.log2_block));
      write_run<E5, LANES, ITERS>(
          at, in, run.len, first, pool + (block << a.c.log2_block) * slot_stride, slot_stride,
          scales + block * block_stride, place, a.whole, [&](int, int i, float (&y)[16]) KV8_INLINE {
            const T* from = rows + (t + i) * row_stride;
            const int64_t p = rotates ? position(t + i) : 0;
            if constexpr (!VEC) {
              by_element(from, at.u, rotates, p, y);
            } else {
              part(from, place, y);
              if (place.turned && p >= 0) {
                float c[8], s[8];
                coefficients(p, at.u, c, s);
                turn_either(y, c, s, rope.neox);
              }
            }
            if (p < 0) {
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = nan32();
            }
            return true;
          });
    }
    t += run.skip;
  }
}

template <bool E5, int LANES, int ITERS, bool VEC>
__global__ void __launch_bounds__(kThreads) kv8_move_kernel(const MoveArgs a) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (unit >= a.units || gated(a.gate)) return;
  constexpr int N = ITERS ? ITERS : 1;
  const Rope& rope = a.rope;
  const Stand<LANES> at(a.c.log2_block);
  // head groups fastest, then windows of tokens, then groups of layers
  const int64_t of_heads = unit / a.head_groups;
  const int row = static_cast<int>(unit - of_heads * a.head_groups) * (64 / at.span) + at.sub;
  const int layer_group = static_cast<int>(of_heads / a.windows);
  const int64_t w = of_heads - layer_group * a.windows;
  const int layer0 = layer_group * a.layers, layer1 = std::min(a.n_layers, layer0 + a.layers);
  const bool in = row < 2 * a.c.heads && 16 * at.u < a.c.head_dim;
  const bool is_v = row >= a.c.heads;
  const int head = is_v ? row - a.c.heads : row;
  const bool rotates = !is_v;
  const Place place = place_of<VEC>(at.u, rotates, rope);
  const int64_t head_at = head * (is_v ? a.c.v_sh : a.c.k_sh), slot_stride = is_v ? a.c.v_ss : a.c.k_ss;
  const int64_t scale_at = head * (is_v ? a.c.vs_sh : a.c.ks_sh), block_stride = is_v ? a.c.vs_sb : a.c.ks_sb;
  const uint64_t* layers = is_v ? a.v_ptrs : a.k_ptrs;
  const uint64_t* layer_scales = is_v ? a.v_scale_ptrs : a.k_scale_ptrs;
  auto usable = [&](int64_t s) { return s >= (a.skip_zero ? 1 : 0) && s < a.c.slots; };
  auto slot_at = [&](int64_t t) -> int64_t {
    const int64_t s = a.dst[t];
    return usable(s) ? s : -1;
  };
  // a rotation by the difference of two positions: the old one's undone, the new
  // one's done, one factor pair for every layer and head
  auto factor = [&](float co, float so, float cn, float sn, float* c, float* s) {
    const float norm = co * co + so * so;
    *c = (cn * co + sn * so) / norm;
    *s = (sn * co - cn * so) / norm;
  };
  struct Moved {
    int64_t src;          // -1: not moved
    int64_t before, now;  // positions; -1: not in the table
    bool same;
    float c[8], s[8];
  };
  auto look_up = [&](int64_t t, Moved& m) KV8_INLINE {
    const int64_t s = a.src[t];
    m.src = usable(s) ? s : -1;
    const int64_t p = a.pairs[t * a.pair_stride], n = a.pairs[t * a.pair_stride + 1];
    m.same = p == n;
    const bool known = p >= 0 && p < rope.rows && n >= 0 && n < rope.rows;
    m.before = known ? p : -1;
    m.now = n;
    if (place.turned && known && !m.same) {
      float co[8], so[8], cn[8], sn[8];
      load8(rope.table, rope.dtype, p * rope.stride + 8 * at.u, co);
      load8(rope.table, rope.dtype, p * rope.stride + rope.dim / 2 + 8 * at.u, so);
      load8(rope.table, rope.dtype, n * rope.stride + 8 * at.u, cn);
      load8(rope.table, rope.dtype, n * rope.stride + rope.dim / 2 + 8 * at.u, sn);
#pragma unroll
      for (int i = 0; i < 8; ++i) factor(co[i], so[i], cn[i], sn[i], &m.c[i], &m.s[i]);
    }
  };
  const int64_t end = std::min<int64_t>(a.n_tokens, (w + 1) * a.window);
  for (int64_t t = w * a.window; t < end;) {
    const Run run = run_at(slot_at, t, a.n_tokens, a.c.log2_block);
    if (run.len) {
      const int64_t block = run.slot >> a.c.log2_block;
      const int first = static_cast<int>(run.slot - (block << a.c.log2_block));
      Moved moved[N];
      if constexpr (ITERS > 0) {
#pragma unroll
        for (int it = 0; it < N; ++it)
          if (it * at.rows + at.r < run.len) look_up(t + it * at.rows + at.r, moved[it]);
      }
      for (int layer = layer0; layer < layer1; ++layer) {
        uint8_t* codes = reinterpret_cast<uint8_t*>(in ? layers[layer] : 0) + head_at;
        float* scales = reinterpret_cast<float*>(in ? layer_scales[layer] : 0) + scale_at;
        const bool whole =
            a.whole && __builtin_amdgcn_ballot_w64(in && (reinterpret_cast<uintptr_t>(codes) & 7) != 0) == 0;
        write_run<E5, LANES, ITERS>(
            at, in, run.len, first, codes + (block << a.c.log2_block) * slot_stride, slot_stride,
            scales + block * block_stride, place, whole, [&](int it, int i, float (&y)[16]) KV8_INLINE {
              if constexpr (ITERS == 0) look_up(t + i, moved[0]);
              const Moved& m = moved[ITERS ? it : 0];
              if (m.src < 0) return false;
              const uint8_t* from = codes + m.src * slot_stride;
              const float scale = scales[(m.src >> a.c.log2_block) * block_stride];
              decode8<E5>(load_codes(from + place.at0, whole), y);
              decode8<E5>(load_codes(from + place.at1, whole), y + 8);
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] *= scale;
              if (!rotates || m.same) return true;
              if (m.before < 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = nan32();
              } else if constexpr (VEC) {
                if (place.turned) turn_either(y, m.c, m.s, rope.neox);
              } else {
                const int half = rope.dim / 2;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  __builtin_amdgcn_sched_barrier(0);
                  const int d = 16 * at.u + e;
                  if (d >= rope.dim) continue;
                  const Pair w = pair_of(d, rope);
                  auto entry = [&](int64_t p, int j) { return load1(rope.table, rope.dtype, p * rope.stride + j); };
                  float c, s;
                  factor(entry(m.before, w.number), entry(m.before, half + w.number), entry(m.now, w.number),
                         entry(m.now, half + w.number), &c, &s);
                  const uint32_t code = from[w.other];
                  const float o =
                      (E5 ? __builtin_amdgcn_cvt_f32_bf8(code, 0) : __builtin_amdgcn_cvt_f32_fp8(code, 0)) * scale;
                  y[e] = w.second ? y[e] * c + o * s : y[e] * c - o * s;
                }
              }
              return true;
            });
      }
    }
    t += run.skip;
  }
}

// Lanes of a row, and the rounds of rows that a wave takes for a block.
int lanes_of(int32_t head_dim) { return head_dim <= 64 ? 4 : 8; }

struct Shape {
  int lanes, iters, per_wave, groups;
};
Shape shape_of(const Cache& c) {
  Shape s;
  s.lanes = lanes_of(c.head_dim);
  const int block = 1 << c.log2_block, most = 64 / s.lanes;
  s.iters = (block + most - 1) / most;
  s.per_wave = 64 / (s.lanes * std::min(block, most));  // heads
  s.groups = (2 * c.heads + s.per_wave - 1) / s.per_wave;
  return s;
}

// Calls f with the kernel's LANES, ITERS and VEC as constants.
template <int N>
struct Number {
  static constexpr int value = N;
};
template <typename F>
void with_shape(const Shape& s, bool vec, F f) {
  auto of_lanes = [&](auto lanes) {
    if (!vec) f(lanes, Number<0>{}, Number<0>{});
    else if (s.iters == 1) f(lanes, Number<1>{}, Number<1>{});
    else if (s.iters == 2) f(lanes, Number<2>{}, Number<1>{});
    else f(lanes, Number<0>{}, Number<1>{});
  };
  if (s.lanes == 4) of_lanes(Number<4>{});
  else of_lanes(Number<8>{});
}

int64_t waves_to_blocks(int64_t waves) { return (waves + kWaves - 1) / kWaves; }

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

int log2_of(int32_t x) { return __builtin_ctz(static_cast<uint32_t>(x)); }

bool float_dtype(int32_t d) { return d == AKV_F32 || d == AKV_F16 || d == AKV_BF16; }

bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace
}  // namespace akv

extern "C" int akv_kv8_append(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                              int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h, int32_t dtype,
                              int64_t n_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                              int32_t rotary_dim, int32_t is_neox, const void* positions, int32_t positions_dtype,
                              const void* cos_sin, int32_t cos_sin_dtype, int64_t rope_stride, int64_t rope_rows,
                              void* q_out, int64_t qo_stride_t, int64_t qo_stride_h, const void* slots,
                              int32_t slots_dtype, void* k_pool, void* v_pool, int32_t format, int64_t pool_slots,
                              int64_t kp_stride_slot, int64_t kp_stride_head, int64_t vp_stride_slot,
                              int64_t vp_stride_head, float* k_scales, float* v_scales, int32_t scale_block,
                              int64_t ks_stride_block, int64_t ks_stride_head, int64_t vs_stride_block,
                              int64_t vs_stride_head, void* stream) {
  using namespace akv;
  const char* who = "akv_kv8_append";
  int rc = check_cache(who, format, kv_heads, head_dim, rotary_dim, scale_block, pool_slots);
  if (rc) return rc;
  if (!float_dtype(dtype) || !float_dtype(cos_sin_dtype))
    return fail(AKV_EINVAL, "%s: dtypes must be float32, float16 or bfloat16", who);
  if (!valid_index_dtype(positions_dtype) || !valid_index_dtype(slots_dtype))
    return fail(AKV_EINVAL, "%s: index vectors must be int32 or int64", who);
  if (n_tokens < 0 || q_heads < 0 || q_heads > 65535 || rope_rows < 0)
    return fail(AKV_EINVAL, "%s: invalid size", who);
  if (q_heads && !rotary_dim) return fail(AKV_EINVAL, "%s: q without a rotation", who);
  if (n_tokens == 0) return AKV_OK;
  if (n_tokens > INT32_MAX) return fail(AKV_EINVAL, "%s: %lld tokens", who, static_cast<long long>(n_tokens));
  if ((q_heads && (!q || !q_out)) || !k || !v || !slots || (rotary_dim && (!positions || !cos_sin)) ||
      (pool_slots > 0 && (!k_pool || !v_pool || !k_scales || !v_scales)))
    return fail(AKV_EINVAL, "%s: null device pointer", who);
  AppendArgs a{};
  a.c = Cache{kp_stride_slot, kp_stride_head, vp_stride_slot, vp_stride_head, ks_stride_block, ks_stride_head,
              vs_stride_block, vs_stride_head, pool_slots, kv_heads, head_dim, log2_of(scale_block)};
  a.rope = Rope{cos_sin, rope_stride, rope_rows, rotary_dim, cos_sin_dtype, is_neox != 0};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.qo_st = qo_stride_t;
  a.qo_sh = qo_stride_h;
  a.k_pool = static_cast<uint8_t*>(k_pool);
  a.v_pool = static_cast<uint8_t*>(v_pool);
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.slots = slots;
  a.positions = positions;
  a.n_tokens = n_tokens;
  a.q_heads = q_heads;
  a.slots64 = slots_dtype == AKV_I64;
  a.pos64 = positions_dtype == AKV_I64;
  // whole chunks of 8 on 16-byte (codes: 8-byte) boundaries, pairs within a lane
  const int e = dtype == AKV_F32 ? 4 : 2, te = cos_sin_dtype == AKV_F32 ? 4 : 2;
  a.whole = aligned(k_pool, 8) && aligned(v_pool, 8) &&
            (kp_stride_slot | kp_stride_head | vp_stride_slot | vp_stride_head) % 8 == 0;
  const bool vec =
      rotary_dim % 16 == 0 && aligned(k, 16) && aligned(v, 16) &&
          ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) * e) % 16 == 0 &&
          (!rotary_dim || (aligned(cos_sin, 16) && rope_stride * te % 16 == 0)) &&
          (!q_heads || (aligned(q, 16) && aligned(q_out, 16) &&
                        ((q_stride_t | q_stride_h | qo_stride_t | qo_stride_h) * e) % 16 == 0));
  const Shape shape = shape_of(a.c);
  a.head_groups = shape.groups;
  a.window = 1;
  while (a.window < scale_block && n_tokens * shape.groups > 16384ll * a.window) a.window *= 2;
  a.kv_units = pool_slots ? (n_tokens + a.window - 1) / a.window * shape.groups : 0;
  const int rounds = (q_heads + 64 / shape.lanes - 1) / (64 / shape.lanes);
  a.q_parts = n_tokens >= 2048 ? 1 : std::max(1, rounds);
  a.q_units = q_heads ? n_tokens * a.q_parts : 0;
  const int64_t blocks = waves_to_blocks(a.kv_units + a.q_units);
  if (blocks == 0) return AKV_OK;
  if (blocks > kMostBlocks) return fail(AKV_EINVAL, "%s: batch too large", who);
  hipStream_t st = as_stream(stream);
  auto start = [&](auto type, auto e5) {
    using T = decltype(type);
    with_shape(shape, vec, [&](auto lanes, auto iters, auto by_chunk) {
      hipLaunchKernelGGL((kv8_append_kernel<T, decltype(e5)::value != 0, decltype(lanes)::value, decltype(iters)::value,
                                            decltype(by_chunk)::value != 0>),
                         dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
    });
  };
  auto by_type = [&](auto e5) {
    if (dtype == AKV_F32) start(float{}, e5);
    else if (dtype == AKV_F16) start(_Float16{}, e5);
    else start(__bf16{}, e5);
  };
  if (format == AKV_E5M2) by_type(Number<1>{});
  else by_type(Number<0>{});
  return check_launch(who);
}

extern "C" int akv_kv8_reposition(const uint64_t* k_ptrs, const uint64_t* v_ptrs, const uint64_t* k_scale_ptrs,
                                  const uint64_t* v_scale_ptrs, int32_t n_layers, int32_t format, int32_t n_heads,
                                  int32_t head_dim, int32_t rotary_dim, int64_t pool_slots, int64_t k_stride_slot,
                                  int64_t k_stride_head, int64_t v_stride_slot, int64_t v_stride_head,
                                  int32_t scale_block, int64_t ks_stride_block, int64_t ks_stride_head,
                                  int64_t vs_stride_block, int64_t vs_stride_head, const int32_t* src,
                                  const int32_t* dst, const int32_t* pairs, int64_t pair_stride, int64_t n_tokens,
                                  const void* cos_sin, int32_t cos_sin_dtype, int64_t rope_stride, int64_t rope_rows,
                                  int32_t is_neox, int32_t skip_unmapped, const int32_t* status, void* stream) {
  using namespace akv;
  const char* who = "akv_kv8_reposition";
  int rc = check_cache(who, format, n_heads, head_dim, rotary_dim, scale_block, pool_slots);
  if (rc) return rc;
  if (rotary_dim == 0) return fail(AKV_EINVAL, "%s: rotary_dim 0 of %d", who, head_dim);
  if (!float_dtype(cos_sin_dtype)) return fail(AKV_EINVAL, "%s: unsupported cos_sin dtype %d", who, cos_sin_dtype);
  if (n_layers < 0 || n_tokens < 0 || rope_rows < 0 || pair_stride < 0) return fail(AKV_EINVAL, "%s: negative size", who);
  if (n_tokens == 0 || n_layers == 0 || pool_slots == 0) return AKV_OK;
  if (n_tokens > INT32_MAX) return fail(AKV_EINVAL, "%s: %lld tokens", who, static_cast<long long>(n_tokens));
  if (!k_ptrs || !v_ptrs || !k_scale_ptrs || !v_scale_ptrs || !src || !dst || !pairs || !cos_sin)
    return fail(AKV_EINVAL, "%s: null device pointer", who);
  MoveArgs a{};
  a.c = Cache{k_stride_slot, k_stride_head, v_stride_slot, v_stride_head, ks_stride_block, ks_stride_head,
              vs_stride_block, vs_stride_head, pool_slots, n_heads, head_dim, log2_of(scale_block)};
  a.rope = Rope{cos_sin, rope_stride, rope_rows, rotary_dim, cos_sin_dtype, is_neox != 0};
  a.k_ptrs = k_ptrs;
  a.v_ptrs = v_ptrs;
  a.k_scale_ptrs = k_scale_ptrs;
  a.v_scale_ptrs = v_scale_ptrs;
  a.src = src;
  a.dst = dst;
  a.pairs = pairs;
  a.pair_stride = pair_stride;
  a.gate = status;
  a.n_tokens = n_tokens;
  a.n_layers = n_layers;
  a.skip_zero = skip_unmapped != 0;
  const int te = cos_sin_dtype == AKV_F32 ? 4 : 2;
  a.whole = (k_stride_slot | k_stride_head | v_stride_slot | v_stride_head) % 8 == 0;
  const bool vec = rotary_dim % 16 == 0 && aligned(cos_sin, 16) && rope_stride * te % 16 == 0;
  const Shape shape = shape_of(a.c);
  a.head_groups = shape.groups;
  a.layers = std::min(n_layers, 4);
  const int64_t layer_groups = (n_layers + a.layers - 1) / a.layers;
  a.window = 1;
  while (a.window < scale_block && n_tokens * shape.groups * layer_groups > 16384ll * a.window) a.window *= 2;
  a.windows = (n_tokens + a.window - 1) / a.window;
  a.units = a.windows * layer_groups * shape.groups;
  const int64_t blocks = waves_to_blocks(a.units);
  if (blocks > kMostBlocks) return fail(AKV_EINVAL, "%s: batch too large", who);
  hipStream_t st = as_stream(stream);
  auto start = [&](auto e5) {
    with_shape(shape, vec, [&](auto lanes, auto iters, auto by_chunk) {
      hipLaunchKernelGGL((kv8_move_kernel<decltype(e5)::value != 0, decltype(lanes)::value, decltype(iters)::value,
                                          decltype(by_chunk)::value != 0>),
                         dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
    });
  };
  if (format == AKV_E5M2) start(Number<1>{});
  else start(Number<0>{});
  return check_launch(who);
}
