// New rows into a cache held in 8 bits, K (and q) rotated on the way (gfx950).
//
// K's row x at position p becomes, pair by pair, (x c - y s, y c + x s) with the p-th row
// (c, s) of the table, in fp32 from its load on; its codes and scales, and V's, are
// those of kv8_rows.h.  q's rows take the same turn and one rounding, in the same launch.
//
// A wave takes a block's tokens of one head (or of several, blocks being small), rows
// being the K heads, then the V heads; a run of tokens belongs to the wave whose
// window holds the run's first entry.  q rows go 64 / LANES heads to a wave (all of a
// token's heads in one wave, its table row read once: 142 us for 137 below, and never less).
//
// Bound by HBM from thousands of tokens on, by the launch below: 32768 tokens of 64 q heads and 8
// KV heads of 64, 647 MB in 136 us, 4.8 TB/s (a copy: 5.16); one token 4.5 us, 64 4.9.  Rotations
// of an odd number of eights, whose halves end inside a chunk, load and store quads instead
// (80 dims of which 40 turn: 284 us; element by element 1239; with all 80 turned 196).
#include "kv8_rows.h"

namespace akv {
namespace {

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
  bool slots64, pos64;
};

template <typename T, bool E5, int LANES, int ITERS, int MODE>
__global__ void __launch_bounds__(kThreads) kv8_append_kernel(const AppendArgs a) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rope& rope = a.rope;
  auto position = [&](int64_t t) -> int64_t {
    const int64_t p = load_index(a.positions, a.pos64, t);
    return p >= 0 && p < rope.rows ? p : -1;
  };
  // cos and sin of a lane's eight pairs
  auto coefficients = [&](int64_t p, int u, bool all, float (&c)[8], float (&s)[8]) KV8_INLINE {
    load8<MODE == kByQuad>(rope.table, rope.dtype, p * rope.stride + 8 * u, c, all ? 4 : 0);
    load8<MODE == kByQuad>(rope.table, rope.dtype, p * rope.stride + rope.dim / 2 + 8 * u, s, all ? 4 : 0);
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
    if constexpr (MODE == kByQuad) {
      x0.load_quads(from + place.at0, place.mid0);
      x1.load_quads(from + place.at1, place.mid1);
    } else {
      x0.load(from + place.at0);
      x1.load(from + place.at1);
    }
    float (&lo)[8] = *reinterpret_cast<float (*)[8]>(y), (&hi)[8] = *reinterpret_cast<float (*)[8]>(y + 8);
    x0.get(lo);
    x1.get(hi);
  };

  if (unit >= a.kv_units) {
    // q rows, 64 / LANES heads of a token
    const int64_t mine = unit - a.kv_units;
    if (mine >= a.q_units) return;
    const int64_t t = mine / a.q_parts;
    const int first = static_cast<int>(mine - t * a.q_parts);
    const int u = threadIdx.x % LANES, sub = (threadIdx.x & 63) / LANES;
    const Place place = place_of<MODE>(u, true, rope);
    const int64_t p = position(t);
    float c[8], s[8];
    if (place.turned && p >= 0) coefficients(p, u, place.all, c, s);
    const int head = first * (64 / LANES) + sub;
    if (head < a.q_heads && 16 * u < a.c.head_dim) {
      const T* from = static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh;
      T* to = static_cast<T*>(a.q_out) + t * a.qo_st + head * a.qo_sh;
      float y[16];
      if constexpr (MODE == kByElement) {
        // (q_out may be q: all of a row is read before any of it is written)
        by_element(from, u, true, p, y);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 16; ++e) to[16 * u + e] = static_cast<T>(p < 0 ? nan32() : y[e]);
      } else {
        part(from, place, y);
        if (place.turned && p >= 0) turn_place<MODE>(y, c, s, rope.neox, place.all);
        if (p < 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = nan32();
        }
        Chunk<T> x0, x1;
        x0.set(*reinterpret_cast<float (*)[8]>(y));
        x1.set(*reinterpret_cast<float (*)[8]>(y + 8));
        if constexpr (MODE == kByQuad) {
          x0.store_quads(to + place.at0, place.mid0);
          x1.store_quads(to + place.at1, place.mid1);
        } else {
          x0.store(to + place.at0);
          x1.store(to + place.at1);
        }
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
  const Place place = place_of<MODE>(at.u, rotates, rope);
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
    const Run run = run_at(slot_at, t, a.n_tokens, a.c.log2_block, t > 0 ? slot_at(t - 1) : -1);
    if (run.len) {
      const int64_t block = run.slot >> a.c.log2_block;
      const int first = static_cast<int>(run.slot - (block << a.c.log2_block));
      int64_t off[ITERS ? ITERS : 1];
#pragma unroll
      for (int it = 0; it < (ITERS ? ITERS : 1); ++it) off[it] = (first + it * at.rows + at.r) * slot_stride + place.at0;
      write_run<E5, LANES, ITERS, MODE, false>(
          at, in, run.len, first, pool + (block << a.c.log2_block) * slot_stride, slot_stride, off,
          place, scales + block * block_stride, [&](int, int i, float (&y)[16], float&) KV8_INLINE {
            const T* from = rows + (t + i) * row_stride;
            const int64_t p = rotates ? position(t + i) : 0;
            if constexpr (MODE == kByElement) {
              by_element(from, at.u, rotates, p, y);
            } else {
              part(from, place, y);
              if (place.turned && p >= 0) {
                float c[8], s[8];
                coefficients(p, at.u, place.all, c, s);
                turn_place<MODE>(y, c, s, rope.neox, place.all);
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

// The rounds of rows that a wave takes for a block, and its heads.
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

// Calls f with the kernel's LANES, ITERS and MODE as constants.
template <typename F>
void with_shape(const Shape& s, Mode mode, F f) {
  auto of_lanes = [&](auto lanes) {
    if (mode == kByElement) f(lanes, Number<0>{}, Number<kByElement>{});
    else if (mode == kByQuad && s.iters == 1) f(lanes, Number<1>{}, Number<kByQuad>{});
    else if (mode == kByQuad) f(lanes, Number<0>{}, Number<kByQuad>{});
    else if (s.iters == 1) f(lanes, Number<1>{}, Number<kByChunk>{});
    else if (s.iters == 2) f(lanes, Number<2>{}, Number<kByChunk>{});
    else f(lanes, Number<0>{}, Number<kByChunk>{});
  };
  if (s.lanes == 4) of_lanes(Number<4>{});
  else of_lanes(Number<8>{});
}

int64_t waves_to_blocks(int64_t waves) { return (waves + kWaves - 1) / kWaves; }

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
  rc = check_apart(who, a.c);
  if (rc) return rc;
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
  // whole chunks on 16-byte boundaries, pairs within a lane
  const int e = dtype == AKV_F32 ? 4 : 2, te = cos_sin_dtype == AKV_F32 ? 4 : 2;
  const bool vec =
      rotary_dim % 8 == 0 && aligned(k, 16) && aligned(v, 16) &&
          ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) * e) % 16 == 0 &&
          (!rotary_dim || (aligned(cos_sin, 16) && rope_stride * te % 16 == 0)) &&
          (!q_heads || (aligned(q, 16) && aligned(q_out, 16) &&
                        ((q_stride_t | q_stride_h | qo_stride_t | qo_stride_h) * e) % 16 == 0));
  const Mode mode = !vec ? kByElement : rotary_dim % 16 ? kByQuad : kByChunk;
  const Shape shape = shape_of(a.c);
  a.head_groups = shape.groups;
  // Entries of a wave: one where its waves are up to kFewWaves, so that no run waits
  // behind another; then more, since most waves find a run that began before them (us
  // by kFewWaves 1024, 4096, 16384, in blocks of 16: 32768 tokens of 8 heads 136, 137, 142 and
  // with one entry always 366; 2048 tokens 9.1, 10.7, 17.5; 512 tokens 4.8, 6.2, 7.5).
  constexpr int64_t kFewWaves = 1024;
  a.window = 1;
  while (a.window < scale_block && n_tokens * shape.groups > kFewWaves * a.window) a.window *= 2;
  a.kv_units = pool_slots ? (n_tokens + a.window - 1) / a.window * shape.groups : 0;
  const int rounds = (q_heads + 64 / shape.lanes - 1) / (64 / shape.lanes);
  a.q_parts = std::max(1, rounds);
  a.q_units = q_heads ? n_tokens * a.q_parts : 0;
  const int64_t blocks = waves_to_blocks(a.kv_units + a.q_units);
  if (blocks == 0) return AKV_OK;
  if (blocks > kMostBlocks) return fail(AKV_EINVAL, "%s: batch too large", who);
  hipStream_t st = as_stream(stream);
  auto start = [&](auto type, auto e5) {
    using T = decltype(type);
    with_shape(shape, mode, [&](auto lanes, auto iters, auto m) {
      hipLaunchKernelGGL((kv8_append_kernel<T, decltype(e5)::value != 0, decltype(lanes)::value, decltype(iters)::value,
                                            decltype(m)::value>),
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
