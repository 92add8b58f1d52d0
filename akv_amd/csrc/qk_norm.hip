// Per-head RMS norms of queries and keys, the position rotation, and the new
// K/V rows' way into the pool, in one pass (gfx950).
//
// For token t and a head's row x of D values
//   y = x / sqrt(mean(x^2) + eps) * w            (fp32, w the head norm's weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)     for the pairs of the first R dims
// with cos | sin the row positions[t] of the table, then one rounding to the
// storage type.  q goes to q_out, k to k_out and / or the pool row slot[t], v is
// copied to the pool.
//
// A stream of rows that is read and written once: bound by HBM.  Vector kernel:
// a row is D / 16 lanes of two 8-element chunks each, the chunks of a rotation
// pair in one lane, so the rotation needs no exchange and the mean two to five
// lane swaps; a wave takes the rows of one token, 64 / lanes at a time, and
// keeps that token's cos / sin and both weights in registers.  32768 tokens of 80
// rows of 64 in bf16: 680 MB in 135 us, 5.0 TB/s, what a large copy reaches; 8191 of
// 24 rows of 128: 103 MB in 22 us (28 from cold caches, where a copy takes 21); one
// token 3.8 us.  fp32: 32768 of 80 rows of 64 264 us, 5.1 TB/s.
#include <type_traits>

#include "row_chunks.h"

namespace akv {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeadDim = 512;

struct NormArgs {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* k_pool;
  void* v_pool;
  // element strides: token (slot for the pools), head
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh, kp_ss, kp_sh, vp_ss, vp_sh;
  const void* q_weight;
  const void* k_weight;
  const void* positions;
  const void* slots;
  const void* table;
  int64_t table_stride, table_rows, pool_slots, n_tokens;
  int32_t q_heads, kv_heads, head_dim, rotary_dim;
  int32_t weight_dtype, table_dtype;
  int32_t rows;   // rows of a token: q, k and, with a pool, v heads
  int32_t parts;  // waves per token
  float eps;
  bool neox, pos64, slots64;
};

// LANES per row: the power of two that holds D / 16 lanes.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(const NormArgs a) {
  constexpr int kRows = 64 / LANES;  // rows of a wave at a time
  const int lane = threadIdx.x & 63;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) +
                       __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = wave / a.parts;
  const int part = static_cast<int>(wave - t * a.parts);
  if (t >= a.n_tokens) return;
  const int u = lane % LANES, sub = lane / LANES;
  const bool in = 16 * u < a.head_dim;
  const bool turned = 16 * u < a.rotary_dim;
  // a neox pair's chunks lie R / 2 apart, every other lane's side by side
  const int at0 = a.neox && turned ? 8 * u : 16 * u;
  const int at1 = a.neox && turned ? 8 * u + a.rotary_dim / 2 : 16 * u + 8;
  const int64_t pos = load_index(a.positions, a.pos64, t);
  const int64_t slot = a.slots ? load_index(a.slots, a.slots64, t) : -1;
  const bool known = pos >= 0 && pos < a.table_rows;
  float c[8], s[8], wq[16], wk[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // without a table row there is no answer: NaN, not an unrotated row
    c[i] = s[i] = known ? 0.f : __builtin_nanf("");
    wq[i] = wq[8 + i] = wk[i] = wk[8 + i] = 1.f;
  }
  if (turned && known) {
    load8(a.table, a.table_dtype, pos * a.table_stride + 8 * u, c);
    load8(a.table, a.table_dtype, pos * a.table_stride + a.rotary_dim / 2 + 8 * u, s);
  }
  if (in && a.q_weight) {
    float x[8];
    load8(a.q_weight, a.weight_dtype, at0, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) wq[i] = x[i];
    load8(a.q_weight, a.weight_dtype, at1, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) wq[8 + i] = x[i];
  }
  if (in && a.k_weight) {
    float x[8];
    load8(a.k_weight, a.weight_dtype, at0, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) wk[i] = x[i];
    load8(a.k_weight, a.weight_dtype, at1, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) wk[8 + i] = x[i];
  }
  const float inv_d = 1.f / static_cast<float>(a.head_dim);
  const bool stored = slot >= 0 && slot < a.pool_slots;
  for (int row = part * kRows + sub; row - sub < a.rows; row += a.parts * kRows) {
    const bool live = in && row < a.rows;
    const bool is_q = row < a.q_heads, is_v = row >= a.q_heads + a.kv_heads;
    const int head = is_q ? row : is_v ? row - a.q_heads - a.kv_heads : row - a.q_heads;
    const T* from = is_q ? static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh
                    : is_v ? static_cast<const T*>(a.v) + t * a.v_st + head * a.v_sh
                           : static_cast<const T*>(a.k) + t * a.k_st + head * a.k_sh;
    Chunk<T> x0{}, x1{};
    if (live) {
      x0.load(from + at0);
      x1.load(from + at1);
    }
    if (live && is_v) {
      if (stored) {
        T* to = static_cast<T*>(a.v_pool) + slot * a.vp_ss + head * a.vp_sh;
        x0.store(to + at0);
        x1.store(to + at1);
      }
    }
    float y0[8], y1[8], sum = 0.f;
    x0.get(y0);
    x1.get(y1);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += y0[i] * y0[i] + y1[i] * y1[i];
    if (!live) sum = 0.f;
#pragma unroll
    for (int off = 1; off < LANES; off <<= 1) sum += __shfl_xor(sum, off);
    if (!live || is_v) continue;
    const float scale = 1.f / __builtin_sqrtf(sum * inv_d + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y0[i] = y0[i] * scale * (is_q ? wq[i] : wk[i]);
      y1[i] = y1[i] * scale * (is_q ? wq[8 + i] : wk[8 + i]);
    }
    if (turned) {
      if (a.neox) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = y0[i], r = y1[i];
          y0[i] = p * c[i] - r * s[i];
          y1[i] = r * c[i] + p * s[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = y0[2 * i], r0 = y0[2 * i + 1], p1 = y1[2 * i], r1 = y1[2 * i + 1];
          y0[2 * i] = p0 * c[i] - r0 * s[i];
          y0[2 * i + 1] = r0 * c[i] + p0 * s[i];
          y1[2 * i] = p1 * c[4 + i] - r1 * s[4 + i];
          y1[2 * i + 1] = r1 * c[4 + i] + p1 * s[4 + i];
        }
      }
    } else if (!known) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y0[i] = y1[i] = c[i];
    }
    x0.set(y0);
    x1.set(y1);
    if (is_q) {
      T* to = static_cast<T*>(a.q_out) + t * a.qo_st + head * a.qo_sh;
      x0.store(to + at0);
      x1.store(to + at1);
    } else {
      if (a.k_out) {
        T* to = static_cast<T*>(a.k_out) + t * a.ko_st + head * a.ko_sh;
        x0.store(to + at0);
        x1.store(to + at1);
      }
      if (stored && known) {
        T* to = static_cast<T*>(a.k_pool) + slot * a.kp_ss + head * a.kp_sh;
        x0.store(to + at0);
        x1.store(to + at1);
      }
    }
  }
}

// Any strides, alignment, head and rotary widths: one wave per row, an element
// per lane and step, the row's normalised values in LDS for the rotation.  Bound by
// its accesses of one element, the table's among them: 32768 tokens of 48 rows of 80
// with 40 rotated 921 us, 0.55 TB/s, where the vector kernel takes 115 with 80.
template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_generic_kernel(const NormArgs a) {
  __shared__ float row_of[kThreads / 64][kMaxHeadDim];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + wave;
  const int64_t t = unit / a.rows;
  const int row = static_cast<int>(unit - t * a.rows);
  const bool live = t < a.n_tokens;
  const bool is_q = row < a.q_heads, is_v = row >= a.q_heads + a.kv_heads;
  const int head = is_q ? row : is_v ? row - a.q_heads - a.kv_heads : row - a.q_heads;
  const int D = a.head_dim, R = a.rotary_dim;
  const T* from = nullptr;
  int64_t slot = -1, pos = -1;
  if (live) {
    from = is_q ? static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh
           : is_v ? static_cast<const T*>(a.v) + t * a.v_st + head * a.v_sh
                  : static_cast<const T*>(a.k) + t * a.k_st + head * a.k_sh;
    pos = load_index(a.positions, a.pos64, t);
    if (a.slots) slot = load_index(a.slots, a.slots64, t);
  }
  const bool stored = slot >= 0 && slot < a.pool_slots;
  const bool known = pos >= 0 && pos < a.table_rows;
  float* y = row_of[wave];
  float sum = 0.f;
  if (live) {
    for (int i = lane; i < D; i += 64) {
      if (is_v) {
        if (stored) static_cast<T*>(a.v_pool)[slot * a.vp_ss + head * a.vp_sh + i] = from[i];
        continue;
      }
      const float x = to_f32(from[i]);
      y[i] = x;
      sum += x * x;
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
  const float scale = 1.f / __builtin_sqrtf(sum * (1.f / static_cast<float>(D)) + a.eps);
  const void* weight = is_q ? a.q_weight : a.k_weight;
  if (live && !is_v)
    for (int i = lane; i < D; i += 64) y[i] = y[i] * scale * (weight ? load1(weight, a.weight_dtype, i) : 1.f);
  __syncthreads();
  if (!live || is_v) return;
  for (int i = lane; i < D; i += 64) {
    float r = known ? y[i] : __builtin_nanf("");
    if (i < R && known) {
      const int half = R / 2;
      const int pair = a.neox ? (i < half ? i : i - half) : i / 2;
      const bool second = a.neox ? i >= half : (i & 1) != 0;
      const int other = a.neox ? (second ? i - half : i + half) : i ^ 1;
      const float c = load1(a.table, a.table_dtype, pos * a.table_stride + pair);
      const float s = load1(a.table, a.table_dtype, pos * a.table_stride + half + pair);
      r = second ? y[i] * c + y[other] * s : y[i] * c - y[other] * s;
    }
    const T v = static_cast<T>(r);
    if (is_q) {
      static_cast<T*>(a.q_out)[t * a.qo_st + head * a.qo_sh + i] = v;
    } else {
      if (a.k_out) static_cast<T*>(a.k_out)[t * a.ko_st + head * a.ko_sh + i] = v;
      if (stored && known) static_cast<T*>(a.k_pool)[slot * a.kp_ss + head * a.kp_sh + i] = v;
    }
  }
}

// Workgroups of a launch: a grid has fewer than 2^32 threads.  More tokens take
// several launches.
constexpr int64_t kMostBlocks = 1 << 23;

// Calls start(args, blocks) for stretches of the tokens, each with `waves` waves.
template <typename T, typename F>
int in_stretches(const NormArgs& args, int64_t waves, F start) {
  const int64_t most = kMostBlocks * (kThreads / 64) / waves;
  for (int64_t t = 0; t < args.n_tokens; t += most) {
    NormArgs a = args;
    a.n_tokens = args.n_tokens - t < most ? args.n_tokens - t : most;
    auto on = [&](auto*& p, int64_t bytes) {
      if (p) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(p) + t * bytes);
    };
    constexpr int64_t e = sizeof(T);
    on(a.q, e * a.q_st), on(a.k, e * a.k_st), on(a.v, e * a.v_st), on(a.q_out, e * a.qo_st), on(a.k_out, e * a.ko_st);
    on(a.positions, a.pos64 ? 8 : 4), on(a.slots, a.slots64 ? 8 : 4);
    start(a, dim3(static_cast<unsigned>((a.n_tokens * waves + kThreads / 64 - 1) / (kThreads / 64))));
    const int rc = check_launch("akv_qk_norm_rope");
    if (rc) return rc;
  }
  return AKV_OK;
}

template <typename T>
int launch_vector(const NormArgs& args, hipStream_t st) {
  NormArgs a = args;
  int lanes = 1;
  while (16 * lanes < a.head_dim) lanes *= 2;
  const int at_once = 64 / lanes;
  const int rounds = (a.rows + at_once - 1) / at_once;
  // a token's rows go to one wave (its cos / sin and the weights are loaded
  // once) unless there are too few tokens to fill the chip with waves (us with one
  // wave and with one per round, 64 + 16 heads of 64: 1024 tokens 8.9, 7.2; 2048
  // 11.5, 12.9; 16384 72.8, 85.6; 32 + 16 heads of 128: 1024 9.5, 8.8; 2048 12.5, 14.8)
  a.parts = a.n_tokens >= 2048 ? 1 : rounds;
  return in_stretches<T>(a, a.parts, [&](const NormArgs& part, dim3 grid) {
    const dim3 block(kThreads);
    switch (lanes) {
      case 1: hipLaunchKernelGGL((qk_norm_kernel<T, 1>), grid, block, 0, st, part); break;
      case 2: hipLaunchKernelGGL((qk_norm_kernel<T, 2>), grid, block, 0, st, part); break;
      case 4: hipLaunchKernelGGL((qk_norm_kernel<T, 4>), grid, block, 0, st, part); break;
      case 8: hipLaunchKernelGGL((qk_norm_kernel<T, 8>), grid, block, 0, st, part); break;
      case 16: hipLaunchKernelGGL((qk_norm_kernel<T, 16>), grid, block, 0, st, part); break;
      default: hipLaunchKernelGGL((qk_norm_kernel<T, 32>), grid, block, 0, st, part); break;
    }
  });
}

template <typename T>
int launch(const NormArgs& a, bool vector, hipStream_t st) {
  if (vector) return launch_vector<T>(a, st);
  return in_stretches<T>(a, a.rows, [&](const NormArgs& part, dim3 grid) {
    hipLaunchKernelGGL(qk_norm_generic_kernel<T>, grid, dim3(kThreads), 0, st, part);
  });
}

}  // namespace
}  // namespace akv

extern "C" int akv_qk_norm_rope(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                int64_t v_stride_h, int32_t dtype, int64_t n_tokens, int32_t q_heads,
                                int32_t kv_heads, int32_t head_dim, int32_t rotary_dim, int32_t is_neox,
                                const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps,
                                const void* positions, int32_t positions_dtype, const void* cos_sin,
                                int32_t cos_sin_dtype, int64_t rope_stride, int64_t rope_rows, void* q_out,
                                int64_t qo_stride_t, int64_t qo_stride_h, void* k_out, int64_t ko_stride_t,
                                int64_t ko_stride_h, const void* slots, int32_t slots_dtype, void* k_pool,
                                void* v_pool, int64_t pool_slots, int64_t kp_stride_slot, int64_t kp_stride_head,
                                int64_t vp_stride_slot, int64_t vp_stride_head, void* stream) {
  using namespace akv;
  auto valid = [](int32_t d) { return d == AKV_F32 || d == AKV_F16 || d == AKV_BF16; };
  if (!valid(dtype) || !valid(weight_dtype) || !valid(cos_sin_dtype))
    return fail(AKV_EINVAL, "akv_qk_norm_rope: dtypes must be float32, float16 or bfloat16");
  if (!valid_index_dtype(positions_dtype) || !valid_index_dtype(slots_dtype))
    return fail(AKV_EINVAL, "akv_qk_norm_rope: index vectors must be int32 or int64");
  if (n_tokens < 0 || q_heads < 0 || kv_heads < 0 || pool_slots < 0 || rope_rows < 0)
    return fail(AKV_EINVAL, "akv_qk_norm_rope: negative size");
  if (head_dim < 1 || head_dim > kMaxHeadDim)
    return fail(AKV_EINVAL, "akv_qk_norm_rope: head_dim %d (1 to %d)", head_dim, kMaxHeadDim);
  if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(AKV_EINVAL, "akv_qk_norm_rope: rotary_dim %d of %d", rotary_dim, head_dim);
  if (!(eps >= 0.f) || eps > 3.4e38f) return fail(AKV_EINVAL, "akv_qk_norm_rope: eps must be finite and not negative");
  if (static_cast<int64_t>(q_heads) + 2 * static_cast<int64_t>(kv_heads) > 65535)
    return fail(AKV_EINVAL, "akv_qk_norm_rope: %d q and %d KV heads", q_heads, kv_heads);
  if (n_tokens == 0 || q_heads + kv_heads == 0) return AKV_OK;
  // (a pool without slots need not have an address: it takes no row)
  const bool pool = k_pool || v_pool || (slots && pool_slots == 0);
  if ((q_heads && (!q || !q_out)) || (kv_heads && !k) || !positions || !cos_sin)
    return fail(AKV_EINVAL, "akv_qk_norm_rope: null device pointer");
  if (pool && ((pool_slots > 0 && (!k_pool || !v_pool)) || (kv_heads && !v) || !slots))
    return fail(AKV_EINVAL, "akv_qk_norm_rope: the pool needs K, V and slots");
  if (kv_heads && !pool && !k_out) return fail(AKV_EINVAL, "akv_qk_norm_rope: the keys have nowhere to go");
  NormArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.k_out = k_out;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.qo_st = qo_stride_t;
  a.qo_sh = qo_stride_h;
  a.ko_st = ko_stride_t;
  a.ko_sh = ko_stride_h;
  a.kp_ss = kp_stride_slot;
  a.kp_sh = kp_stride_head;
  a.vp_ss = vp_stride_slot;
  a.vp_sh = vp_stride_head;
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.positions = positions;
  a.slots = pool ? slots : nullptr;
  a.table = cos_sin;
  a.table_stride = rope_stride;
  a.table_rows = rope_rows;
  a.pool_slots = pool ? pool_slots : 0;
  a.n_tokens = n_tokens;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.rotary_dim = rotary_dim;
  a.weight_dtype = weight_dtype;
  a.table_dtype = cos_sin_dtype;
  a.rows = q_heads + kv_heads * (pool ? 2 : 1);
  a.eps = eps;
  a.neox = is_neox != 0;
  a.pos64 = positions_dtype == AKV_I64;
  a.slots64 = slots_dtype == AKV_I64;
  // the vector kernel: whole lanes of 16 elements in both the rotated part and
  // the row, and 16-byte aligned chunks of 8 everywhere
  const int esize = dtype == AKV_F32 ? 4 : 2;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  auto strided = [&](int64_t x, int64_t y) { return ((x | y) * esize) % 16 == 0; };
  const int tsize = cos_sin_dtype == AKV_F32 ? 4 : 2;
  const bool vector = head_dim % 16 == 0 && rotary_dim % 16 == 0 && aligned(q) && aligned(k) && aligned(v) &&
                      aligned(q_out) && aligned(k_out) && aligned(k_pool) && aligned(v_pool) && aligned(q_weight) &&
                      aligned(k_weight) && aligned(cos_sin) && (rope_stride * tsize) % 16 == 0 &&
                      (!q_heads || (strided(q_stride_t, q_stride_h) && strided(qo_stride_t, qo_stride_h))) &&
                      (!kv_heads || strided(k_stride_t, k_stride_h)) &&
                      (!k_out || strided(ko_stride_t, ko_stride_h)) &&
                      (!pool || (strided(v_stride_t, v_stride_h) && strided(kp_stride_slot, kp_stride_head) &&
                                 strided(vp_stride_slot, vp_stride_head)));
  hipStream_t st = as_stream(stream);
  if (dtype == AKV_F32) return launch<float>(a, vector, st);
  if (dtype == AKV_F16) return launch<_Float16>(a, vector, st);
  return launch<__bf16>(a, vector, st);
}
