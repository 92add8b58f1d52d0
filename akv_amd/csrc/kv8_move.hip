// Kept rows of a cache held in 8 bits to fresh slots and new positions, all layers (gfx950).
#include "kv8_rows.h"

namespace akv {
namespace {

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
  int64_t pair_stride, n_tokens, windows;
  int32_t window, n_layers, layers;  // entries and layers of a workgroup
  int32_t heads_at_once;             // of a wave, for a block's rows
  bool skip_zero;
};

// Layers of a workgroup, whose list entries and factors it gets once (us with 2, 4, 6, 9
// and 12: 19.9k tokens of 36 layers, 8 heads of 64, 425, 382, 381, 382, 386; 16.4k of 32 layers, 8
// heads of 128 in blocks of 16, 656, 499, 483, 484, 487), fewer where the workgroups are
// fewer than kFullChip (2.4k tokens of 2 layers, 2 heads of 64: 8.2, with both layers 9.3).
constexpr int kMostLayers = 6;  // (at most 64: a lane holds the addresses of one)
constexpr int64_t kFullChip = 2048;
constexpr int kMostWindow = 64;  // entries
constexpr int kMostListed = kMostWindow + kMostBlock;

// What becomes of an entry's row.
enum Fate : int32_t { kTurned, kAtItsPlace, kUnknown, kLeft };

// A workgroup takes a window of the list's entries in a few layers, all heads.  The
// entries come to LDS once, the rotations' factors (a pair each, by the difference of two
// positions, the same for every layer and head) once a run; then a wave takes K or V of
// 64 / LANES rows at a time: of one block of a head (ITERS rounds of its rows, several
// heads where they leave lanes), or, with blocks of one slot (SINGLE), of any tokens and
// heads.  The next rows are on their way while one lot is turned and stored.  Windows are
// numbered fastest, so that the device works through few layers at a time.
//
// Bound by HBM: 19.9k scattered tokens of 36 layers, 8 heads of 64: 1.57 GB in 381 us, 4.1
// TB/s; 16.4k of 32 layers, 8 heads of 128, in blocks and pages of 16: 2.17 GB in 483 us, 4.5 TB/s
// (a copy: 5.16).  In blocks of 32 and 64, a wave's rounds held as codes and decoded three times,
// 649 and 659-739 us (with the values kept in registers, a wave a SIMD, 1530 and 973; 52 to 71 registers
// of the eight rounds' are spilled): one wave has all of a block and head.  Blocks of 2, 4 and 8: 740,
// 600, 546, since a workgroup has one block, of which few rows fill its waves, behind the whole chain of
// loads; where that chain is all, 16.4k tokens of a layer's 2 heads of 64, 49, 28 and 17 us, blocks of 1 9.8.
// The arithmetic hides behind it (without any of it 441 and 532 us in an
// earlier order).  What is missing in the first are the scales: 32 bytes a token and
// layer, alone in their lines; with none of them stored a raw copy of these rows takes 307 us,
// with them 460.
template <bool E5, int LANES, int ITERS, bool SINGLE, int MODE>
__global__ void __launch_bounds__(kThreads, SINGLE ? 1 : ITERS <= 2 ? 3 : 2) kv8_move_kernel(const MoveArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int kRows = 64 / LANES;
  __shared__ int32_t s_dst[1 + kMostListed], s_src[kMostListed], s_old[kMostListed], s_new[kMostListed];
  __shared__ int32_t s_fate[kMostWindow];
  extern __shared__ __attribute__((aligned(16))) float s_factor[];  // cosines, then sines, of window x half pairs
  if (gated(a.gate)) return;
  const Rope& rope = a.rope;
  const int layer_group = static_cast<int>(blockIdx.x / a.windows);
  const int64_t t0 = (blockIdx.x - layer_group * a.windows) * a.window;
  const int layer0 = layer_group * a.layers, layers = std::min(a.n_layers - layer0, a.layers);
  const int listed = static_cast<int>(std::min<int64_t>(a.n_tokens - t0, SINGLE ? a.window : a.window + (1 << a.c.log2_block)));
  if (listed <= 0) return;
  auto usable = [&](int64_t s) { return s >= (a.skip_zero ? 1 : 0) && s < a.c.slots; };
  for (int i = threadIdx.x; i < listed + 1; i += kThreads) {
    const int64_t t = t0 + i - 1;
    const int32_t s = t >= 0 ? a.dst[t] : -1;
    s_dst[i] = usable(s) ? s : -1;
    if (i == 0) continue;
    s_src[i - 1] = a.src[t];
    s_old[i - 1] = a.pairs[t * a.pair_stride];
    s_new[i - 1] = a.pairs[t * a.pair_stride + 1];
  }
  const int half = rope.dim / 2, heads = a.c.heads, most_factors = a.window * half;
  const Stand<LANES> at(SINGLE ? 0 : a.c.log2_block);
  const bool in_row = 16 * at.u < a.c.head_dim;
  // lane l: the addresses of the workgroup's l-th layer
  const int mine_at = layer0 + std::min(lane, layers - 1);
  const uint64_t my_k = a.k_ptrs[mine_at], my_v = a.v_ptrs[mine_at];
  const uint64_t my_ks = a.k_scale_ptrs[mine_at], my_vs = a.v_scale_ptrs[mine_at];
  __syncthreads();

  const int window = static_cast<int>(std::min<int64_t>(a.window, a.n_tokens - t0));
  for (int e0 = 0; e0 < window;) {
    // the run from entry e0 on: its rows, and their first slot
    int len = window, first = 0;
    int64_t block = 0;
    if constexpr (!SINGLE) {
      const Run run = run_at([&](int64_t i) -> int64_t { return s_dst[1 + i]; }, e0, listed, a.c.log2_block, s_dst[e0]);
      if (run.len == 0) {
        e0 += run.skip;
        continue;
      }
      len = run.len;
      block = run.slot >> a.c.log2_block;
      first = static_cast<int>(run.slot - (block << a.c.log2_block));
    }
    // its rows' fates and factors
    bool plain = first == 0, at_place = false;
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const int64_t p = s_old[e0 + i], n = s_new[e0 + i];
      const bool known = p >= 0 && p < rope.rows && n >= 0 && n < rope.rows;
      const int fate = !usable(s_src[e0 + i]) ? kLeft : p == n ? kAtItsPlace : known ? kTurned : kUnknown;
      s_fate[i] = fate;
      plain &= (fate == kTurned || fate == kAtItsPlace) && (!SINGLE || s_dst[1 + e0 + i] >= 0);
      at_place |= fate == kAtItsPlace;
    }
    for (int i = threadIdx.x; i < len * half; i += kThreads) {
      const int row = i / half, pair = i - row * half;
      const int64_t p = s_old[e0 + row], n = s_new[e0 + row];
      if (p == n || p < 0 || p >= rope.rows || n < 0 || n >= rope.rows) continue;
      auto entry = [&](int64_t q, int j) { return load1(rope.table, rope.dtype, q * rope.stride + j); };
      const float co = entry(p, pair), so = entry(p, half + pair), cn = entry(n, pair), sn = entry(n, half + pair);
      const float norm = co * co + so * so;
      s_factor[i] = (cn * co + sn * so) / norm;
      s_factor[most_factors + i] = (sn * co - cn * so) / norm;
    }
    const bool some_at_place = __syncthreads_or(at_place);
    const bool fast = __syncthreads_and(MODE != kByElement && plain);

    // lots of rows: K's, then V's; a wave takes every fourth
    const int lots = SINGLE ? (len * heads + kRows - 1) / kRows : (heads + a.heads_at_once - 1) / a.heads_at_once;
    const int mine = (2 * lots - wave + kWaves - 1) / kWaves;  // of a layer
    auto any_run = [&]() KV8_INLINE {
      for (int l = 0; l < layers; ++l) {
        for (int n = wave; n < 2 * lots; n += kWaves) {
          const bool is_v = n >= lots;
          const int lot = is_v ? n - lots : n;
          int entry0 = 0, head = lot * a.heads_at_once + at.sub;  // the lane's row of round 0
          bool in = in_row && at.sub < a.heads_at_once && head < heads;
          int64_t to_block = block;
          if constexpr (SINGLE) {
            const int row = lot * kRows + lane / LANES;
            entry0 = row / heads;
            head = row - entry0 * heads;
            in = in_row && entry0 < len;
            to_block = in ? s_dst[1 + e0 + entry0] : -1;
          }
          const Place place = place_of<MODE>(at.u, !is_v, rope);
          const int64_t slot_stride = is_v ? a.c.v_ss : a.c.k_ss, head_at = head * (is_v ? a.c.v_sh : a.c.k_sh);
          const int64_t scale_stride = is_v ? a.c.vs_sb : a.c.ks_sb, scale_at = head * (is_v ? a.c.vs_sh : a.c.ks_sh);
          uint8_t* codes = reinterpret_cast<uint8_t*>(lane_value(is_v ? my_v : my_k, l)) + head_at;
          float* scales = reinterpret_cast<float*>(lane_value(is_v ? my_vs : my_ks, l)) + scale_at;
          const int64_t off = (first + at.r) * slot_stride + place.at0;
          write_run<E5, LANES, 0, MODE, true>(
              at, in && to_block >= 0, SINGLE ? 1 : len, first, codes + (to_block << a.c.log2_block) * slot_stride,
              slot_stride, &off, place, scales + to_block * scale_stride,
              [&](int, int i, float (&z)[16], float& by) KV8_INLINE {
                const int entry = entry0 + i, fate = s_fate[entry];
                if (fate == kLeft) return false;
                const int64_t src = s_src[e0 + entry];
                const uint8_t* from = codes + src * slot_stride;
                by = load_scale(scales + (src >> a.c.log2_block) * scale_stride);
                decode8<E5>(load_chunk<MODE>(from + place.at0, place.mid0), z);
                decode8<E5>(load_chunk<MODE>(from + place.at1, place.mid1), z + 8);
                if (is_v || fate == kAtItsPlace) return true;
                const float* f = s_factor + entry * half;
                if (fate == kUnknown) {
#pragma unroll
                  for (int e = 0; e < 16; ++e) z[e] = nan32();
                } else if constexpr (MODE != kByElement) {
                  if (place.turned) {
                    float c[8], s[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                      const int pair = 8 * at.u + (MODE == kByChunk || i < 4 || place.all ? i : 0);
                      c[i] = f[pair], s[i] = f[most_factors + pair];
                    }
                    turn_place<MODE>(z, c, s, rope.neox, place.all);
                  }
                } else {
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    __builtin_amdgcn_sched_barrier(0);  // (few elements in flight: registers)
                    const int d = 16 * at.u + e;
                    if (d >= rope.dim) continue;
                    const Pair pair = pair_of(d, rope);
                    const float c = f[pair.number], s = f[most_factors + pair.number];
                    const uint32_t code = *((const global_byte*)from + pair.other);
                    const float o = E5 ? __builtin_amdgcn_cvt_f32_bf8(code, 0) : __builtin_amdgcn_cvt_f32_fp8(code, 0);
                    z[e] = pair.second ? z[e] * c + o * s : z[e] * c - o * s;
                  }
                }
                return true;
              });
        }
      }
    };
    bool done = false;
    if constexpr (MODE != kByElement) {
      const int total = mine * layers;
      if (fast && total > 0) {
        done = true;
      // every row goes its way: no branch with loads or stores, lanes past the heads, dims
      // and rows do their neighbours' work again, so that waits for loads count the stores
      // behind them and do not wait for those
      const int u = std::min(at.u, a.c.head_dim / 16 - 1);
      struct Ahead {
        u32x2 lo[ITERS], hi[ITERS];
        float scale[ITERS];
        uint8_t* to[ITERS];
        float* to_scale;
        int entry[ITERS];
        Place place;
        bool is_v;
      };
      int l = 0, n = wave;  // the next lot's
      auto fetch = [&](Ahead& x) KV8_INLINE {
        const bool is_v = n >= lots;
        const int lot = is_v ? n - lots : n;
        uint8_t* codes = reinterpret_cast<uint8_t*>(lane_value(is_v ? my_v : my_k, l));
        float* scales = reinterpret_cast<float*>(lane_value(is_v ? my_vs : my_ks, l));
        const int64_t slot_stride = is_v ? a.c.v_ss : a.c.k_ss, head_stride = is_v ? a.c.v_sh : a.c.k_sh;
        const int64_t scale_stride = is_v ? a.c.vs_sb : a.c.ks_sb, scale_head = is_v ? a.c.vs_sh : a.c.ks_sh;
        const Place place = place_of<MODE>(u, !is_v, rope);
        x.is_v = is_v;
        x.place = place;
        const int apart = place.at1 - place.at0;
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
          int entry, head;
          if constexpr (SINGLE) {
            const int row = std::min(lot * kRows + lane / LANES, len * heads - 1);
            entry = row / heads;
            head = row - entry * heads;
          } else {
            entry = std::min(it * at.rows + at.r, len - 1);
            head = std::min(lot * a.heads_at_once + std::min(at.sub, a.heads_at_once - 1), heads - 1);
          }
          const int64_t src = s_src[e0 + entry];
          const int64_t to_block = SINGLE ? s_dst[1 + e0 + entry] : block;
          const int64_t in_row = head * head_stride + place.at0;
          x.entry[it] = entry;
          x.scale[it] = load_scale(scales + (src >> a.c.log2_block) * scale_stride + head * scale_head);
          x.lo[it] = load_chunk<MODE>(codes + src * slot_stride + in_row, place.mid0);
          x.hi[it] = load_chunk<MODE>(codes + src * slot_stride + in_row + apart, place.mid1);
          x.to[it] = codes + ((to_block << a.c.log2_block) + (SINGLE ? 0 : entry)) * slot_stride + in_row;
          x.to_scale = scales + to_block * scale_stride + head * scale_head;
        }
        // (behind the last lot it is done again)
        if (n + kWaves < 2 * lots) {
          n += kWaves;
        } else if (l + 1 < layers) {
          n = wave;
          ++l;
        }
      };
      auto put = [&](Ahead& x) KV8_INLINE {
        constexpr int kHeld = ITERS <= 2 ? ITERS : 1;  // rounds whose values are held; of more the codes, taken twice
        if constexpr (kHeld < ITERS) fetch(x);
        float z[kHeld][16], unit_of[ITERS], top = 0.f;
        uint8_t* to[ITERS];
        float* to_scale = x.to_scale;
        const Place place = x.place;
        const int apart = place.at1 - place.at0;
        const bool turns = !x.is_v && 16 * u < rope.dim;
        int entry[ITERS];
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
          unit_of[it] = x.scale[it];
          to[it] = x.to[it];
          entry[it] = x.entry[it];
        }
        auto decode = [&](int it, float (&y)[16]) KV8_INLINE {
          if constexpr (kHeld < ITERS) {
            // (as if unknown: the values of a round are not kept from the first time)
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" : "+v"(x.lo[it]), "+v"(x.hi[it]));
          }
          decode8<E5>(x.lo[it], y);
          decode8<E5>(x.hi[it], y + 8);
        };
        auto turn_row = [&](int it, float (&y)[16]) KV8_INLINE {
          if (!turns || (some_at_place && s_fate[entry[it]] == kAtItsPlace)) return;
          float c[8], s[8];
          const float* f = s_factor + entry[it] * half + 8 * u;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int pair = MODE == kByChunk || i < 4 || place.all ? i : 0;
            c[i] = f[pair], s[i] = f[most_factors + pair];
          }
          turn_place<MODE>(y, c, s, rope.neox, place.all);
        };
        if constexpr (kHeld == ITERS) {
#pragma unroll
          for (int it = 0; it < ITERS; ++it) decode(it, z[it]);
          fetch(x);
#pragma unroll
          for (int it = 0; it < ITERS; ++it) turn_row(it, z[it]);
        }
        auto settle = [&](bool finite_only) KV8_INLINE {
          top = 0.f;
#pragma unroll
          for (int it = 0; it < ITERS; ++it) {
            if constexpr (kHeld < ITERS) {
              decode(it, z[0]);
              turn_row(it, z[0]);
            }
            top = __builtin_fmaxf(top, largest_of(z[it % kHeld], unit_of[it], finite_only));
          }
          top = group_max<LANES>(top, at.span);
        };
        settle(false);
        if (__builtin_amdgcn_ballot_w64(!(top < INFINITY))) settle(true);
        const float scale = fitting<E5>(top);
        const float inverse = __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, scale));
#pragma unroll
        for (int it = 0; it < ITERS; ++it) {
          if constexpr (kHeld < ITERS) {
            decode(it, z[0]);
            turn_row(it, z[0]);
          }
          float (&y)[16] = z[it % kHeld];
          float f = inverse * unit_of[it];
          f = f == INFINITY && unit_of[it] < INFINITY ? 0x1.fffffep127f : f;  // (a row of zeros)
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] *= f;
          const u32x2 lo = encode8<E5>(y), hi = encode8<E5>(y + 8);
          if constexpr (SINGLE) {
            // past the caches: scattered rows' scales, 4 bytes a head, lie in lines that other
            // tokens' are read from and written to (380 us for 404; blocks of 16: 537 for 528)
            if constexpr (MODE == kByQuad) {
              const uint32_t words[4] = {lo[0], lo[1], hi[0], hi[1]};
              const int ats[4] = {0, place.mid0, apart, apart + place.mid1};
#pragma unroll
              for (int i = 0; i < 4; ++i) __builtin_nontemporal_store(words[i], (global_any_u32*)(to[it] + ats[i]));
            } else {
              __builtin_nontemporal_store(lo, (global_any_u32x2*)to[it]);
              __builtin_nontemporal_store(hi, (global_any_u32x2*)(to[it] + apart));
            }
          } else {
            store_chunk<MODE>(to[it], place.mid0, lo);
            store_chunk<MODE>(to[it] + apart, place.mid1, hi);
          }
        }
        store_scale(to_scale, scale);
      };
      Ahead x;
      if constexpr (ITERS <= 2) fetch(x);
      put(x);  // (by itself: behind it the loads are always followed by stores)
#pragma nounroll
      for (int q = 1; q < total; ++q) put(x);
      }
    }
    if (!done) any_run();
    e0 += len;
    __syncthreads();  // (the next run's factors take these' place)
  }
}

}  // namespace
}  // namespace akv

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
  rc = check_apart(who, a.c);
  if (rc) return rc;
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
  // (codes and the table at any address: the one's accesses need no alignment, the other
  // is read element by element.  4096 tokens of 8 layers, 8 heads of 64: 21 us, in blocks of 16 30;
  // element by element 51 and 87)
  const bool vec = rotary_dim % 8 == 0;
  const int lanes = lanes_of(head_dim), rows = std::min(scale_block, 64 / lanes), rounds = scale_block / rows;
  const bool single = scale_block == 1;
  a.heads_at_once = std::min(64 / (lanes * rows), n_heads);
  // entries of a workgroup: rows for its four waves
  a.window = single ? std::max(1, std::min(kMostWindow, kThreads / (lanes * n_heads))) : scale_block;
  a.windows = (n_tokens + a.window - 1) / a.window;
  a.layers = std::min(n_layers, kMostLayers);
  while (a.layers > 1 && a.windows * ((n_layers + a.layers - 1) / a.layers) < kFullChip) --a.layers;
  const int64_t blocks = a.windows * ((n_layers + a.layers - 1) / a.layers);
  if (blocks > kMostBlocks) return fail(AKV_EINVAL, "%s: batch too large", who);
  hipStream_t st = as_stream(stream);
  const dim3 threads(kThreads), grid(static_cast<unsigned>(blocks));
  const unsigned lds = static_cast<unsigned>(a.window) * rotary_dim * sizeof(float);
  auto start = [&](auto e5, auto n, auto mode) {
    constexpr bool kE5 = decltype(e5)::value != 0;
    constexpr int kLanes = decltype(n)::value, kMode = decltype(mode)::value;
    if (single) hipLaunchKernelGGL((kv8_move_kernel<kE5, kLanes, 1, true, kMode>), grid, threads, lds, st, a);
    else if (rounds == 1 || kMode == kByElement) hipLaunchKernelGGL((kv8_move_kernel<kE5, kLanes, 1, false, kMode>), grid, threads, lds, st, a);
    else if constexpr (kMode == kByElement) return;
    else if (rounds == 2) hipLaunchKernelGGL((kv8_move_kernel<kE5, kLanes, 2, false, kMode>), grid, threads, lds, st, a);
    else if (rounds == 4) hipLaunchKernelGGL((kv8_move_kernel<kE5, kLanes, 4, false, kMode>), grid, threads, lds, st, a);
    else if constexpr (kLanes == 8)
      hipLaunchKernelGGL((kv8_move_kernel<kE5, 8, 8, false, kMode>), grid, threads, lds, st, a);
  };
  auto by_lanes = [&](auto e5, auto mode) {
    if (lanes == 4) start(e5, Number<4>{}, mode);
    else start(e5, Number<8>{}, mode);
  };
  auto by_form = [&](auto e5) {
    if (!vec) by_lanes(e5, Number<kByElement>{});
    else if (rotary_dim % 16) by_lanes(e5, Number<kByQuad>{});
    else by_lanes(e5, Number<kByChunk>{});
  };
  if (format == AKV_E5M2) by_form(Number<1>{});
  else by_form(Number<0>{});
  return check_launch(who);
}
