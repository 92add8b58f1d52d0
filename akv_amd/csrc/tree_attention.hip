// Attention of drafted tokens over a cache (gfx950, MFMA): the step that
// verifies a tree of tokens per request.
//
// Request b has n = qo_indptr[b + 1] - qo_indptr[b] drafted tokens and
// L = kv_indptr[b + 1] - kv_indptr[b] keys, whose last n are the drafted
// tokens' own (their K/V rows are in the pool already).  Key j of token i is
// visible when
//   j < L - n:   j >= key_starts[i]      (a sliding window's first key; or all)
//   otherwise:   bit j - (L - n) of token i's mask  (or j - (L - n) <= i: a chain)
// and o_ih = sum_j e^s_j v_j / (sum_j e^s_j + e^sink_h), s_j = scale q_ih . k_j
// over the visible keys; a row that sees none is 0.  A key whose slot lies
// outside the pool is a hole that no token sees.
//
// The n tokens x G heads of a KV head's group are the rows of one product with
// that head's keys, so K and V are read once for a block of 64 SUB rows, and
// again for every further one.  All the batch's tiles of keys lie on a line (a
// request's blocks of rows far apart), and 512 workgroups of four waves, two per
// CU, take equal stretches of it; where a cut falls among a request's tiles, a
// second launch merges the parts.  Tiles of
// K and V stream into LDS (two places) while the one before is worked on, 32 keys
// (a quarter of a tile at D = 64) at a time, 16 SUB rows per wave:
//   S^T[32 x 16 SUB] = K . Q^T              v_mfma_f32_16x16x32
//   P^T = 2^(scale log2(e) S^T - m)         rounded once to the storage type
//   l += 1^T . P^T,  O^T[D x 16 SUB] += V^T . P^T
// (the matrix cores take P in V's type; the sum takes the rounded weights too, so
// that they add up to one.  A row's error against 64 bits is 0.0023 of it in bf16
// and 0.00027 in fp16; the output's own rounding alone is 0.0017 and 0.00021).
// A block with at most half (a quarter of) its rows has two (four) waves share
// each group of rows: they take the quarters in turn and meet at the end.
// P^T leaves the first product in the operand layout of the second; V^T comes
// through ds_read_b64_tr_b16.  m is a row's first maximum and moves only when the
// weights outgrow their types.
//
// Bound: HBM while a KV head has up to about 128 rows (16 tokens x 8 heads of 64
// over 32 requests of 20k keys: 1.30 GB in 272-306 us, 4.3-4.8 TB/s; 5 to 32 tokens x
// 4 heads of 128 over 12 paged requests: 0.50 GB in 124 us, 4.0 TB/s); matrix and
// vector work above (64 tokens over 8 requests of 25k: 203 GFLOP in 255-284 us,
// 720-800 TFLOP/s); round trips where there is little (8 tokens over 4096 keys: 13
// us and 5 for the merge; a window's 145 keys x 32 requests: 16-17 us).  Every
// instance moves 120 to 198 scalars to vector lanes, SUB = 4 takes all 256 vector
// registers and keeps one in scratch.
//
// Lane layouts (verified on gfx950): v_mfma_f32_16x16x32 -- lane l supplies
// A[l%16][k(l,i)], B[k(l,i)][l%16] for i < 8 and holds D[4(l/16)+i][l%16];
// ds_read_b64_tr_b16 -- within each 16-lane group, lane j receives element j%4
// of the 8-byte rows read by lanes j/4 + 4i, i < 4.
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

// Keys of a tile (32 KiB of K and V), and the tiles in LDS: one is worked on while
// the next streams in.  (Four places for half the keys, with three tiles on their
// way, took 2-8% longer: a barrier and the loads' addresses for every 64 keys.)
constexpr int keys_of(int d) { return d == 64 ? 128 : 64; }
constexpr int kBuffers = 2;

// Workgroups of a launch that shares the keys out: two per CU.
constexpr int kGroupsShift = 9, kGroups = 1 << kGroupsShift;
// What a piece costs beside its tiles (indices, the first tiles' latency, its
// result), and the least a workgroup is given, in tiles of 64 keys.  (us with a
// cost of 1, 3 and 6, 64 / 8 heads of 64: 16 requests of 1500 keys 27.4, 26.1, 26.4; 32
// of 3000 56.5, 56.6, 58.9.  A least share of 4: 4 requests of 2000 19.6 for 21.0,
// one of 1000 17.7 for 16.3.)
constexpr int kPieceCost = 3, kLeastShare = 2;

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

// Chunk swizzles: 16-byte chunk c of row r lies at chunk c ^ swz(r).  K (16-byte
// operand reads of 16 rows): distinct banks for the rows of a read.  V (8-byte
// transposed reads): a row's chunk pair stays adjacent, distinct bank groups for
// 8 consecutive rows.
template <int D>
__device__ __forceinline__ int swz_k(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
template <int D>
__device__ __forceinline__ int swz_v(int r) { return D == 64 ? r & 6 : (r & 7) << 1; }

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

template <int D>
struct alignas(16) TileLds {
  char k[keys_of(D) * D * 2];  // key-major, 16-byte chunks swizzled per row (swz_k)
  char v[keys_of(D) * D * 2];  // key-major, read transposed, swizzled (swz_v)
};

// D: 64 or 128, the tile's head width; NARROW: head_dim is less.  SUB: a wave's
// row subtiles of 16.
template <typename T, int D, int SUB, bool NARROW>
__global__ void __launch_bounds__(kThreads, 2) tree_attention_kernel(const TreeArgs a) {
  using x4 = typename Vec<T>::x4;
  using x8 = typename Vec<T>::x8;
  constexpr int kKeys = keys_of(D);
  constexpr int kQuarters = kKeys / 32;
  constexpr int kSteps = D / 32;
  constexpr int kDTiles = D / 16;
  constexpr int kChunks = D / 8;             // 16-byte chunks of a row
  constexpr int kLoadRows = 64 / kChunks;    // rows of one wave-wide load
  constexpr int kWaveKeys = kKeys / kWaves;  // keys of a tile that a wave asks for
  constexpr int kEntryTiles = 64 / kWaveKeys;  // tiles whose keys of this wave fill a vector register
  constexpr int kOver = (kPieceCost * 64 + kKeys - 1) / kKeys;
  constexpr int kGroupRows = 16 * SUB;       // rows of a wave
  constexpr int R = kWaves * kGroupRows;     // rows of a block
  __shared__ TileLds<D> buffers[kBuffers];
  __shared__ int32_t s_entry[kWaves][2][64];  // list entries of the waves' keys, kEntryTiles tiles at a time
  __shared__ uint32_t s_dead[2 * kEntryTiles][kQuarters];  // the tiles' keys that no token sees
  __shared__ float s_m[kWaves][kGroupRows], s_l[kWaves][kGroupRows];
  __shared__ int64_t s_out[R];  // where the rows go
  // for the masked quarters: the rows' tokens, first keys and first mask words
  __shared__ uint64_t s_words[kWaves][kGroupRows][kWordsKept];
  __shared__ int32_t s_tok[kWaves][kGroupRows], s_start[kWaves][kGroupRows];
  __shared__ int32_t s_odd;                      // V rows held infinities or NaN that some row does not see
  __shared__ uint64_t s_list[kWaves];            // and the keys that did
  static_assert(kWaves * kGroupRows * D * 4 <= sizeof(buffers), "the waves' results fit the tiles");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // One wave's view of the batch.  A request costs its tiles and kPieceCost for
  // every block of rows; block rb's cost is 0 where the request has no such rows.
  auto units_of = [&](int64_t len, int32_t rows, int rb) -> int32_t {
    if (a.key_starts && len > a.max_len) len = a.max_len;  // what a window reaches is not known here
    const int64_t tiles = len > kKeys ? (len + kKeys - 1) / kKeys : 1;
    return rb * R < rows ? static_cast<int32_t>(tiles + kOver) : 0;
  };
  struct Cost {
    int32_t units, rows;
  };
  auto keys_in = [&](int64_t b) -> int64_t {
    const int64_t len = load_index(a.kv_indptr, a.indptr64, b + 1) - load_index(a.kv_indptr, a.indptr64, b);
    return len < 0 ? 0 : len < kMostKeys ? len : kMostKeys;
  };
  auto cost_of = [&](int64_t b, int rb) -> Cost {
    int64_t q0 = load_index(a.qo_indptr, a.indptr64, b), q1 = load_index(a.qo_indptr, a.indptr64, b + 1);
    q0 = q0 < 0 ? 0 : q0;
    q1 = q1 > a.n_tokens ? a.n_tokens : q1;
    const int32_t rows = q1 > q0 ? static_cast<int32_t>(q1 - q0) * a.group : 0;
    return Cost{units_of(keys_in(b), rows, rb), rows};
  };
  int32_t lane_units = 0;  // of request `lane`, for the block of rows last summed
  auto sum_of = [&](int rb, int32_t* most_rows) -> int64_t {
    int64_t sum = 0;
    int32_t most = 0;
    lane_units = 0;
    for (int b = lane; b < a.n_requests; b += 64) {
      const Cost c = cost_of(b, rb);
      if (b < 64) lane_units = c.units;
      sum += c.units;
      most = max(most, c.rows);
    }
    *most_rows = uniform(__ockl_wfred_max_i32(most));
    return uniform(static_cast<int64_t>(__ockl_wfred_add_i64(sum)));
  };

  if (gated(a.gate)) return;
  int b, g, rb, blocks = 0;
  int64_t off = 0, budget = 0;
  const int group_id = blockIdx.x;
  if (a.whole) {
    // a workgroup per request, KV head and row_blocks-th block of rows
    const int pair = group_id / a.row_blocks;
    rb = group_id - pair * a.row_blocks;
    g = pair / a.n_requests;
    b = pair - g * a.n_requests;
  } else {
    // all work on a line: blocks of rows, KV heads, requests (fastest).  The
    // workgroups take equal stretches of it; a cut falls among a request's tiles.
    int32_t most_rows;
    int64_t sum = sum_of(0, &most_rows);
    blocks = (most_rows + R - 1) / R;
    int64_t all = sum;
    const int32_t first_units = lane_units;
    for (int i = 1; i < blocks; ++i) {
      int32_t unused;
      all += sum_of(i, &unused);
    }
    all *= a.kv_heads;
    lane_units = first_units;
    if (all == 0) return;
    // 2^k stretches: all of the workgroups, or as many as get their least share
    int k = kGroupsShift;
    while (k > 0 && (static_cast<int64_t>((kLeastShare * 64 + kKeys - 1) / kKeys) << k) > all) --k;
    if (group_id >> k) return;
    auto cut = [&](int64_t i) { return (all >> k) * i + (((all & ((1 << k) - 1)) * i) >> k); };  // all * i / 2^k
    int64_t x = cut(group_id);
    budget = cut(group_id + 1) - x;
    rb = 0;
    while (x >= sum * a.kv_heads) {
      int32_t unused;
      x -= sum * a.kv_heads;
      sum = sum_of(++rb, &unused);
    }
    for (g = 0; x >= sum; ++g) x -= sum;
    b = 0;
    for (int b0 = 0; b0 < a.n_requests; b0 += 64) {
      const int32_t mine = b0 == 0 ? lane_units : b0 + lane < a.n_requests ? cost_of(b0 + lane, rb).units : 0;
      const int64_t until = __ockl_wfscan_add_i64(mine, true);
      const uint64_t past = __builtin_amdgcn_ballot_w64(until > x);
      if (past) {
        const int at = __builtin_ctzll(past);
        b = b0 + at;
        off = uniform(x - __shfl(until - mine, at));
        break;
      }
      x -= __shfl(until, 63);
    }
  }

  for (;;) {
    // (in scalar registers: the loop has no vector register to spare)
    int64_t q0 = uniform(load_index(a.qo_indptr, a.indptr64, b)), q1 = uniform(load_index(a.qo_indptr, a.indptr64, b + 1));
    const int64_t kv0 = uniform(load_index(a.kv_indptr, a.indptr64, b));
    const int len = static_cast<int>(uniform(keys_in(b)));
    if (q0 < 0) q0 = 0;
    if (q1 > a.n_tokens) q1 = a.n_tokens;
    const int n = static_cast<int>(q1 > q0 ? q1 - q0 : 0);
    const int rows = n * a.group;
    const int old = len > n ? len - n : 0;
    if (a.whole && rb * R >= rows) return;
    // the keys that some token of the request sees begin here
    int lo = 0, hi_start = 0;
    if (a.key_starts) {
      lo = old;
      for (int i = lane; i < n; i += 64) {
        const int s = min(max(a.key_starts[q0 + i], 0), old);
        lo = min(lo, s);
        hi_start = max(hi_start, s);
      }
      lo = uniform(__ockl_wfred_min_i32(lo));
      hi_start = uniform(__ockl_wfred_max_i32(hi_start));
    }
    // the piece: units [off, stop) of the request's, the first kPieceCost of them
    // for no tile, the others for equal parts of its tiles
    const int units = units_of(len, rows, rb);
    const int stop = a.whole || budget > units - off ? units : static_cast<int>(off + budget);
    const bool first = off == 0, last = stop == units;
    const int all_tiles = (len - lo + kKeys - 1) / kKeys;
    auto tile_of = [&](int64_t unit) -> int {
      const int64_t at = unit > kOver ? unit - kOver : 0;
      return static_cast<int>(units - kOver == all_tiles ? at : at * all_tiles / (units - kOver));
    };
    const int begin = lo + uniform(tile_of(off)) * kKeys;
    const int end = min(lo + uniform(tile_of(stop)) * kKeys, len);
    const int tiles = end > begin ? (end - begin + kKeys - 1) / kKeys : 0;

    // (an empty pool holds no key: every slot is a hole, and zeros are read)
    const bool pool = a.pool_slots > 0;
    const char* kbase = pool ? a.k + g * a.k_sh : reinterpret_cast<const char*>(zero_row);
    const char* vbase = pool ? a.v + g * a.v_sh : reinterpret_cast<const char*>(zero_row);
    const uint32_t k_ss = pool ? a.k_ss : 0, v_ss = pool ? a.v_ss : 0;
    const int32_t* list = a.kv_indices + (a.paged ? b * a.table_stride : kv0);
    // entries of the list that exist
    const int64_t left = a.paged ? a.table_width : kv0 < 0 ? 0 : a.table_width - kv0;
    const int32_t width = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(left, 0), 0x7fffffff));
    const int32_t* entries = width > 0 ? list : reinterpret_cast<const int32_t*>(zero_row);
    const int last_entry = max(width - 1, 0);
    // The wave's keys of kEntryTiles tiles at a time: lane l has key l % kWaveKeys
    // of tile l / kWaveKeys.  Their list entries come to LDS kEntryTiles tiles ahead.
    const int my_key = lane / kWaveKeys * kKeys + kWaveKeys * wave + lane % kWaveKeys;
    auto fetch = [&](int e) {
      const uint32_t j = min(begin + e * (kEntryTiles * kKeys) + my_key, end - 1);  // past the end: the last key's
      const int32_t at = a.paged ? j / static_cast<uint32_t>(a.page_size) : j;
      load_4(entries + min(at, last_entry), uniform(lds_address(s_entry[wave][e & 1])));
    };
    uint32_t slots = 0;
    auto look_up = [&](int e) {
      const uint32_t key = begin + e * (kEntryTiles * kKeys) + my_key, j = min(key, static_cast<uint32_t>(end - 1));
      const int32_t entry = s_entry[wave][e & 1][lane];
      uint64_t slot = static_cast<uint32_t>(entry);
      uint32_t at = j;
      if (a.paged) {
        const uint32_t page = a.page_size;
        at = j / page;
        slot = slot * page + (j - at * page);
      }
      const bool there = entry >= 0 && at < static_cast<uint32_t>(width) && slot < static_cast<uint64_t>(a.pool_slots);
      // a hole reads slot 0; the mask keeps it from every row
      slots = there ? static_cast<uint32_t>(slot) : 0;
      const uint64_t dead = __builtin_amdgcn_ballot_w64(!there || key >= static_cast<uint32_t>(end));
      if (lane < kEntryTiles) {
        const uint32_t mine = static_cast<uint32_t>(dead >> (kWaveKeys * lane));
        char* to = reinterpret_cast<char*>(s_dead[(e & 1) * kEntryTiles + lane]) + kWaveKeys / 8 * wave;
        if constexpr (kWaveKeys == 32)
          *reinterpret_cast<uint32_t*>(to) = mine;
        else
          *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(mine);
      }
    };
    // a wave's keys of a tile, straight into LDS: lane l of a load fills bytes
    // 16 l of a 1 KiB block, chunk position l % kChunks of a row
    auto stage = [&](int it) {
      if (it % kEntryTiles == 0) {
        look_up(it / kEntryTiles);
        fetch(it / kEntryTiles + 1);
      }
      TileLds<D>& t = buffers[it % kBuffers];
  #pragma unroll
      for (int u = 0; u < kWaveKeys / kLoadRows; ++u) {
        const int mine = u * kLoadRows + lane / kChunks, r = kWaveKeys * wave + mine;
        const uint64_t from = __shfl(slots, it % kEntryTiles * kWaveKeys + mine);
        const int ck = (lane % kChunks) ^ swz_k<D>(r), cv = (lane % kChunks) ^ swz_v<D>(r);
        const char* krow = kbase + from * k_ss + 16 * ck;
        const char* vrow = vbase + from * v_ss + 16 * cv;
        if (NARROW) {  // dims past head_dim read zeros
          krow = 8 * ck < a.head_dim ? krow : reinterpret_cast<const char*>(zero_row);
          vrow = 8 * cv < a.head_dim ? vrow : reinterpret_cast<const char*>(zero_row);
        }
        const int place = (kWaveKeys * wave + u * kLoadRows) * D * 2;
        load_16(krow, uniform(lds_address(t.k + place)));
        load_16(vrow, uniform(lds_address(t.v + place)));
      }
    };
    if (tiles > 0) fetch(0);
    if (threadIdx.x == 0) s_odd = 0;
    // groups of rows, and the waves that share one
    int groups = kWaves, sharers = 1;
    while (groups > 1 && sharers < kQuarters && rows - rb * R <= (groups >> 1) * kGroupRows) {
      groups >>= 1;
      sharers <<= 1;
    }
    const int row0 = rb * R + (wave & (groups - 1)) * kGroupRows;
    const int share = uniform(wave / groups);
    // this lane's rows: r = row0 + 16 s + col, token r / G, head g G + r % G
    // (rows past the last repeat it and are never stored)
    x8 qop[SUB][kSteps];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int r = min(row0 + 16 * s + col, rows - 1);
      const int tok = r / a.group;
      const T* row = static_cast<const T*>(a.q) + (q0 + tok) * a.q_st +
                     static_cast<int64_t>(g * a.group + r - tok * a.group) * a.q_sh;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        u32x4 w = {0u, 0u, 0u, 0u};
        const int c = 4 * st + quad;
        if (!NARROW || 8 * c < a.head_dim) w = *((const global_u32x4*)row + c);
        qop[s][st] = __builtin_bit_cast(x8, w);
      }
    }
    f32x4 acc[SUB][kDTiles];
    float neg_m[SUB], l[SUB];  // l: 0 while the row has seen no key
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      neg_m[s] = 0.f;
      l[s] = 0.f;
#pragma unroll
      for (int t = 0; t < kDTiles; ++t) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool unset = true;  // some row of the wave has seen no key yet
    x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.f);

    // word w of a token's mask row
    auto mask_word = [&](int tok, int w) -> uint64_t {
      if (a.mask) return w < a.mask_words ? a.mask[(q0 + tok) * a.mask_stride + w] : 0;
      const int i = tok - 64 * w;
      return i >= 63 ? ~0ull : i < 0 ? 0 : (2ull << i) - 1;
    };
    auto start_of = [&](int tok) -> int { return a.key_starts ? min(max(a.key_starts[q0 + tok], 0), old) : 0; };
    // what a row sees of the 32 keys from k0 on: those from `start` on, and the
    // drafted ones by its words
    auto visible = [&](int k0, int start, auto word) -> uint32_t {
      const int base = k0 - old;
      uint64_t bits = ~0ull;
      if (base > -32) {
        if (base < 0) {
          bits = word(0) << -base | ((1ull << -base) - 1);
        } else {
          const int w = base >> 6, by = base & 63;
          bits = word(w) >> by;
          if (by > 32) bits |= word(w + 1) << (64 - by);
        }
      }
      const int hidden = start - k0;
      if (hidden >= 32) bits = 0; else if (hidden > 0) bits &= ~0ull << hidden;
      return static_cast<uint32_t>(bits);
    };
    if (lane < kGroupRows) {
      const int tok = min(row0 + lane, rows - 1) / a.group;
      s_tok[wave][lane] = tok;
      s_start[wave][lane] = start_of(tok);
#pragma unroll
      for (int w = 0; w < kWordsKept; ++w) s_words[wave][lane][w] = mask_word(tok, w);
    }
    // A weight of 0 does not hide an infinity or NaN from the product.  Where
    // rows see different keys such values are cleared (by every wave that uses
    // them) and the block takes note: its rows get them back at the end.
    auto clear_odd = [&](char* quarter, uint32_t dead) {
      u16x2 top = {0, 0};  // largest bits without the sign
#pragma unroll
      for (int i = 0; i < kDTiles; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(quarter + 1024 * i + 16 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
      }
      if (!__builtin_amdgcn_ballot_w64(not_finite<T>(top.x) || not_finite<T>(top.y))) return;
      bool noted = false;
#pragma nounroll
      for (int i = 0; i < kDTiles; ++i) {
        s16x8* here = reinterpret_cast<s16x8*>(quarter + 1024 * i + 16 * lane);
        s16x8 w = *here;
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool one = not_finite<T>(w[e]);
          odd |= one;
          w[e] = one ? 0 : w[e];
        }
        if (odd) *here = w;
        noted |= odd && !(dead >> ((64 * i + lane) / kChunks) & 1);
      }
      if (noted) s_odd = 1;
    };
    // this lane's operands in quarter 0: K chunks 4 st + quad of row col, and the
    // source of its transposed V reads (row 4 quad + col / 4, dims 16 dt + 4 (col
    // % 4)); the swizzles are the same in every quarter
    uint32_t k_at[kSteps], v_at[kDTiles];
    const int vr = 4 * quad + (col >> 2);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) k_at[st] = col * D * 2 + 16 * ((4 * st + quad) ^ swz_k<D>(col));
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt)
      v_at[dt] = vr * D * 2 + 16 * ((2 * dt + (col >> 1 & 1)) ^ swz_v<D>(vr)) + 8 * (col & 1);
    // scores of the 32 keys of a quarter: S^T[16 j + 4 quad + i][row 16 s + col]
    auto scores = [&](const TileLds<D>& t, int kk, f32x4 (&sc)[2][SUB]) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const x8 kop = __builtin_bit_cast(x8, *reinterpret_cast<const u32x4*>(t.k + (64 * kk + 32 * j) * D + k_at[st]));
#pragma unroll
          for (int s = 0; s < SUB; ++s)
            sc[j][s] = product(kop, qop[s][st], st == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[j][s]);
        }
      }
    };
    // O^T += V^T . P^T: lane col of group quad receives V[key][16 dt + col] for
    // keys 4 quad + i (i < 4) of the quarter, then 16 keys on.  Reads are two
    // tiles of 16 dims ahead of the products, the first two before the
    // exponentials; barriers for the compiler's schedule keep them there (1% to 2%).
    auto v_tile = [&](const TileLds<D>& t, int kk, int dt) -> x8 {
      const s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t.v + 64 * kk * D + v_at[dt]));
      const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(t.v + (64 * kk + 32) * D + v_at[dt]));
      return __builtin_bit_cast(x8, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto values = [&](const TileLds<D>& t, int kk, const x8 (&p)[SUB], x8 v0, x8 v1) {
      x8 v[2] = {v0, v1};
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) acc[s][dt] = product(v[dt & 1], p[s], acc[s][dt]);
        if (dt + 2 < kDTiles) v[dt & 1] = v_tile(t, kk, dt + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // 32 keys that every row sees, when every row has a maximum; false, with
    // nothing done, where a sum outgrows kHuge
    auto quick = [&](const TileLds<D>& t, int kk) -> bool {
      f32x4 sc[2][SUB];
      scores(t, kk, sc);
      const x8 v0 = v_tile(t, kk, 0), v1 = v_tile(t, kk, 1);
      __builtin_amdgcn_sched_barrier(0);
      x8 p[SUB];
      float sum[SUB];
      bool huge = false;
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        f32x4 e0, e1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e0[i] = __builtin_amdgcn_exp2f(fmaf(sc[0][s][i], a.scale_log2, neg_m[s]));
          e1[i] = __builtin_amdgcn_exp2f(fmaf(sc[1][s][i], a.scale_log2, neg_m[s]));
        }
        p[s] = __builtin_shufflevector(__builtin_convertvector(e0, x4), __builtin_convertvector(e1, x4), 0, 1, 2, 3, 4,
                                       5, 6, 7);
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        sum[s] = l[s] + product(ones, p[s], f32x4{0.f, 0.f, 0.f, 0.f})[0];
        huge |= sum[s] > kHuge;
      }
      if (__builtin_amdgcn_ballot_w64(huge)) return false;
#pragma unroll
      for (int s = 0; s < SUB; ++s) l[s] = sum[s];
      values(t, kk, p, v0, v1);
      return true;
    };
    // any 32 keys; k0: the first one's rank
    auto quarter = [&](TileLds<D>& t, int kk, int k0, uint32_t dead) {
      const bool masked = dead != 0 || k0 + 32 > old || k0 < hi_start;
      f32x4 sc[2][SUB];
      scores(t, kk, sc);
      if (masked) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          const int in = 16 * s + col;
          const uint32_t seen = ~dead & visible(k0, s_start[wave][in], [&](int w) -> uint64_t {
            return w < kWordsKept ? s_words[wave][in][w] : mask_word(s_tok[wave][in], w);
          });
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[j][s][i] = seen >> (16 * j + 4 * quad + i) & 1 ? sc[j][s][i] : -INFINITY;
        }
      }
      // A row's m is its maximum over the first quarter it sees a key of, and then
      // stays put: the sum tells when it should not have.  A sum past kHuge (a
      // score ~32 above m in the log2 domain, 16 in fp16, whose weight is then
      // infinite) takes the quarter again with exact maxima.
      x8 p[SUB];
      float sum[SUB];
      for (bool exact = unset;; exact = true) {
        if (exact) {
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            const float m0 = max3(sc[0][s][0], sc[0][s][1], sc[0][s][2]);
            const float m1 = max3(sc[0][s][3], sc[1][s][0], sc[1][s][1]);
            const float mx = column_max(max3(m0, m1, max2(sc[1][s][2], sc[1][s][3])));
            const float over = fmaf(mx, a.scale_log2, neg_m[s]);  // above m
            const bool any = l[s] != 0.f;
            // (a sum near kHuge whose large weights lie behind moves by 2^16)
            const bool down = l[s] > 0.5f * kHuge && !(over > 16.f);
            const bool move = any ? over > 0.f : mx > -INFINITY;
            const float alpha = down ? 0x1p-16f : move && any ? __builtin_amdgcn_exp2f(-over) : 1.f;
            l[s] *= alpha;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) acc[s][dt] *= alpha;
            neg_m[s] = down ? neg_m[s] - 16.f : move ? -(mx * a.scale_log2) : neg_m[s];
          }
        }
        bool huge = false;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          f32x4 e0, e1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e0[i] = __builtin_amdgcn_exp2f(fmaf(sc[0][s][i], a.scale_log2, neg_m[s]));
            e1[i] = __builtin_amdgcn_exp2f(fmaf(sc[1][s][i], a.scale_log2, neg_m[s]));
          }
          p[s] = __builtin_shufflevector(__builtin_convertvector(e0, x4), __builtin_convertvector(e1, x4), 0, 1, 2, 3,
                                         4, 5, 6, 7);
          sum[s] = l[s] + product(ones, p[s], f32x4{0.f, 0.f, 0.f, 0.f})[0];
          huge |= sum[s] > kHuge;
        }
        if (exact || !__builtin_amdgcn_ballot_w64(huge)) break;
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) l[s] = sum[s];
      if (unset) {
        bool none = false;
#pragma unroll
        for (int s = 0; s < SUB; ++s) none |= l[s] == 0.f;
        unset = __builtin_amdgcn_ballot_w64(none) != 0;
      }
      if (masked) clear_odd(t.v + 64 * kk * D, dead);
      values(t, kk, p, v_tile(t, kk, 0), v_tile(t, kk, 1));
    };
    __builtin_amdgcn_s_waitcnt(0);  // (one the compiler sees: Q has arrived)
    __syncthreads();
    if (tiles > 0) stage(0);
    arrive();
    // this wave's quarters of a tile
    uint32_t quarters = 0;
#pragma unroll
    for (int kk = 0; kk < kQuarters; ++kk) quarters |= (kk & (sharers - 1)) == share ? 1u << kk : 0;
#pragma nounroll
    for (int it = 0; it < tiles; ++it) {
      // into the place that was last read before the barrier
      if (it + 1 < tiles) stage(it + 1);
      TileLds<D>& t = buffers[it % kBuffers];
      const int t0 = begin + it * kKeys;
      const uint32_t* dead = s_dead[it % (2 * kEntryTiles)];
      uint32_t holes = dead[0];
#pragma unroll
      for (int kk = 1; kk < kQuarters; ++kk) holes |= dead[kk];
      uint32_t todo = quarters;
      if (!unset && t0 + kKeys <= old && t0 >= hi_start && uniform(holes) == 0) {
#pragma unroll
        for (int kk = 0; kk < kQuarters; ++kk)
          if (todo >> kk & 1 && quick(t, kk)) todo &= ~(1u << kk);
      }
#pragma nounroll
      for (; todo; todo &= todo - 1) {
        const int kk = __builtin_ctz(todo), k0 = t0 + 32 * kk;
        if (k0 >= end) break;
        quarter(t, kk, k0, uniform(dead[kk]));
      }
      arrive();
    }

    // the waves' O rows [row][dim] over the tiles, four-float groups turned by
    // the row for the banks; the sharers of a group meet there
    auto result_of = [&](int w) -> float* {
      return reinterpret_cast<float*>(buffers) + w * kGroupRows * D;
    };
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int r = 16 * s + col;
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
        *reinterpret_cast<f32x4*>(result_of(wave) + r * D + ((16 * dt + 4 * quad) ^ (col & 7) << 2)) = acc[s][dt];
      if (quad == 0) {
        s_m[wave][r] = l[s] == 0.f ? -INFINITY : -neg_m[s];
        s_l[wave][r] = l[s];
      }
    }
    __syncthreads();
    const int here = min(rows - rb * R, groups * kGroupRows);
    // an unfinished piece: a stretch has at most one that continues an earlier
    // stretch's, and one that the next continues
    const int64_t place = 2 * group_id + (first ? 1 : 0);
    float* part = a.part_o + place * R * D;
    float* part_ml = a.part_ml + place * R * 2;
    // a thread per row: the sharers' factors, with the sink and the sum when the
    // piece is all of it
    const int mine = here_only(threadIdx.x);
    if (mine < here) {
      const int r = rb * R + mine, token = r / a.group, head = g * a.group + r - token * a.group;
      const int64_t row = q0 + token;
      const int group = mine / kGroupRows, in = mine % kGroupRows;
      float m = -INFINITY, lt = 0.f;
      for (int w = group; w < kWaves; w += groups) m = fmaxf(m, s_m[w][in]);
      // a wave that has seen no key carries m = -inf, l = 0 and O = 0
      float base = m == -INFINITY ? 0.f : m;
      for (int w = group; w < kWaves; w += groups) lt += s_l[w][in] * __builtin_amdgcn_exp2f(s_m[w][in] - base);
      float scale = 1.f;
      if (first && last) {
        if (a.sinks) {
          const float sink = a.sinks[head] * kLog2e, top = fmaxf(m, sink);
          const float by = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
          lt = lt * by + (top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - top));
          scale = by;
        }
        s_out[mine] = row * a.o_st + head * a.o_sh;
      } else {
        *reinterpret_cast<f32x2*>(part_ml + 2 * mine) = f32x2{m, lt};
      }
      scale *= inverse(lt);
      for (int w = group; w < kWaves; w += groups) s_m[w][in] = __builtin_amdgcn_exp2f(s_m[w][in] - base) * scale;
      if (!a.whole) {
        int32_t* owner = a.owner + 4 * (row * a.q_heads + head);
        if (first) {
          owner[0] = last ? -1 : group_id;
          owner[2] = mine;
        }
        if (last) owner[1] = group_id;
      }
    }
    __syncthreads();
    constexpr int kRowsAtOnce = kThreads / (D / 4);
    const int d = 4 * (mine % (D / 4));
    if (!NARROW || d < a.head_dim) {
#pragma unroll 2
      for (int r = mine / (D / 4); r < here; r += kRowsAtOnce) {
        const int group = r / kGroupRows, in = r % kGroupRows;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int w = group; w < kWaves; w += groups)
          o += *reinterpret_cast<const f32x4*>(result_of(w) + in * D + (d ^ (in & 7) << 2)) * s_m[w][in];
        if (first && last)
          store_four<T>(a, s_out[r] + d, o);
        else
          *reinterpret_cast<f32x4*>(part + r * D + d) = o;
      }
    }
    // values cleared from the products go back, unweighted, to the rows that see
    // them: whatever their weights, the results are the infinity or NaN
    if (s_odd) {
      for (int base = begin; base < end; base += kThreads) {
        auto v_row = [&](int j) -> const T* {
          const uint32_t per = a.paged ? a.page_size : 1, at = static_cast<uint32_t>(j) / per;
          if (static_cast<int64_t>(at) >= width || list[at] < 0) return nullptr;
          const uint64_t slot = static_cast<uint64_t>(list[at]) * per + (static_cast<uint32_t>(j) - at * per);
          return slot < static_cast<uint64_t>(a.pool_slots) ? reinterpret_cast<const T*>(vbase + slot * v_ss) : nullptr;
        };
        const int key = base + static_cast<int>(threadIdx.x);
        const T* row = key < end ? v_row(key) : nullptr;
        bool odd = false;
        for (int d = 0; row && d < a.head_dim; ++d) odd |= not_finite<T>(__builtin_bit_cast(short, row[d]));
        const uint64_t odds = __builtin_amdgcn_ballot_w64(odd);
        if (lane == 0) s_list[wave] = odds;
        __syncthreads();
        for (int u = threadIdx.x; u < here * (D / 4); u += kThreads) {
          const int r = rb * R + u / (D / 4), d = 4 * (u % (D / 4));
          const int token = r / a.group, head = g * a.group + r - token * a.group;
          if (NARROW && d >= a.head_dim) continue;
          for (int w = 0; w < kWaves; ++w)
            for (uint64_t rest = s_list[w]; rest; rest &= rest - 1) {
              const int j = base + 64 * w + __builtin_ctzll(rest);
              if (!(visible(j, start_of(token), [&](int w) { return mask_word(token, w); }) & 1)) continue;
              const T* v = v_row(j) + d;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (!not_finite<T>(__builtin_bit_cast(short, v[i]))) continue;
                const float x = static_cast<float>(v[i]);
                if (!(first && last)) {
                  part[(r - rb * R) * D + d + i] += x;
                  continue;
                }
                const int64_t at = (q0 + token) * a.o_st + head * a.o_sh + d + i;
                if (a.out_f32)
                  static_cast<float*>(a.out)[at] += x;
                else
                  static_cast<T*>(a.out)[at] = static_cast<T>(static_cast<float>(static_cast<T*>(a.out)[at]) + x);
              }
            }
        }
        __syncthreads();
      }
    }
    __syncthreads();
    if (a.whole) {
      rb += a.row_blocks;
      continue;
    }
    budget -= stop - off;
    if (budget <= 0) return;
    // the next request on the line
    off = 0;
    for (++b;;) {
      int found = -1;
      for (int b0 = b; b0 < a.n_requests && found < 0; b0 += 64) {
        const uint64_t live = __builtin_amdgcn_ballot_w64(b0 + lane < a.n_requests && cost_of(b0 + lane, rb).units > 0);
        if (live) found = b0 + __builtin_ctzll(live);
      }
      if (found >= 0) {
        b = found;
        break;
      }
      b = 0;
      if (++g == a.kv_heads) {
        g = 0;
        if (++rb >= blocks) return;
      }
    }
  }
}

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

int tile_dim(int32_t head_dim) { return head_dim <= 64 ? 64 : 128; }

// A wave's row subtiles for requests of up to `rows` rows: a tile has keys for
// four waves (two at D = 128) to share a group of rows, so the rows are dealt out
// to two (four) groups before a wave takes more of them.  (us for 16 requests of
// 4096 keys, 64 / 8 heads of 64, the waves' rows halved, as here, doubled: 64 rows a
// KV head 39.1, 38.6, 38.9, 128 rows 47.0, 46.7, 47.0; 32 / 8 heads of 128: 64 rows
// 60.5, 61.2, 64.1, 128 rows 86.0, 73.6, 72.9.)
int subtiles_for(int d, int64_t rows) {
  const int most = d == 64 ? 4 : 2;
  const int64_t groups = d == 64 ? 2 : 4;
  int sub = 1;
  while (sub < most && rows > 16 * groups * sub) sub *= 2;
  return sub;
}

// Workgroups of 256 threads in a launch: a grid has fewer than 2^32 threads, and
// what is beyond is left out without an error.
constexpr int64_t kMostBlocks = 1 << 23;

struct Launch {
  int d, sub;
  bool whole;
  int32_t row_blocks;
};

// Where a block of rows is one workgroup's from its first key to its last: the
// second launch and the pieces cost 6 to 10 us, more than a cut saves on up to four
// tiles (8 tokens, 64 / 8 heads of 64, one request, us whole and cut: 384 keys
// 14.3, 15.9; 512: 15.8, 16.0; 768: 18.7, 14.6), or, where the workgroups fill half
// the chip, on up to 1024 keys (the same with 16 requests of 1024: 21.7, 24.6, of
// 2048: 32.6, 29.3; 64 requests of 8 to 1024: 27.9, 41.2; with one of 1024 among
// 63 of 100: 25.0, 29.5; 65 requests of 1024, a round and a bit: 47.9, 45.5).
constexpr int64_t kWholeTiles = 4, kWholeKeys = 1024, kWholeGroups = 128;

// Rows of a KV head that a request may have.
int64_t most_rows(int64_t n_tokens, int64_t q_heads, int64_t kv_heads, int64_t max_new) {
  return std::max<int64_t>(1, std::min(max_new, n_tokens)) * (q_heads / kv_heads);
}

Launch plan(int64_t n_tokens, int64_t n_requests, int64_t q_heads, int64_t kv_heads, int32_t head_dim,
            int64_t max_len, int64_t max_new) {
  Launch p;
  p.d = tile_dim(head_dim);
  const int64_t rows = most_rows(n_tokens, q_heads, kv_heads, max_new);
  p.sub = subtiles_for(p.d, rows);
  auto blocks = [&]() -> int64_t { return (rows + 16 * kWaves * p.sub - 1) / (16 * kWaves * p.sub); };
  p.whole = max_len <= kWholeTiles * keys_of(p.d) ||
            (max_len <= kWholeKeys && n_requests * kv_heads * blocks() >= kWholeGroups);
  // (32 requests, 8 KV heads, 128 rows of 64 over a window's 145 keys: 16.5 us in
  // blocks of 128 rows, 18.2 in 256; 128 requests of 64 rows: no difference)
  if (p.whole && p.sub == 4 && n_requests * kv_heads * ((rows + 127) / 128) <= kGroups) p.sub = 2;
  // (further blocks of rows follow in the same workgroup)
  const int64_t room = std::max<int64_t>(1, kMostBlocks / std::max<int64_t>(1, n_requests * kv_heads));
  p.row_blocks = static_cast<int32_t>(std::min(blocks(), std::min<int64_t>(room, 4096)));
  return p;
}

int64_t owner_bytes(int64_t n_tokens, int64_t q_heads) { return 16 * n_tokens * q_heads; }

int64_t cut_bytes(int d, int sub, int64_t n_tokens, int64_t q_heads) {
  return owner_bytes(n_tokens, q_heads) + 2ll * kGroups * (16 * kWaves * sub) * (d + 2) * 4;
}

// What a launch needs.
int64_t partial_bytes(const Launch& p, int64_t n_tokens, int64_t q_heads) {
  return p.whole ? 16 : cut_bytes(p.d, p.sub, n_tokens, q_heads);
}

// What every batch of up to these sizes and bounds needs: a batch that fills the
// chip runs whole, but one of fewer requests under the same bounds is cut.
int64_t largest_bytes(int64_t n_tokens, int64_t q_heads, int64_t kv_heads, int32_t head_dim, int64_t max_len,
                      int64_t max_new) {
  const int d = tile_dim(head_dim);
  if (max_len <= kWholeTiles * keys_of(d)) return 16;
  return cut_bytes(d, subtiles_for(d, most_rows(n_tokens, q_heads, kv_heads, max_new)), n_tokens, q_heads);
}

template <typename T, int D, int SUB>
void start(const TreeArgs& a, dim3 grid, hipStream_t st) {
  if (a.head_dim < D)
    hipLaunchKernelGGL((tree_attention_kernel<T, D, SUB, true>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tree_attention_kernel<T, D, SUB, false>), grid, dim3(kThreads), 0, st, a);
}

// Few rows are cut into many pieces each, and many rows fill the chip: a wave per
// row up to kFewRows, D / 4 lanes beyond (both launches, us by the wave and by the
// lanes: 512 rows of one request of 8192 keys 22.6, 31.5; 4096 rows 42.8, 44.8; 16384
// rows of 16 requests of 4096 49.7, 46.8).  Up to kFewestRows all of a row's pieces
// are on their way at once, 16 per way, 4 beyond (128 rows of 128 dims over 4096 keys
// 16.8, 18.3; 512 rows over 8192 21.1, 22.1; 4096 rows 44.2, 41.2).
constexpr int64_t kFewRows = 4096, kFewestRows = 512;

template <typename T, int D, int WAYS, int AHEAD>
void merge_by(const TreeArgs& a, const Launch& p, hipStream_t st) {
  constexpr int kRows = 256 / (D / 4 * WAYS);
  const int64_t rows = a.n_tokens * a.q_heads;
  for (int64_t row0 = 0; row0 < rows; row0 += kMostBlocks * kRows) {
    const dim3 grid(static_cast<unsigned>(std::min(kMostBlocks, (rows - row0 + kRows - 1) / kRows)));
    hipLaunchKernelGGL((tree_combine_kernel<T, D, WAYS, AHEAD>), grid, dim3(256), 0, st, a, 16 * kWaves * p.sub, row0);
  }
}

template <typename T, int D>
void merge(const TreeArgs& a, const Launch& p, hipStream_t st) {
  constexpr int kWays = 64 / (D / 4);
  const int64_t rows = a.n_tokens * a.q_heads;
  if (rows <= kFewestRows)
    merge_by<T, D, kWays, 16>(a, p, st);
  else if (rows <= kFewRows)
    merge_by<T, D, kWays, 4>(a, p, st);
  else
    merge_by<T, D, 1, 4>(a, p, st);
}

template <typename T>
int launch(const TreeArgs& a, const Launch& p, hipStream_t st) {
  const int64_t blocks = p.whole ? static_cast<int64_t>(a.n_requests) * a.kv_heads * a.row_blocks : kGroups;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (p.d == 64) {
    if (p.sub == 1) start<T, 64, 1>(a, grid, st);
    else if (p.sub == 2) start<T, 64, 2>(a, grid, st);
    else start<T, 64, 4>(a, grid, st);
  } else {
    if (p.sub == 1) start<T, 128, 1>(a, grid, st);
    else start<T, 128, 2>(a, grid, st);
  }
  int rc = check_launch("akv_tree_attention");
  if (rc || p.whole) return rc;
  if (p.d == 64)
    merge<T, 64>(a, p, st);
  else
    merge<T, 128>(a, p, st);
  return check_launch("akv_tree_attention (combine)");
}

bool sizes_ok(int64_t n_tokens, int32_t n_requests, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
              int64_t max_len, int64_t max_new) {
  return n_tokens >= 0 && n_requests >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 &&
         head_dim > 0 && head_dim <= 128 && head_dim % 8 == 0 && max_len >= 0 && max_new >= 0;
}

}  // namespace
}  // namespace akv

extern "C" int64_t akv_tree_attention_workspace_bytes(int64_t n_tokens, int32_t n_requests, int32_t q_heads,
                                                       int32_t kv_heads, int32_t head_dim, int64_t max_len,
                                                       int64_t max_new) {
  using namespace akv;
  if (!sizes_ok(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len, max_new)) return -1;
  return largest_bytes(n_tokens, q_heads, kv_heads, head_dim, max_len, max_new);
}

extern "C" int akv_tree_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_buffer,
                                  const void* v_buffer, int64_t k_stride_slot, int64_t k_stride_head,
                                  int64_t v_stride_slot, int64_t v_stride_head, int64_t pool_slots, int32_t dtype,
                                  int64_t n_tokens, int32_t n_requests, int32_t q_heads, int32_t kv_heads,
                                  int32_t head_dim, const void* qo_indptr, const void* kv_indptr,
                                  int32_t indptr_dtype, const int32_t* kv_indices, int64_t table_stride,
                                  int64_t table_width, int32_t page_size, const uint64_t* tree_mask,
                                  int64_t mask_stride, int32_t mask_words, const int32_t* key_starts,
                                  const float* sinks, float scale, void* out, int32_t out_dtype, int64_t out_stride_t,
                                  int64_t out_stride_h, int64_t max_len, int64_t max_new, void* workspace,
                                  int64_t workspace_bytes, const int32_t* status, void* stream) {
  using namespace akv;
  if (n_tokens < 0 || n_requests < 0 || max_len < 0 || max_new < 0 || pool_slots < 0 || table_width < 0 ||
      table_stride < 0 || mask_words < 0)
    return fail(AKV_EINVAL, "akv_tree_attention: negative size");
  if (n_tokens == 0 || n_requests == 0) return AKV_OK;
  if (head_dim < 8 || head_dim > 128 || head_dim % 8)
    return fail(AKV_EINVAL, "akv_tree_attention: head_dim %d (multiples of 8 up to 128)", head_dim);
  if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0)
    return fail(AKV_EINVAL, "akv_tree_attention: %d q heads over %d KV heads", q_heads, kv_heads);
  if (dtype != AKV_BF16 && dtype != AKV_F16)
    return fail(AKV_EINVAL, "akv_tree_attention: q, K and V must be bf16 or fp16");
  if (out_dtype != dtype && out_dtype != AKV_F32)
    return fail(AKV_EINVAL, "akv_tree_attention: the output must have q's type or be f32");
  if (!valid_index_dtype(indptr_dtype)) return fail(AKV_EINVAL, "akv_tree_attention: indptrs must be int32 or int64");
  if (page_size < 1) return fail(AKV_EINVAL, "akv_tree_attention: page_size must be positive");
  if (table_stride == 0 && page_size != 1)
    return fail(AKV_EINVAL, "akv_tree_attention: pages need a block table (a list holds one slot per key)");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(AKV_EINVAL, "akv_tree_attention: scale must be positive and finite");
  // (an empty pool or list need not have an address: every key is a hole then)
  if (!q || (pool_slots > 0 && (!k_buffer || !v_buffer)) || !qo_indptr || !kv_indptr ||
      (table_width > 0 && !kv_indices) || !out || !workspace)
    return fail(AKV_EINVAL, "akv_tree_attention: null device pointer");
  if ((q_stride_t | q_stride_h | k_stride_slot | k_stride_head | v_stride_slot | v_stride_head) % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_buffer) |
        reinterpret_cast<uintptr_t>(v_buffer) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0)
    return fail(AKV_EINVAL, "akv_tree_attention: q, K and V rows and the workspace must be 16-byte aligned");
  if (pool_slots > 0xffffffffLL || (k_stride_slot | v_stride_slot) >> 31 || n_tokens > 0x7f000000LL / q_heads ||
      static_cast<int64_t>(n_requests) * kv_heads > 0x7fffffffLL / 4096)
    return fail(AKV_EINVAL, "akv_tree_attention: batch too large");
  const Launch p = plan(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len, max_new);
  const int64_t need = partial_bytes(p, n_tokens, q_heads);
  if (workspace_bytes < need)
    return fail(AKV_EINVAL, "akv_tree_attention: workspace holds %lld bytes, needs %lld",
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  TreeArgs a{};
  a.q = q;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = static_cast<const char*>(k_buffer);
  a.v = static_cast<const char*>(v_buffer);
  a.k_ss = 2 * k_stride_slot;
  a.k_sh = 2 * k_stride_head;
  a.v_ss = 2 * v_stride_slot;
  a.v_sh = 2 * v_stride_head;
  a.pool_slots = pool_slots;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.kv_indices = kv_indices;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.mask = tree_mask;
  a.mask_stride = mask_stride;
  a.mask_words = mask_words;
  a.key_starts = key_starts;
  a.sinks = sinks;
  a.gate = status;
  a.scale_log2 = scale * kLog2e;
  a.out = out;
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.owner = static_cast<int32_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + owner_bytes(n_tokens, q_heads));
  a.part_ml = a.part_o + 2ll * kGroups * (16 * kWaves * p.sub) * p.d;
  a.n_tokens = n_tokens;
  a.max_len = max_len;
  a.n_requests = n_requests;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.row_blocks = p.row_blocks;
  a.whole = p.whole;
  a.indptr64 = indptr_dtype == AKV_I64;
  a.out_f32 = out_dtype == AKV_F32;
  a.out_vectors = (out_stride_t | out_stride_h) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(out) % (out_dtype == AKV_F32 ? 16 : 8) == 0;
  a.paged = table_stride != 0;
  hipStream_t st = as_stream(stream);
  if (dtype == AKV_F16) return launch<_Float16>(a, p, st);
  return launch<__bf16>(a, p, st);
}
