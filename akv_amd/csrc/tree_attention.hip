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
// again for every further one.  Workgroup = (chunk of keys, KV head, request,
// block of rows), four waves, two workgroups per CU.  Tiles of K and V stream
// into LDS (global_load_lds, two buffers) while the one before is worked on, in
// 32-key quarters, 16 SUB rows per wave:
//   S^T[32 x 16 SUB] = K . Q^T              v_mfma_f32_16x16x32
//   P^T = 2^(scale log2(e) S^T - m)         in the storage type
//   l += 1^T . P^T,  O^T[D x 16 SUB] += V^T . P^T
// A block with at most half (a quarter of) its rows has two (four) waves share
// each group of rows: they take the quarters in turn and meet at the end.
// P^T leaves the first product in the operand layout of the second; V^T comes
// through ds_read_b64_tr_b16.  m is a row's first maximum and moves only when the
// weights outgrow their types.  A second launch merges the chunks and the sink.
//
// Lane layouts (verified on gfx950): v_mfma_f32_16x16x32 -- lane l supplies
// A[l%16][k(l,i)], B[k(l,i)][l%16] for i < 8 and holds D[4(l/16)+i][l%16];
// ds_read_b64_tr_b16 -- within each 16-lane group, lane j receives element j%4
// of the 8-byte rows read by lanes j/4 + 4i, i < 4.
#include <algorithm>
#include <cmath>

#include "common.h"

namespace akv {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) u32x4 global_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHuge = 18446744073709551616.f;  // 2^64: a weight sum above it may have overflowed the product

// Keys of a tile: 32 KiB of K and V either way.
constexpr int keys_of(int d) { return d == 64 ? 128 : 64; }

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
  float* part_o;   // [chunks][tokens][q heads][D]
  float* part_ml;  // [chunks][tokens][q heads][2]
  int32_t* used;   // [tokens]: chunks of the token's request
  int64_t n_tokens, max_len;
  int32_t n_requests, q_heads, kv_heads, group, head_dim, mask_words, page_size;
  int32_t chunks, row_blocks, heads_last;
  bool indptr64, out_f32, paged;
};

// Workgroups that a batch's keys are shared out over: four per CU.
constexpr int64_t kTargetGroups = 4 * 256;

// Keys of a chunk for a request that reaches `span` of a batch's `total` keys.
template <int D>
__device__ __forceinline__ int64_t chunk_keys_of(const TreeArgs& a, int64_t span, int64_t total) {
  const int64_t reach = a.max_len * a.n_requests;
  if (total > reach) total = reach;
  const int64_t work = total * a.kv_heads * a.row_blocks;
  int64_t most = (work / kTargetGroups + keys_of(D) - 1) / keys_of(D) * keys_of(D);
  const int64_t least = (span + a.chunks - 1) / a.chunks;
  if (most < keys_of(D)) most = keys_of(D);
  if (most < least) most = (least + 63) / 64 * 64;
  const int64_t n = span > 0 ? (span + most - 1) / most : 1;
  return n > 1 ? ((span + n - 1) / n + 63) / 64 * 64 : most;
}

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

__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = uniform(static_cast<int32_t>(v)), hi = uniform(static_cast<int32_t>(v >> 32));
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

// Four dims of a token's head, normalised; a weight sum of 0: nothing was seen.
template <typename T>
__device__ __forceinline__ void store_row(const TreeArgs& a, int64_t token, int head, int d, f32x4 o, float l) {
  const int64_t at = token * a.o_st + head * a.o_sh + d;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = l == 0.f ? 0.f : o[i] / l;
    if (a.out_f32)
      static_cast<float*>(a.out)[at + i] = x;
    else
      static_cast<T*>(a.out)[at + i] = static_cast<T>(x);
  }
}

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

// Reads from a tile.  In asm, with their wait: the compiler takes every LDS read
// for one that may meet the rows streaming into the other buffer, and would wait
// for those first.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p));
}

// Two 16-byte chunks of the K row at either address, 16 rows apart by STRIDE.
template <int STRIDE>
__device__ __forceinline__ void read_k(uint32_t a0, uint32_t a1, u32x4 (&lo)[2], u32x4 (&hi)[2]) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %4 offset:%6\n\tds_read_b128 %3, %5 offset:%6\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(hi[0]), "=&v"(hi[1])
      : "v"(a0), "v"(a1), "i"(STRIDE)
      : "memory");
}

// Four transposed operands: 4 x 16 dims of 32 keys.
template <int STRIDE>
__device__ __forceinline__ void read_v(const uint32_t (&at)[4], s16x4 (&lo)[4], s16x4 (&hi)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "i"(STRIDE)
      : "memory");
}

__device__ __forceinline__ u32x4 read_16(uint32_t at) {
  u32x4 w;
  asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(w) : "v"(at) : "memory");
  return w;
}

template <int D>
struct TileLds {
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
  constexpr int kGroupRows = 16 * SUB;       // rows of a wave
  constexpr int R = kWaves * kGroupRows;     // rows of a block
  __shared__ __attribute__((aligned(256))) TileLds<D> buffers[2];
  __shared__ __attribute__((aligned(16))) uint32_t s_dead[2][4];  // keys of the buffers' quarters that no token sees
  __shared__ float s_m[kWaves][kGroupRows], s_l[kWaves][kGroupRows];
  __shared__ int32_t s_tok[kWaves][kGroupRows];  // the rows' tokens, for the masked quarters
  __shared__ int32_t s_odd;                      // V rows held infinities or NaN that some row does not see
  __shared__ uint64_t s_list[kWaves];            // and the keys that did
  static_assert(kWaves * kGroupRows * D * 4 <= sizeof(buffers), "the waves' results fit the tiles");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  // block id -> (unit, row block): a unit's row blocks lie 8 apart, on one XCD
  const uint32_t round = 8 * a.row_blocks;
  const uint32_t unit = blockIdx.x / round * 8 + blockIdx.x % 8;
  const int rb0 = blockIdx.x % round / 8;
  const uint32_t pair = unit / a.chunks;
  const int chunk = unit - pair * a.chunks;
  if (pair >= static_cast<uint32_t>(a.n_requests) * a.kv_heads) return;
  const int b = a.heads_last ? pair % a.n_requests : pair / a.kv_heads;
  const int g = a.heads_last ? pair / a.n_requests : pair % a.kv_heads;
  // in scalar registers: the loop has no vector register to spare
  int64_t q0 = uniform(load_index(a.qo_indptr, a.indptr64, b)), q1 = uniform(load_index(a.qo_indptr, a.indptr64, b + 1));
  const int64_t kv0 = uniform(load_index(a.kv_indptr, a.indptr64, b));
  const int64_t len64 = uniform(load_index(a.kv_indptr, a.indptr64, b + 1)) - kv0;
  const int64_t total = uniform(load_index(a.kv_indptr, a.indptr64, a.n_requests)) -
                        uniform(load_index(a.kv_indptr, a.indptr64, 0));
  if (gated(a.gate)) return;
  if (q0 < 0) q0 = 0;
  if (q1 > a.n_tokens) q1 = a.n_tokens;
  const int n = static_cast<int>(q1 > q0 ? q1 - q0 : 0);
  const int rows = n * a.group;
  if (rb0 * R >= rows) return;
  const int len = static_cast<int>(len64 > 0 ? len64 : 0);
  const int old = len > n ? len - n : 0;
  // the keys that some token of the request sees begin here
  int lo = 0, hi_start = 0;
  if (a.key_starts) {
    lo = old;
    for (int i = lane; i < n; i += 64) {
      const int s = min(max(a.key_starts[q0 + i], 0), old);
      lo = min(lo, s);
      hi_start = max(hi_start, s);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      lo = min(lo, __shfl_xor(lo, off));
      hi_start = max(hi_start, __shfl_xor(hi_start, off));
    }
    lo = uniform(lo);
    hi_start = uniform(hi_start);
  }
  const int span = len - lo;
  const int64_t chunk_keys = uniform(chunk_keys_of<D>(a, span, total));
  const int used = span > 0 ? uniform(static_cast<int32_t>((span + chunk_keys - 1) / chunk_keys)) : 1;
  if (chunk >= used) return;
  const int begin = lo + static_cast<int>(chunk * chunk_keys);
  const int end = static_cast<int>(std::min<int64_t>(begin + chunk_keys, len));
  const int tiles = (end - begin + kKeys - 1) / kKeys;
  if (chunk == 0 && g == 0 && rb0 == 0)
    for (int i = threadIdx.x; i < n; i += kThreads) a.used[q0 + i] = used;

  // (an empty pool holds no key: every slot is a hole, and zeros are read)
  const bool pool = a.pool_slots > 0;
  const char* kbase = pool ? a.k + g * a.k_sh : reinterpret_cast<const char*>(zero_row);
  const char* vbase = pool ? a.v + g * a.v_sh : reinterpret_cast<const char*>(zero_row);
  const int64_t k_ss = pool ? a.k_ss : 0, v_ss = pool ? a.v_ss : 0;
  const int32_t* list = a.kv_indices + (a.paged ? b * a.table_stride : kv0);
  // entries of the list that exist
  const int64_t left = a.paged ? a.table_width : a.table_width - kv0;
  const int32_t width = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(left, 0), 0x7fffffff));
  const uint32_t dead_at = lds_address(s_dead), tile_at = lds_address(buffers);
  const int my_key = kWaveKeys * wave + (lane & (kWaveKeys - 1));  // of a tile
  // the list entry of this lane's key of tile it (past the end: the last key's),
  // one tile ahead; what it means is worked out when the tile is asked for
  auto fetch = [&](int it) -> int32_t {
    const uint32_t j = min(begin + it * kKeys + my_key, end - 1);
    const int32_t at = a.paged ? j / static_cast<uint32_t>(a.page_size) : j;
    return width > 0 ? list[min(at, width - 1)] : -1;
  };
  // a wave's keys of a tile, straight into LDS: lane l of a load fills bytes
  // 16 l of a 1 KiB block, chunk position l % kChunks of a row
  auto stage = [&](int it, int32_t entry) {
    TileLds<D>& t = buffers[it & 1];
    const uint32_t key = begin + it * kKeys + my_key, j = min(key, static_cast<uint32_t>(end - 1));
    uint32_t at = j, off = 0, per = 1;
    if (a.paged) {
      per = a.page_size;
      at = j / per;
      off = j - at * per;
    }
    const uint64_t slot64 = static_cast<uint64_t>(static_cast<uint32_t>(entry)) * per + off;
    const bool there = entry >= 0 && at < static_cast<uint32_t>(width) && slot64 < static_cast<uint64_t>(a.pool_slots);
    // a hole reads slot 0; the mask keeps it from every row
    const uint32_t slot = there ? static_cast<uint32_t>(slot64) : 0;
    const uint32_t dead = static_cast<uint32_t>(
        __builtin_amdgcn_ballot_w64(!there || key >= static_cast<uint32_t>(end)));
    if (lane == 0) {
      if constexpr (kWaveKeys == 32)
        asm volatile("ds_write_b32 %0, %1" ::"v"(dead_at + 16 * (it & 1) + 4 * wave), "v"(dead) : "memory");
      else
        asm volatile("ds_write_b16 %0, %1" ::"v"(dead_at + 16 * (it & 1) + 2 * wave), "v"(dead) : "memory");
    }
#pragma unroll
    for (int u = 0; u < kWaveKeys / kLoadRows; ++u) {
      const int mine = u * kLoadRows + lane / kChunks, r = kWaveKeys * wave + mine;
      const uint64_t from = __shfl(slot, mine);
      const int ck = (lane % kChunks) ^ swz_k<D>(r), cv = (lane % kChunks) ^ swz_v<D>(r);
      const char* krow = kbase + from * k_ss + 16 * ck;
      const char* vrow = vbase + from * v_ss + 16 * cv;
      if (NARROW) {  // dims past head_dim read zeros
        krow = 8 * ck < a.head_dim ? krow : reinterpret_cast<const char*>(zero_row);
        vrow = 8 * cv < a.head_dim ? vrow : reinterpret_cast<const char*>(zero_row);
      }
      const int place = (kWaveKeys * wave + u * kLoadRows) * D * 2;
      __builtin_amdgcn_global_load_lds(krow, (lds_void*)(t.k + place), 16, 0, 0);
      __builtin_amdgcn_global_load_lds(vrow, (lds_void*)(t.v + place), 16, 0, 0);
    }
  };

  for (int rb = rb0; rb * R < rows; rb += a.row_blocks) {
    int32_t entry = tiles > 0 ? fetch(0) : -1;
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
      s_tok[wave][16 * s + col] = tok;
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
    f32x4 acc[SUB][kDTiles], lacc[SUB];  // l: four equal copies; 0 while the row has seen no key
    float neg_m[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      neg_m[s] = 0.f;
      lacc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < kDTiles; ++t) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool unset = true;  // some row of the wave has seen no key yet
    x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.f);

    // what a token sees of the 32 keys from k0 on
    auto visible = [&](int tok, int k0) -> uint32_t {
      const int base = k0 - old;
      uint64_t bits = ~0ull;
      if (base > -32) {
        auto word = [&](int w) -> uint64_t {
          if (a.mask) return w < a.mask_words ? a.mask[(q0 + tok) * a.mask_stride + w] : 0;
          const int i = tok - 64 * w;
          return i >= 63 ? ~0ull : i < 0 ? 0 : (2ull << i) - 1;
        };
        if (base < 0) {
          bits = word(0) << -base | ((1ull << -base) - 1);
        } else {
          const int w = base >> 6, by = base & 63;
          bits = word(w) >> by;
          if (by > 32) bits |= word(w + 1) << (64 - by);
        }
      }
      if (a.key_starts) {
        const int hidden = min(max(a.key_starts[q0 + tok], 0), old) - k0;
        if (hidden >= 32) bits = 0; else if (hidden > 0) bits &= ~0ull << hidden;
      }
      return static_cast<uint32_t>(bits);
    };
    // A weight of 0 does not hide an infinity or NaN from the product.  Where
    // rows see different keys such values are cleared (by every wave that uses
    // them) and the block takes note: its rows get them back at the end.
    auto clear_odd = [&](uint32_t at, uint32_t dead) {
      bool noted = false;
#pragma nounroll
      for (int i = 0; i < kDTiles; ++i) {
        const uint32_t here = at + 1024 * i + 16 * lane;
        s16x8 w = __builtin_bit_cast(s16x8, read_16(here));
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool one = not_finite<T>(w[e]);
          odd |= one;
          w[e] = one ? 0 : w[e];
        }
        if (odd) asm volatile("ds_write_b128 %0, %1" ::"v"(here), "v"(w) : "memory");
        noted |= odd && !(dead >> ((64 * i + lane) / kChunks) & 1);
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): cleared before they are read
      if (__builtin_amdgcn_ballot_w64(noted) && lane == 0)
        asm volatile("ds_write_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" ::"v"(lds_address(&s_odd)), "v"(1) : "memory");
    };
    // this lane's operand addresses in quarter 0: K chunks quad of row col, and
    // the source of its transposed V reads (row 4 quad + col / 4, dims 4 (col % 4))
    const uint32_t k_at = col * D * 2 + 16 * (quad ^ swz_k<D>(col));
    const int vr = 4 * quad + (col >> 2);
    const uint32_t v_at = kKeys * D * 2 + vr * D * 2 + 16 * ((col >> 1 & 1) ^ swz_v<D>(vr)) + 8 * (col & 1);
    // 32 keys, from row 32 kk of a tile on; k0: the first one's rank
    auto quarter = [&](uint32_t at, int k0, uint32_t dead) {
      const bool masked = dead != 0 || k0 + 32 > old || k0 < hi_start;
      f32x4 sc[2][SUB];
#pragma unroll
      for (int h = 0; h < kSteps / 2; ++h) {
        // k-steps 2 h and 2 h + 1: chunks 4 and 8 on (the swizzle is an xor)
        u32x4 lo[2], hi[2];
        read_k<16 * D * 2>((at + k_at) ^ (128 * h), (at + k_at) ^ (128 * h + 64), lo, hi);
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            sc[0][s] = product(__builtin_bit_cast(x8, lo[st]), qop[s][2 * h + st],
                               h + st == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[0][s]);
            sc[1][s] = product(__builtin_bit_cast(x8, hi[st]), qop[s][2 * h + st],
                               h + st == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[1][s]);
          }
      }
      if (masked) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          const uint32_t seen = visible(s_tok[wave][16 * s + col], k0) & ~dead;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[j][s][i] = seen >> (16 * j + 4 * quad + i) & 1 ? sc[j][s][i] : -INFINITY;
        }
      }
      // A row's m is its maximum over the first quarter it sees a key of, and then
      // stays put: the sum tells when it should not have.  A sum past kHuge (a
      // score ~64 above m in the log2 domain, 16 in fp16, whose weight is then
      // infinite) takes the quarter again with exact maxima.
      x8 p[SUB];
      float before[SUB];
#pragma unroll
      for (int s = 0; s < SUB; ++s) before[s] = lacc[s][0];
      for (bool exact = unset;; exact = true) {
        if (exact) {
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            const float m0 = max3(sc[0][s][0], sc[0][s][1], sc[0][s][2]);
            const float m1 = max3(sc[0][s][3], sc[1][s][0], sc[1][s][1]);
            const float mx = column_max(max3(m0, m1, max2(sc[1][s][2], sc[1][s][3])));
            const float over = fmaf(mx, a.scale_log2, neg_m[s]);  // above m
            const bool any = before[s] != 0.f;
            const bool move = any ? over > 0.f : mx > -INFINITY;
            const float alpha = move && any ? __builtin_amdgcn_exp2f(-over) : 1.f;
            before[s] *= alpha;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) acc[s][dt] *= alpha;
            neg_m[s] = move ? -(mx * a.scale_log2) : neg_m[s];
            lacc[s] = f32x4{before[s], before[s], before[s], before[s]};
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
          lacc[s] = product(ones, p[s], lacc[s]);
        }
#pragma unroll
        for (int s = 0; s < SUB; ++s) huge |= lacc[s][0] > kHuge;
        if (exact || !__builtin_amdgcn_ballot_w64(huge)) break;
      }
      if (unset) {
        bool none = false;
#pragma unroll
        for (int s = 0; s < SUB; ++s) none |= lacc[s][0] == 0.f;
        unset = __builtin_amdgcn_ballot_w64(none) != 0;
      }
      // transposing reads: lane col of group quad receives V[key][16 dt + col]
      // for keys 4 quad + i (i < 4) of the quarter, then 16 keys on; dt = 4 h + e
      auto v_operands = [&](int h, x8 (&v)[4]) {
        uint32_t from[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) from[e] = (at + v_at) ^ (32 * (4 * h + e));
        s16x4 lo[4], hi[4];
        read_v<16 * D * 2>(from, lo, hi);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = __builtin_bit_cast(x8, __builtin_shufflevector(lo[e], hi[e], 0, 1, 2, 3, 4, 5, 6, 7));
      };
      if (masked) clear_odd(at + kKeys * D * 2, dead);
#pragma unroll
      for (int h = 0; h < kDTiles / 4; ++h) {
        x8 v[4];
        v_operands(h, v);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int s = 0; s < SUB; ++s) acc[s][4 * h + e] = product(v[e], p[s], acc[s][4 * h + e]);
      }
    };
    if (tiles > 0) {
      stage(0, entry);
      if (tiles > 1) entry = fetch(1);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    // tile it from one buffer while tile it + 1 streams into the other
#pragma nounroll
    for (int it = 0; it < tiles; ++it) {
      const int buf = it & 1;
      if (it + 1 < tiles) {
        stage(it + 1, entry);
        if (it + 2 < tiles) entry = fetch(it + 2);
      }
      const int t0 = begin + it * kKeys;
      const uint32_t cur = tile_at + buf * static_cast<uint32_t>(sizeof(TileLds<D>));
      const u32x4 dead = read_16(dead_at + 16 * buf);
#pragma nounroll
      for (int kk = share; kk < kQuarters; kk += sharers) {
        const int k0 = t0 + 32 * kk;
        if (k0 >= end) break;
        const uint32_t word = kk == 0 ? dead[0] : kk == 1 ? dead[1] : kk == 2 ? dead[2] : dead[3];
        quarter(cur + kk * 64 * D, k0, __builtin_amdgcn_readfirstlane(word));
      }
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }

    // the waves' O rows [row][dim] over the tiles, four-float groups turned by
    // the row for the banks; the sharers of a group meet there
    auto result_of = [&](int w) -> float* {
      return reinterpret_cast<float*>(&buffers[0]) + w * kGroupRows * D;
    };
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int r = 16 * s + col;
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt)
        *reinterpret_cast<f32x4*>(result_of(wave) + r * D + ((16 * dt + 4 * quad) ^ (col & 7) << 2)) = acc[s][dt];
      if (quad == 0) {
        s_m[wave][r] = lacc[s][0] == 0.f ? -INFINITY : -neg_m[s];
        s_l[wave][r] = lacc[s][0];
      }
    }
    __syncthreads();
    const int here = min(rows - rb * R, groups * kGroupRows);
    for (int u = threadIdx.x; u < here * (D / 4); u += kThreads) {
      const int r = u / (D / 4), d = 4 * (u % (D / 4));
      if (NARROW && d >= a.head_dim) continue;
      const int token = (rb * R + r) / a.group, head = g * a.group + rb * R + r - token * a.group;
      const int group = r / kGroupRows, in = r % kGroupRows;
      float m = -INFINITY, l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      for (int w = group; w < kWaves; w += groups) m = fmaxf(m, s_m[w][in]);
      // a wave that has seen no key carries m = -inf, l = 0 and O = 0
      const float base = m == -INFINITY ? 0.f : m;
      for (int w = group; w < kWaves; w += groups) {
        const float by = __builtin_amdgcn_exp2f(s_m[w][in] - base);
        l += s_l[w][in] * by;
        o += *reinterpret_cast<const f32x4*>(result_of(w) + in * D + (d ^ (in & 7) << 2)) * by;
      }
      if (used > 1) {
        const int64_t at = (static_cast<int64_t>(chunk) * a.n_tokens + q0 + token) * a.q_heads + head;
        *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = o;
        if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * at) = f32x2{m, l};
        continue;
      }
      if (a.sinks) {
        const float sink = a.sinks[head] * kLog2e;
        const float mt = fmaxf(m, sink);
        const float by = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mt);
        o *= by;
        l = l * by + (mt == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - mt));
      }
      store_row<T>(a, q0 + token, head, d, o, l);
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
        const int mine = base + static_cast<int>(threadIdx.x);
        const T* row = mine < end ? v_row(mine) : nullptr;
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
              if (!(visible(token, j) & 1)) continue;
              const T* v = v_row(j) + d;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (!not_finite<T>(__builtin_bit_cast(short, v[i]))) continue;
                const float x = static_cast<float>(v[i]);
                if (used > 1) {
                  a.part_o[((static_cast<int64_t>(chunk) * a.n_tokens + q0 + token) * a.q_heads + head) * D + d + i] += x;
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
  }
}

// Merges a row's chunks and the sink: a wave per (token, head).  Lane c takes
// chunk c's maximum and sum; then D / 4 lanes each take the chunks in turn, four
// dims a lane.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeArgs a) {
  constexpr int kLanes = D / 4, kWays = 64 / kLanes, kAhead = 4;
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + uniform(static_cast<int32_t>(threadIdx.x >> 6));
  const int64_t token = row / a.q_heads;
  const int head = static_cast<int>(row - token * a.q_heads);
  if (token >= a.n_tokens || token >= load_index(a.qo_indptr, a.indptr64, a.n_requests) ||
      token < load_index(a.qo_indptr, a.indptr64, 0))
    return;
  if (gated(a.gate)) return;
  const int used = uniform(a.used[token]);
  if (used <= 1) return;
  const int64_t step = a.n_tokens * a.q_heads;
  const f32x2* ml = reinterpret_cast<const f32x2*>(a.part_ml) + row;
  const int d = 4 * (lane % kLanes), way = lane / kLanes;
  const float* from = a.part_o + row * D + d;
  const float sink = a.sinks ? a.sinks[head] * kLog2e : -INFINITY;
  float m = sink;
  for (int c = lane; c < used; c += 64) m = fmaxf(m, ml[c * step].x);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off));
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < used; c0 += 64) {
    f32x2 mine = {-INFINITY, 0.f};
    if (c0 + lane < used) mine = ml[(c0 + lane) * step];
    const float w = __builtin_amdgcn_exp2f(mine.x - base);
    l += mine.y * w;
    const int count = used - c0 < 64 ? used - c0 : 64;
    for (int c = 0; c < count; c += kWays * kAhead) {
      f32x4 x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int at = c + i * kWays + way;
        x[i] = *reinterpret_cast<const f32x4*>(from + (c0 + (at < count ? at : 0)) * step * D);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int at = c + i * kWays + way;
        const float by = __shfl(w, at & 63);
        if (at < count) o += x[i] * by;
      }
    }
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) l += __shfl_xor(l, off);
#pragma unroll
  for (int off = kLanes; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], off);
  if (a.sinks && m != -INFINITY) l += __builtin_amdgcn_exp2f(sink - base);
  if (way == 0 && d < a.head_dim) store_row<T>(a, token, head, d, o, l);
}

int tile_dim(int32_t head_dim) { return head_dim <= 64 ? 64 : 128; }

// A wave's row subtiles for requests of up to `rows` rows: as many as the rows
// fill, since waves that share rows read every key once.
int subtiles_for(int d, int64_t rows) {
  const int most = d == 64 ? 4 : 2;
  int sub = 1;
  while (sub < most && rows > 16 * sub) sub *= 2;
  return sub;
}

struct Launch {
  int d, sub;
  int32_t row_blocks, chunks;
};

Launch plan(int64_t n_tokens, int64_t n_requests, int64_t kv_heads, int64_t group, int32_t head_dim, int64_t max_len,
            int64_t max_new) {
  Launch p;
  p.d = tile_dim(head_dim);
  const int64_t rows = std::max<int64_t>(1, std::min(max_new, n_tokens)) * group;
  p.sub = subtiles_for(p.d, rows);
  const int64_t block = 16 * kWaves * p.sub, pass = keys_of(p.d);
  p.row_blocks = static_cast<int32_t>(std::min<int64_t>((rows + block - 1) / block, 4096));
  // chunks: as many as give every CU its share of a batch whose requests all
  // have max_len keys, four times as many for a few long ones among short ones
  const int64_t keys = std::max<int64_t>(pass, n_requests * max_len * kv_heads * p.row_blocks / kTargetGroups);
  int64_t chunks = std::min((max_len + pass - 1) / pass, 4 * ((max_len + keys - 1) / keys));
  chunks = std::max<int64_t>(1, std::min<int64_t>(chunks, 4096));
  // odd, so that the first chunks of the pairs go round all XCDs
  p.chunks = static_cast<int32_t>(chunks > 1 ? chunks | 1 : 1);
  return p;
}

int64_t partial_bytes(const Launch& p, int64_t n_tokens, int64_t q_heads) {
  const int64_t rows = p.chunks > 1 ? p.chunks * n_tokens * q_heads : 0;
  return rows * (p.d + 2) * 4 + (n_tokens + 3) / 4 * 16;
}

template <typename T, int D, int SUB>
void start(const TreeArgs& a, dim3 grid, hipStream_t st) {
  if (a.head_dim < D)
    hipLaunchKernelGGL((tree_attention_kernel<T, D, SUB, true>), grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((tree_attention_kernel<T, D, SUB, false>), grid, dim3(kThreads), 0, st, a);
}

template <typename T>
int launch(const TreeArgs& a, const Launch& p, hipStream_t st) {
  const int64_t units = static_cast<int64_t>(a.n_requests) * a.kv_heads * a.chunks;
  const int64_t blocks = (units + 7) / 8 * 8 * a.row_blocks;
  if (blocks > 0x7fffffffLL) return fail(AKV_EINVAL, "akv_tree_attention: batch too large");
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
  if (rc || a.chunks == 1) return rc;
  const dim3 merge(static_cast<unsigned>((a.n_tokens * a.q_heads + 3) / 4));
  if (p.d == 64)
    hipLaunchKernelGGL((tree_combine_kernel<T, 64>), merge, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((tree_combine_kernel<T, 128>), merge, dim3(256), 0, st, a);
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
  return partial_bytes(plan(n_tokens, n_requests, kv_heads, q_heads / kv_heads, head_dim, max_len, max_new), n_tokens,
                       q_heads);
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
  if (!q || !k_buffer || !v_buffer || !qo_indptr || !kv_indptr || !kv_indices || !out || !workspace)
    return fail(AKV_EINVAL, "akv_tree_attention: null device pointer");
  if ((q_stride_t | q_stride_h | k_stride_slot | k_stride_head | v_stride_slot | v_stride_head) % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_buffer) |
        reinterpret_cast<uintptr_t>(v_buffer) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0)
    return fail(AKV_EINVAL, "akv_tree_attention: q, K and V rows and the workspace must be 16-byte aligned");
  if (pool_slots > 0xffffffffLL || n_tokens > 0x7fffffffLL / q_heads || static_cast<int64_t>(n_requests) * kv_heads > 0x7fffffffLL / 4096)
    return fail(AKV_EINVAL, "akv_tree_attention: batch too large");
  const Launch p = plan(n_tokens, n_requests, kv_heads, q_heads / kv_heads, head_dim, max_len, max_new);
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
  a.used = static_cast<int32_t*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + (n_tokens + 3) / 4 * 16);
  a.part_ml = a.part_o + static_cast<int64_t>(p.chunks) * n_tokens * q_heads * p.d;
  a.n_tokens = n_tokens;
  a.max_len = max_len;
  a.n_requests = n_requests;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.chunks = p.chunks;
  a.row_blocks = p.row_blocks;
  a.heads_last = p.chunks < 8;
  a.indptr64 = indptr_dtype == AKV_I64;
  a.out_f32 = out_dtype == AKV_F32;
  a.paged = table_stride != 0;
  hipStream_t st = as_stream(stream);
  if (dtype == AKV_F16) return launch<_Float16>(a, p, st);
  return launch<__bf16>(a, p, st);
}
