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
// that head's keys, so K and V are read once for R = 16 SUB rows, and again for
// every further R.  Workgroup = (chunk of keys, KV head, request, block of R
// rows) of four waves; all hold the same rows and take the keys in turn, KEYS
// at a time: K straight into registers in the operand layout, V into the
// wave's own LDS tile, both asked for one pass ahead.  No barrier until the
// waves meet at the end.
//   S^T[KEYS x 16 SUB] = K . Q^T            v_mfma_f32_16x16x32
//   P^T = 2^(scale log2(e) S^T - m)         in the storage type
//   l += 1^T . P^T,  O^T[D x 16 SUB] += V^T . P^T
// P^T leaves the first product in the operand layout of the second; V^T comes
// through ds_read_b64_tr_b16.  m follows a row's maximum when that exceeds it
// by more than 2^8.  A second launch merges the chunks and the sink.
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
constexpr float kSlack = 8.f;  // log2-domain excess at which a row's maximum moves

// Keys of a wave's pass: 32 K registers and an 8 KiB V tile either way.
constexpr int keys_of(int d) { return d == 64 ? 64 : 32; }
constexpr int pass_of(int d) { return kWaves * keys_of(d); }

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
  int64_t most = (work / kTargetGroups + pass_of(D) - 1) / pass_of(D) * pass_of(D);
  const int64_t least = (span + a.chunks - 1) / a.chunks;
  if (most < pass_of(D)) most = pass_of(D);
  if (most < least) most = (least + 63) / 64 * 64;
  const int64_t n = span > 0 ? (span + most - 1) / most : 1;
  return n > 1 ? ((span + n - 1) / n + 63) / 64 * 64 : most;
}

static __device__ __attribute__((aligned(16))) const uint32_t zero_row[64] = {};

// 16-byte chunk c of V row r sits at chunk c ^ swz(r) of its LDS row.
template <int D>
__device__ __forceinline__ int swz(int r) { return D == 64 ? r & 6 : (r & 7) << 1; }

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

// Whether any of the eight 16-bit values of a word is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(u32x4 w) {
  constexpr uint32_t e = sizeof(T) == 2 && __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & e) == e || (w[i] >> 16 & e) == e;
  return bad;
}

// Maximum over the lanes col, col + 16, col + 32, col + 48 of a column.
__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}

template <int D>
struct WaveTile {
  char rows[kWaves][keys_of(D) * D * 2];
};

// D: 64 or 128, the tile's head width (head_dim <= D).  SUB: row subtiles of 16.
template <typename T, int D, int SUB>
__global__ void __launch_bounds__(kThreads, 2) tree_attention_kernel(const TreeArgs a) {
  using x4 = typename Vec<T>::x4;
  using x8 = typename Vec<T>::x8;
  constexpr int kKeys = keys_of(D), kPass = pass_of(D);
  constexpr int kTiles = kKeys / 16;
  constexpr int kSteps = D / 32;
  constexpr int kDTiles = D / 16;
  constexpr int kChunks = D / 8;       // 16-byte chunks of a row
  constexpr int kVRows = 64 / kChunks;  // V rows of one wave-wide load
  constexpr int R = 16 * SUB;
  __shared__ __attribute__((aligned(16))) WaveTile<D> tile0;
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  static_assert(16 * D * 4 <= kKeys * D * 2, "a subtile's results fit a wave's tile");

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
  int64_t q0 = load_index(a.qo_indptr, a.indptr64, b), q1 = load_index(a.qo_indptr, a.indptr64, b + 1);
  const int64_t kv0 = load_index(a.kv_indptr, a.indptr64, b);
  int64_t len64 = load_index(a.kv_indptr, a.indptr64, b + 1) - kv0;
  const int64_t total = load_index(a.kv_indptr, a.indptr64, a.n_requests) - load_index(a.kv_indptr, a.indptr64, 0);
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
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi_start = __builtin_amdgcn_readfirstlane(hi_start);
  }
  const int span = len - lo;
  const int64_t chunk_keys = chunk_keys_of<D>(a, span, total);
  const int used = span > 0 ? static_cast<int>((span + chunk_keys - 1) / chunk_keys) : 1;
  if (chunk >= used) return;
  const int begin = lo + static_cast<int>(chunk * chunk_keys);
  const int end = static_cast<int>(std::min<int64_t>(begin + chunk_keys, len));
  if (chunk == 0 && g == 0 && rb0 == 0)
    for (int i = threadIdx.x; i < n; i += kThreads) a.used[q0 + i] = used;

  const char* kbase = a.k + g * a.k_sh;
  const char* vbase = a.v + g * a.v_sh;
  const int32_t* list = a.kv_indices + (a.paged ? b * a.table_stride : kv0);
  // entries of the list that exist
  const int64_t width = a.paged ? a.table_width : a.table_width - kv0;
  // the slot of key j, or -1: past the chunk, or a hole
  auto slot_at = [&](int j) -> int64_t {
    if (j >= end) return -1;
    int64_t at = j, off = 0;
    if (a.paged) {
      const uint32_t page = a.page_size;
      at = static_cast<uint32_t>(j) / page;
      off = static_cast<uint32_t>(j) - static_cast<uint32_t>(at) * page;
    }
    if (at >= width) return -1;
    const int64_t entry = list[at];
    const int64_t slot = a.paged ? entry * a.page_size + off : entry;
    return entry >= 0 && slot < a.pool_slots ? slot : -1;
  };

  for (int rb = rb0; rb * R < rows; rb += a.row_blocks) {
    // this lane's rows: r = R rb + 16 s + col, token r / G, head g G + r % G
    // (rows past the last repeat it and are never stored)
    int tok[SUB];
    x8 qop[SUB][kSteps];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int r = min(rb * R + 16 * s + col, rows - 1);
      tok[s] = r / a.group;
      const T* row = static_cast<const T*>(a.q) + (q0 + tok[s]) * a.q_st +
                     static_cast<int64_t>(g * a.group + r - tok[s] * a.group) * a.q_sh;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        u32x4 w = {0u, 0u, 0u, 0u};
        const int c = 4 * st + quad;
        if (8 * c < a.head_dim) w = *((const global_u32x4*)row + c);
        qop[s][st] = __builtin_bit_cast(x8, w);
      }
    }
    f32x4 acc[SUB][kDTiles], lacc[SUB];
    float neg_m[SUB];  // -m; 0 while the row has seen no finite score
    bool seen[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      neg_m[s] = 0.f;
      seen[s] = false;
      lacc[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < kDTiles; ++t) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    x8 ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = static_cast<T>(1.f);

    u32x4 k[kTiles][kSteps];
    uint64_t dead = 0;  // keys of the pass in k that no token sees
    auto ask = [&](int64_t slot, WaveTile<D>& to) {
      dead = __builtin_amdgcn_ballot_w64(slot < 0);
#pragma unroll
      for (int j = 0; j < kTiles; ++j) {
        const int64_t at = __shfl(slot, 16 * j + col);
        const char* row = at < 0 ? reinterpret_cast<const char*>(zero_row) : kbase + at * a.k_ss;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const int c = 4 * st + quad;
          k[j][st] = u32x4{0u, 0u, 0u, 0u};
          if (8 * c < a.head_dim) k[j][st] = *((const global_u32x4*)row + c);
        }
      }
#pragma unroll
      for (int u = 0; u < kKeys / kVRows; ++u) {
        const int r = u * kVRows + lane / kChunks;
        int c = (lane % kChunks) ^ swz<D>(r);
        // dims past head_dim are never stored: any finite or other value will do
        if (8 * c >= a.head_dim) c = 0;
        const int64_t at = __shfl(slot, r);
        const char* row = at < 0 ? reinterpret_cast<const char*>(zero_row) : vbase + at * a.v_ss;
        __builtin_amdgcn_global_load_lds(row + 16 * c, (lds_void*)(to.rows[wave] + u * kVRows * D * 2), 16, 0, 0);
      }
    };
    // what row s sees of the 64 keys from t0 on, given the keys that are there
    auto visible = [&](int s, int t0, uint64_t there) -> uint64_t {
      const int base = t0 - old;
      uint64_t bits = ~0ull;
      if (base > -64) {
        auto word = [&](int w) -> uint64_t {
          if (a.mask) return w < a.mask_words ? a.mask[(q0 + tok[s]) * a.mask_stride + w] : 0;
          const int i = tok[s] - 64 * w;
          return i >= 63 ? ~0ull : i < 0 ? 0 : (2ull << i) - 1;
        };
        if (base < 0) {
          bits = word(0) << -base | ((1ull << -base) - 1);
        } else {
          const int w = base >> 6, by = base & 63;
          bits = word(w) >> by;
          if (by) bits |= word(w + 1) << (64 - by);
        }
      }
      if (a.key_starts) {
        const int hidden = min(max(a.key_starts[q0 + tok[s]], 0), old) - t0;
        if (hidden >= 64) bits = 0; else if (hidden > 0) bits &= ~0ull << hidden;
      }
      return bits & there;
    };
    auto step = [&](int t0, WaveTile<D>& cur) {
      T* vt = reinterpret_cast<T*>(cur.rows[wave]);
      const bool masked = dead != 0 || t0 + kKeys > old || t0 < hi_start;
      uint64_t seen_bits[SUB];
      x8 p[SUB][kTiles / 2];
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        f32x4 sc[kTiles];
#pragma unroll
        for (int j = 0; j < kTiles; ++j) {
          sc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < kSteps; ++st) sc[j] = product(__builtin_bit_cast(x8, k[j][st]), qop[s][st], sc[j]);
        }
        if (masked) {
          seen_bits[s] = visible(s, t0, ~dead);
#pragma unroll
          for (int j = 0; j < kTiles; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[j][i] = seen_bits[s] >> (16 * j + 4 * quad + i) & 1 ? sc[j][i] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[j][i]);
        top = column_max(top);
        const float over = fmaf(top, a.scale_log2, neg_m[s]);  // above m
        const bool move = seen[s] ? over > kSlack : top > -INFINITY;
        if (__builtin_amdgcn_ballot_w64(move)) {
          const float alpha = move && seen[s] ? __builtin_amdgcn_exp2f(-over) : 1.f;
          lacc[s] *= alpha;
#pragma unroll
          for (int t = 0; t < kDTiles; ++t) acc[s][t] *= alpha;
          neg_m[s] = move ? -(top * a.scale_log2) : neg_m[s];
          seen[s] |= move;
        }
#pragma unroll
        for (int jj = 0; jj < kTiles / 2; ++jj) {
          f32x4 e0, e1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e0[i] = __builtin_amdgcn_exp2f(fmaf(sc[2 * jj][i], a.scale_log2, neg_m[s]));
            e1[i] = __builtin_amdgcn_exp2f(fmaf(sc[2 * jj + 1][i], a.scale_log2, neg_m[s]));
          }
          const x4 p0 = __builtin_convertvector(e0, x4), p1 = __builtin_convertvector(e1, x4);
          p[s][jj] = __builtin_shufflevector(p0, p1, 0, 1, 2, 3, 4, 5, 6, 7);
          lacc[s] = product(ones, p[s][jj], lacc[s]);
        }
      }
      // transposing read: lane col of group quad receives V[key][16 t + col]
      // for keys 32 jj + 4 quad + i (i < 4), then 16 keys on
      auto v_operand = [&](int jj, int t) -> x8 {
        const int r0 = 32 * jj + 4 * quad + (col >> 2), r1 = r0 + 16;
        const int c = 2 * t + ((col & 3) >> 1), h = 4 * (col & 1);
        const s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + r0 * D + 8 * (c ^ swz<D>(r0)) + h));
        const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vt + r1 * D + 8 * (c ^ swz<D>(r1)) + h));
        return __builtin_bit_cast(x8, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
      };
      if (masked) {
        // A weight of 0 does not hide an infinity or NaN: such V rows are added
        // key by key to the rows that see them, and cleared for the product.
        constexpr int kShare = 64 / kKeys;  // lanes per key
        const int key = lane / kShare;
        lds_u32x4* row = (lds_u32x4*)(vt + key * D);
        bool bad = false;
#pragma unroll
        for (int c = 0; c < kChunks / kShare; ++c) {
          const int cc = c + lane % kShare * (kChunks / kShare);
          if (8 * cc < a.head_dim) bad |= not_finite<T>(row[cc ^ swz<D>(key)]);
        }
        if (kShare == 2) bad |= __shfl_xor(static_cast<int>(bad), 1) != 0;
        for (uint64_t rest = __builtin_amdgcn_ballot_w64(bad); rest;) {
          const int kk = __builtin_ctzll(rest) / kShare;
          rest &= ~(((1ull << kShare) - 1) << (kk * kShare));
          const int jj = kk >> 5, mine = kk & 31;
#pragma unroll
          for (int t = 0; t < kDTiles; ++t) {
            x8 v1 = v_operand(jj, t);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (4 * quad + (i & 3) + 16 * (i >> 2) != mine) v1[i] = static_cast<T>(0.f);
#pragma unroll
            for (int s = 0; s < SUB; ++s) {
              const x8 pj = kTiles == 4 && jj ? p[s][kTiles / 2 - 1] : p[s][0];
              const f32x4 add = product(v1, pj, f32x4{0.f, 0.f, 0.f, 0.f});
              if (seen_bits[s] >> kk & 1) acc[s][t] += add;
            }
          }
        }
        if (bad) {
#pragma unroll
          for (int c = 0; c < kChunks / kShare; ++c)
            row[(c + lane % kShare * (kChunks / kShare)) ^ swz<D>(key)] = u32x4{0u, 0u, 0u, 0u};
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // the clears are in LDS before the reads below
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int jj = 0; jj < kTiles / 2; ++jj)
#pragma unroll
        for (int t = 0; t < kDTiles; ++t) {
          const x8 vop = v_operand(jj, t);
#pragma unroll
          for (int s = 0; s < SUB; ++s) acc[s][t] = product(vop, p[s][jj], acc[s][t]);
        }
      // this tile's reads are done before its place is filled again
      __builtin_amdgcn_s_waitcnt(0xc07f);
      asm volatile("" ::: "memory");
    };
    for (int t0 = begin + wave * kKeys; t0 < end; t0 += kPass) {
      ask(slot_at(t0 + lane % kKeys), tile0);
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      step(t0, tile0);
    }

    // the waves meet, 16 rows at a time: O rows [row][dim] over their V tiles,
    // four-float groups turned by the row for the banks
    float* om = reinterpret_cast<float*>(tile0.rows[wave]);
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < kDTiles; ++t)
        *reinterpret_cast<f32x4*>(om + col * D + ((16 * t + 4 * quad) ^ (col & 7) << 2)) = acc[s][t];
      if (quad == 0) {
        s_m[wave][col] = seen[s] ? -neg_m[s] : -INFINITY;
        s_l[wave][col] = lacc[s][0];
      }
      __syncthreads();
      for (int u = threadIdx.x; u < 16 * (D / 4); u += kThreads) {
        const int row = u / (D / 4), d = 4 * (u % (D / 4));
        const int r = rb * R + 16 * s + row;
        if (r >= rows || d >= a.head_dim) continue;
        const int token = r / a.group, head = g * a.group + r - token * a.group;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_m[w][row]);
        // a wave without a finite score carries m = -inf, and O = l = 0 or NaN
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float mw = s_m[w][row];
          const float sw = mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mw - base);
          l += s_l[w][row] * sw;
          o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(tile0.rows[w]) + row * D +
                                               (d ^ (row & 7) << 2)) * sw;
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
          const float by = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mt);
          o *= by;
          l = l * by + (mt == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - mt));
        }
        const int64_t at = (q0 + token) * a.o_st + head * a.o_sh + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = l == 0.f ? 0.f : o[i] / l;
          if (a.out_f32)
            static_cast<float*>(a.out)[at + i] = x;
          else
            static_cast<T*>(a.out)[at + i] = static_cast<T>(x);
        }
      }
    }
    __syncthreads();
  }
}

// Merges a row's chunks and the sink: D / 4 lanes per (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_combine_kernel(const TreeArgs a) {
  constexpr int kLanes = D / 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const int d = 4 * (threadIdx.x % kLanes);
  const int64_t token = row / a.q_heads;
  const int head = static_cast<int>(row - token * a.q_heads);
  if (token >= a.n_tokens || token >= load_index(a.qo_indptr, a.indptr64, a.n_requests) ||
      token < load_index(a.qo_indptr, a.indptr64, 0) || d >= a.head_dim)
    return;
  if (gated(a.gate)) return;
  const int used = a.used[token];
  if (used <= 1) return;
  const int64_t step = a.n_tokens * a.q_heads;
  const float sink = a.sinks ? a.sinks[head] * kLog2e : -INFINITY;
  float m = sink;
  for (int c = 0; c < used; ++c) m = fmaxf(m, a.part_ml[2 * (c * step + row)]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = a.sinks && m != -INFINITY ? __builtin_amdgcn_exp2f(sink - base) : 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = 0; c < used; ++c) {
    const int64_t at = c * step + row;
    const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * at);
    const f32x4 oc = *reinterpret_cast<const f32x4*>(a.part_o + at * D + d);
    const float w = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - base);
    l += ml.y * w;
    o += oc * w;
  }
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

int tile_dim(int32_t head_dim) { return head_dim <= 64 ? 64 : 128; }

// Row subtiles of a workgroup for requests of up to `rows` rows.
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
  const int64_t block = 16 * p.sub, pass = pass_of(p.d);
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
  hipLaunchKernelGGL((tree_attention_kernel<T, D, SUB>), grid, dim3(kThreads), 0, st, a);
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
  const int64_t rows = a.n_tokens * a.q_heads, per = 256 / (p.d / 4);
  const dim3 merge(static_cast<unsigned>((rows + per - 1) / per));
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
  if (n_tokens > 0x7fffffffLL / q_heads || static_cast<int64_t>(n_requests) * kv_heads > 0x7fffffffLL / 4096)
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
