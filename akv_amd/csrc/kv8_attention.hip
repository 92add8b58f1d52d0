// Attention of new tokens over a cache held in 8 bits (gfx950, MFMA): one token
// per request, a tree of drafted ones, or a chunk of a prompt.
//
// Request b has n = qo_indptr[b + 1] - qo_indptr[b] new tokens and L = kv_indptr[b + 1] -
// kv_indptr[b] keys, whose last n are the tokens' own.  Key j of token i is visible
// when
//   j < L - n:   j < first_keys or j >= key_starts[i]
//   otherwise:   bit j - (L - n) of token i's mask  (or j - (L - n) <= i: a chain)
// and, with a key's codes k_j, v_j and the scales a_j, c_j of its block and head,
//   o_ih = sum_j e^s_j c_j v_j / (sum_j e^s_j + e^sink_h),  s_j = scale a_j (q_ih . k_j)
// over the visible keys; a row that sees none is 0.  A key whose slot lies
// outside the pool is a hole that no token sees.
//
// The n tokens x G heads of a KV head's group are the rows of one product with
// that head's keys, so K and V are read once for a block of 64 SUB rows.  All the
// batch's tiles of keys lie on a line, and 512 workgroups of four waves take equal
// stretches of it; where a cut falls among a request's tiles, a second launch
// merges the parts.  What a window hides of every token is left out: the first keys
// and those from the lowest start on are numbered as one list.  Codes stream into
// LDS as they are (two places) while the tile before is worked on, 32 keys at a time,
// 16 SUB rows per wave; they become bf16 (or fp16, for fp16 queries) in the operands'
// registers, exactly, since those types hold every 8-bit float:
//   S^T[32 x 16 SUB] = K . Q^T               v_mfma_f32_16x16x32
//   P^T = 2^(scale log2(e) a_j S^T - m),     l += P in fp32, lane by lane
//   O^T[D x 16 SUB] += V^T . (c_j P^T)       c_j P rounded to bf16
// With fp16 queries c_j P is the sum of two bf16 values (16 bits of it), since c_j
// takes it out of fp16's range.  A code row is 64 or 128 bytes: a lane's 16 bytes of K
// are its operands of two products (the dims of a product may come in any order that
// Q's follow), V^T comes through ds_read_b64_tr_b8.  m is a row's first maximum and
// moves only when the weights outgrow their types.
//
// Bound, for few rows, by HBM: 32 requests of 20000 keys, 8 heads of 64, one token each, blocks
// of 1: 690 MB in 157 us, 4.4 TB/s, of which the scales, 32 bytes a key in lines of 128, make
// 5.9 of what is really read; in blocks of 16 134 us.  For many rows by the vector
// instructions: a part of 32 keys and 64 rows takes 198 of them (32 exponentials, 32
// scalings before and 32 behind them, 32 sums, 48 conversions) beside 32 products, and they are issued 67%
// of the time: 512 tokens of 64 heads over 16000 keys 223 us, 0.6 PFLOP/s.  Few keys are
// bound by the launches and the chain list - slot - code - product: one request of 4096
// keys 18 us, of which the merge is 4.  A prologue of 6 us and the pieces' results (64 KB
// of 128 rows of 128 dims) make what is left of 12 requests of up to 20000 keys.
// The instances of the most rows do not fit 256 registers: 24 are spilled (64 dims, 4 subtiles;
// pairs of heads 36), 19 (128 dims, 2 subtiles), with fp16 queries 54, 68 and 27; written
// once a workgroup and read once a piece, around its tiles, never among them.
//
// What it does badly: a window over new tokens takes a mask, and with a mask every block of
// rows visits all of the request's new keys and those from its lowest start on, masked (a
// window of 128, 64 heads of 64: chunks of 128 tokens 33 us, of 512 74, of 4096 1318).
//
// Lane layouts (verified on gfx950): v_mfma_f32_16x16x32 -- lane l supplies
// A[l%16][k(l,i)], B[k(l,i)][l%16] for i < 8 and holds D[4(l/16)+i][l%16];
// ds_read_b64_tr_b8 -- within each 16-lane group, lane j receives byte j%8
// of the 8-byte rows read by lanes j/8 + 2i, i < 8.
#include "tree_common.h"

namespace akv {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

#define KV8_INLINE __attribute__((always_inline))

// Keys of a tile (16 or 32 KiB of K and V), and the tiles in LDS.  (256 keys of 64 bytes: one
// request of 4096 keys, 16 tokens, 28.1 us for 26.6, of 60000 28.7 for 27.6, long ones alike; 64
// keys of 128 bytes in four places: 32 requests of 20000 keys 182 for 169.)
constexpr int kKeys = 128, kBuffers = 2;

// What a piece costs beside its tiles, in keys (64 to 512: all within 3%), and the least a
// stretch is given, in what as many keys cost a request whose rows one wave has: 128 as long as
// there is a CU for each, else 256 (us with 128, with 256, one token, 8 heads of 64: 1 request
// of 2000 keys 16.0, 17.1, of 4096 16.2, 17.2, of 8192 18.3, 17.1; of 128: 17.1, 18.5; 17.6, 18.8;
// 22.4, 19.7).  More waves' rows make a tile dearer, and a piece's own cost holds no key, so
// in small batches stretches come without a tile and leave pieces of zeros for the merge: one
// request of 2000 keys 16 of 128 stretches, with four waves' rows 128 of 256; of 4096 16 and 8
// of 256; of 60000 none.
constexpr int kPieceCost = 256;
constexpr int least_share(int log2_groups) { return log2_groups > 8 ? 256 : 128; }

// What a tile costs a request by the waves that share its rows out: four of them (the rows
// of one wave, read by all) 2, two 3, none 4 (us of 12 requests of 11000 keys, 8 heads of
// 128: 4 rows a head 84, 64 rows 111, 128 rows 157; mixed, 4 to 64 rows: 276 for 303 with
// equal costs, of 20 to 128 rows 150 for 157).
constexpr int cost_of_groups(int groups) { return groups == 1 ? 2 : groups == 2 ? 3 : 4; }

struct Kv8Args {
  TreeArgs t;
  const float* k_scales;
  const float* v_scales;
  int64_t ks_sb, ks_sh, vs_sb, vs_sh;
  int32_t log2_block, first_keys;
  int32_t block_rows;  // rows of a block where a workgroup has two heads
};

// 16-byte chunk c of row r lies at chunk c ^ swz(r): the 16 rows of an operand read
// (K), and the rows 4 g + i, 16 + 4 g + i of a transposed read's lanes (V), take
// distinct banks.
template <int W>
__device__ __forceinline__ int swz_k(int r) { return W == 64 ? (r >> 2) & 3 : (r >> 1) & 7; }
template <int W>
__device__ __forceinline__ int swz_v(int r) {
  return W == 64 ? (r >> 2 & 1) | (r >> 4 & 1) << 1 : (r >> 1 & 3) | (r >> 4 & 1) << 2;
}

// Eight codes as an operand of the matrix cores.
template <typename T, bool E5>
__device__ __forceinline__ typename Vec<T>::x8 operand(u32x2 w) {
  typedef T T2 __attribute__((ext_vector_type(2)));
  T2 x[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (__is_same(T, __bf16)) {
      x[2 * i] = E5 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w[i], 1.f, false)
                    : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.f, false);
      x[2 * i + 1] = E5 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w[i], 1.f, true)
                        : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.f, true);
    } else {
      x[2 * i] = E5 ? __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w[i], 1.f, false)
                    : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, false);
      x[2 * i + 1] = E5 ? __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w[i], 1.f, true)
                        : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, true);
    }
  }
  const auto lo = __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3), hi = __builtin_shufflevector(x[2], x[3], 0, 1, 2, 3);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// 0x80 in the bytes that are infinities or NaN.
template <bool E5>
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) {
  return E5 ? ((w & 0x7c7c7c7cu) + 0x04040404u) & 0x80808080u : ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

template <int W>
struct alignas(16) CodeTile {
  char k[kKeys * W];  // key-major, 16-byte chunks swizzled per row (swz_k)
  char v[kKeys * W];  // key-major, read transposed, swizzled (swz_v)
};

// T: q's type.  D: 64 or 128, the tile's head width.  SUB: a wave's row subtiles of 16.
// HEADS: a workgroup's KV heads, side by side in a tile's rows; of two, waves 0 and 1
// have the first and the others the second.  To the line of work, the cuts and the
// merge the two are one head of twice the group (`ka.t` comes so): row r of a block
// is that of token r / (2 G) and of the first head while r % (2 G) < G.
template <typename T, bool E5, int D, int SUB, int HEADS>
__global__ void __launch_bounds__(kThreads, 2) kv8_attention_kernel(const Kv8Args ka) {
  const TreeArgs& a = ka.t;
  using x8 = typename Vec<T>::x8;
  using b4 = Vec<__bf16>::x4;
  using b8 = Vec<__bf16>::x8;
  constexpr bool kSplit = !__is_same(T, __bf16);  // weights as two bf16 values
  constexpr int W = D * HEADS;                 // bytes of a tile's row
  constexpr int kParts = kKeys / 32;
  constexpr int kSteps = D / 32;
  constexpr int kDTiles = D / 16;
  constexpr int kChunks = W / 16;              // 16-byte chunks of a row
  constexpr int kLoadRows = 64 / kChunks;      // rows of one wave-wide load
  constexpr int kWaveKeys = kKeys / kWaves;    // keys of a tile that a wave asks for
  constexpr int kEntryTiles = 64 / kWaveKeys;  // tiles whose keys of this wave fill a vector register
  constexpr int kHeadWaves = kWaves / HEADS;   // waves of a head
  constexpr int kOver = 2 * kPieceCost / kKeys;
  constexpr int kGroupRows = 16 * SUB;         // rows of a wave
  const int R = HEADS == 1 ? kWaves * kGroupRows : ka.block_rows;  // rows of a block
  // (and behind them the waves' results)
  constexpr int kPlaces = std::max<int>(kBuffers, kWaves * kGroupRows * D * 4 / sizeof(CodeTile<W>));
  __shared__ CodeTile<W> buffers[kPlaces];
  __shared__ __attribute__((aligned(16))) float s_scale[kBuffers][kWaves][2][kWaveKeys * HEADS];  // the tiles' a_j and c_j
  __shared__ int32_t s_entry[kWaves][2][64];  // list entries of the waves' keys, kEntryTiles tiles at a time
  __shared__ uint32_t s_dead[2 * kEntryTiles][kParts];  // the tiles' keys that no token sees
  __shared__ float s_m[kWaves][kGroupRows], s_l[kWaves][kGroupRows];
  // for the masked parts: the rows' tokens, first keys and first mask words
  __shared__ uint64_t s_words[kWaves][kGroupRows][kWordsKept];
  __shared__ int32_t s_tok[kWaves][kGroupRows], s_start[kWaves][kGroupRows];
  int64_t* s_out = reinterpret_cast<int64_t*>(s_words);  // behind the tiles: where the rows go
  static_assert(kWaves * kGroupRows * D * 4 <= sizeof(buffers), "the waves' results fit the tiles");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  auto keys_in = [&](int64_t b) -> int64_t {
    const int64_t len = load_index(a.kv_indptr, a.indptr64, b + 1) - load_index(a.kv_indptr, a.indptr64, b);
    return len < 0 ? 0 : len < kMostKeys ? len : kMostKeys;
  };
  // keys that block rb of a request's rows reaches: a chain's end with its last token
  auto reach = [&](int64_t len, int32_t n, int rb) -> int64_t {
    const int64_t tokens = ((rb + 1) * static_cast<int64_t>(R) + a.group - 1) / a.group;
    return a.mask || tokens >= n || n > len ? len : len - n + tokens;
  };
  // groups of rows that a head's `left` rows from a block's first on make
  auto groups_of = [&](int left) -> int {
    int groups = kHeadWaves;
    while (groups > 1 && left <= (groups >> 1) * kGroupRows) groups >>= 1;
    return groups;
  };
  // One wave's view of the batch.  A request costs its tiles, by what the waves have to do
  // there, and kOver for every block of rows; block rb's cost is 0 where it has no such rows.
  auto units_of = [&](int64_t len, int32_t n, int rb) -> int32_t {
    len = reach(len, n, rb);
    if (a.key_starts && len > a.max_len) len = a.max_len;  // what a window reaches is not known here
    const int64_t tiles = len > kKeys ? (len + kKeys - 1) / kKeys : 1;
    const int64_t left = static_cast<int64_t>(n) * a.group - static_cast<int64_t>(rb) * R;
    if (left <= 0) return 0;
    const int groups = groups_of(static_cast<int>(std::min<int64_t>(left, R)) / HEADS);
    return static_cast<int32_t>(tiles * cost_of_groups(groups)) + kOver;
  };
  struct Cost {
    int32_t units, rows;
  };
  auto cost_of = [&](int64_t b, int rb) -> Cost {
    int64_t q0 = load_index(a.qo_indptr, a.indptr64, b), q1 = load_index(a.qo_indptr, a.indptr64, b + 1);
    q0 = q0 < 0 ? 0 : q0;
    q1 = q1 > a.n_tokens ? a.n_tokens : q1;
    const int32_t n = q1 > q0 ? static_cast<int32_t>(q1 - q0) : 0;
    return Cost{units_of(keys_in(b), n, rb), n * a.group};
  };
  auto sum_of = [&](int rb) -> int64_t {
    int64_t sum = 0;
    for (int b = lane; b < a.n_requests; b += 64) sum += cost_of(b, rb).units;
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
    // (Every wave adds up the longest request's blocks of rows over all requests: a
    // prompt of 8192 tokens among 63 requests of one, 64 heads of 64, takes 1405 us, the two
    // apart 1263 and 30.)
    int32_t most = 0;
    for (int i = lane; i < a.n_requests; i += 64) most = max(most, cost_of(i, 0).rows);
    blocks = (uniform(__ockl_wfred_max_i32(most)) + R - 1) / R;
    const int64_t items = static_cast<int64_t>(blocks) * a.n_requests;
    int64_t mine = 0;
    for (int64_t i = lane; i < items; i += 64) {
      const int64_t at = items >> 31 ? i / a.n_requests : static_cast<uint32_t>(i) / static_cast<uint32_t>(a.n_requests);
      mine += cost_of(i - at * a.n_requests, static_cast<int>(at)).units;
    }
    const int64_t until = __ockl_wfscan_add_i64(mine, true);
    const int64_t all = uniform(__shfl(until, 63)) * a.kv_heads;
    if (all == 0) return;
    // 2^k stretches: all of the workgroups, or as many as get their least share
    int k = kGroupsShift;
    while (k > 0 && (static_cast<int64_t>(2 * least_share(k) / kKeys) << k) > all) --k;
    if (group_id >> k) return;
    auto cut = [&](int64_t i) { return (all >> k) * i + (((all & ((1 << k) - 1)) * i) >> k); };  // all * i / 2^k
    int64_t x = cut(group_id);
    budget = cut(group_id + 1) - x;
    if (items <= 64) {
      // a lane has an item, all of a block's side by side
      rb = __builtin_ctzll(__builtin_amdgcn_ballot_w64(until * a.kv_heads > x)) / a.n_requests;
      const int at = rb * a.n_requests;
      const int64_t before = uniform(__shfl(until - mine, at));
      const int64_t sum = uniform(__shfl(until, at + a.n_requests - 1)) - before;
      x -= before * a.kv_heads;
      for (g = 0; x >= sum; ++g) x -= sum;
      const int item = __builtin_ctzll(__builtin_amdgcn_ballot_w64(until - before > x));
      off = x - (uniform(__shfl(until - mine, item)) - before);
      b = item - at;
    } else {
      rb = 0;
      int64_t sum = sum_of(0);
      while (x >= sum * a.kv_heads) {
        x -= sum * a.kv_heads;
        sum = sum_of(++rb);
      }
      for (g = 0; x >= sum; ++g) x -= sum;
      b = 0;
      for (int b0 = 0; b0 < a.n_requests; b0 += 64) {
        const int32_t units = b0 + lane < a.n_requests ? cost_of(b0 + lane, rb).units : 0;
        const int64_t up = __ockl_wfscan_add_i64(units, true);
        const uint64_t past = __builtin_amdgcn_ballot_w64(up > x);
        if (past) {
          const int at = __builtin_ctzll(past);
          b = b0 + at;
          off = uniform(x - __shfl(up - units, at));
          break;
        }
        x -= __shfl(up, 63);
      }
    }
  }

  for (;;) {
    // (in scalar registers: the loop has no vector register to spare)
    int64_t q0 = uniform(load_index(a.qo_indptr, a.indptr64, b)), q1 = uniform(load_index(a.qo_indptr, a.indptr64, b + 1));
    const int64_t kv0 = uniform(load_index(a.kv_indptr, a.indptr64, b));
    const int all_keys = static_cast<int>(uniform(keys_in(b)));
    if (q0 < 0) q0 = 0;
    if (q1 > a.n_tokens) q1 = a.n_tokens;
    const int n = static_cast<int>(q1 > q0 ? q1 - q0 : 0);
    const int rows = n * a.group;
    const int old = all_keys > n ? all_keys - n : 0;
    if (a.whole && static_cast<int64_t>(rb) * R >= rows) return;
    const int len = static_cast<int>(reach(all_keys, n, rb));
    // the earlier keys that some token of the request sees: the first ones, and those
    // from `lo` on.  Key number v of them all has rank v, or v + gap from `kept` on.
    const int kept = min(ka.first_keys, old);
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
    const int gap = max(lo - kept, 0);
    const int count = max(len - gap, 0);
    // the piece: units [off, stop) of the request's, the first kOver of them
    // for no tile, the others for equal parts of its tiles
    const int units = units_of(all_keys, n, rb);
    const int stop = a.whole || budget > units - off ? units : static_cast<int>(off + budget);
    const bool first = off == 0, last = stop == units;
    const int all_tiles = (count + kKeys - 1) / kKeys;
    auto tile_of = [&](int64_t unit) -> int {
      const int64_t at = unit > kOver ? unit - kOver : 0;
      return static_cast<int>(units - kOver == all_tiles ? at : at * all_tiles / (units - kOver));
    };
    const int begin = uniform(tile_of(off)) * kKeys;
    const int end = min(uniform(tile_of(stop)) * kKeys, count);
    const int tiles = end > begin ? (end - begin + kKeys - 1) / kKeys : 0;

    // (an empty pool holds no key: every slot is a hole, and zeros are read)
    const bool pool = a.pool_slots > 0;
    const char* kbase = pool ? a.k + static_cast<int64_t>(HEADS) * g * a.k_sh : reinterpret_cast<const char*>(zero_row);
    const char* vbase = pool ? a.v + static_cast<int64_t>(HEADS) * g * a.v_sh : reinterpret_cast<const char*>(zero_row);
    const float* ks_base = pool ? ka.k_scales + HEADS * g * ka.ks_sh : reinterpret_cast<const float*>(zero_row);
    const float* vs_base = pool ? ka.v_scales + HEADS * g * ka.vs_sh : reinterpret_cast<const float*>(zero_row);
    const uint32_t k_ss = pool ? a.k_ss : 0, v_ss = pool ? a.v_ss : 0;
    const int64_t ks_sb = pool ? ka.ks_sb : 0, vs_sb = pool ? ka.vs_sb : 0;
    // from the first head to the second
    const int64_t k_next = pool ? a.k_sh : 0, v_next = pool ? a.v_sh : 0;
    const int64_t ks_next = pool ? ka.ks_sh : 0, vs_next = pool ? ka.vs_sh : 0;
    const int32_t* list = a.kv_indices + (a.paged ? b * a.table_stride : kv0);
    // entries of the list that exist
    const int64_t left = a.paged ? a.table_width : kv0 < 0 ? 0 : a.table_width - kv0;
    const int32_t width = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(left, 0), 0x7fffffff));
    const int32_t* entries = width > 0 ? list : reinterpret_cast<const int32_t*>(zero_row);
    const int last_entry = max(width - 1, 0);
    // The wave's keys of kEntryTiles tiles at a time: lane l has key l % kWaveKeys
    // of tile l / kWaveKeys.  Their list entries come to LDS kEntryTiles tiles ahead.
    const int my_key = lane / kWaveKeys * kKeys + kWaveKeys * wave + lane % kWaveKeys;
    auto rank_of = [&](int e) -> uint32_t {
      const int v = min(begin + e * (kEntryTiles * kKeys) + my_key, end - 1);  // past the end: the last key's
      return v + (v >= kept ? gap : 0);
    };
    auto fetch = [&](int e) {
      const uint32_t j = rank_of(e);
      const int32_t at = a.paged ? j / static_cast<uint32_t>(a.page_size) : j;
      load_4(entries + min(at, last_entry), uniform(lds_address(s_entry[wave][e & 1])));
    };
    uint32_t slots = 0;
    auto look_up = [&](int e) {
      const uint32_t j = rank_of(e);
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
      const bool past = begin + e * (kEntryTiles * kKeys) + my_key >= end;
      const uint64_t dead = __builtin_amdgcn_ballot_w64(!there || past);
      if (lane < kEntryTiles) {
        uint32_t* to = s_dead[(e & 1) * kEntryTiles + lane] + wave;
        *to = static_cast<uint32_t>(dead >> (kWaveKeys * lane));
      }
    };
    // a wave's keys of a tile, straight into LDS: lane l of a load fills bytes
    // 16 l of a 1 KiB block, chunk position l % kChunks of a row
    auto stage = [&](int it) {
      if (it % kEntryTiles == 0) {
        look_up(it / kEntryTiles);
        fetch(it / kEntryTiles + 1);
      }
      CodeTile<W>& t = buffers[it % kBuffers];
#pragma unroll
      for (int u = 0; u < kWaveKeys / kLoadRows; ++u) {
        const int mine = u * kLoadRows + lane / kChunks, r = kWaveKeys * wave + mine;
        const uint64_t from = __shfl(slots, it % kEntryTiles * kWaveKeys + mine);
        const int ck = (lane % kChunks) ^ swz_k<W>(r), cv = (lane % kChunks) ^ swz_v<W>(r);
        const int dk = 16 * ck % D, dv = 16 * cv % D;
        const char* krow = kbase + from * k_ss + dk;
        const char* vrow = vbase + from * v_ss + dv;
        if constexpr (HEADS == 2) {
          krow += 16 * ck < D ? 0 : k_next;
          vrow += 16 * cv < D ? 0 : v_next;
        }
        // dims past head_dim read zeros
        krow = dk < a.head_dim ? krow : reinterpret_cast<const char*>(zero_row);
        vrow = dv < a.head_dim ? vrow : reinterpret_cast<const char*>(zero_row);
        const int place = (kWaveKeys * wave + u * kLoadRows) * W;
        load_16(krow, uniform(lds_address(t.k + place)));
        load_16(vrow, uniform(lds_address(t.v + place)));
      }
      // a_j of the wave's keys, then c_j, 64 lanes at a time; of two heads those of a
      // key side by side
#pragma unroll
      for (int u = 0; u < 2 * HEADS * kWaveKeys; u += 64) {
        const bool is_v = u + lane >= HEADS * kWaveKeys;
        const uint32_t block = __shfl(slots, it % kEntryTiles * kWaveKeys + lane / HEADS % kWaveKeys) >> ka.log2_block;
        const float* from = is_v ? vs_base + block * vs_sb : ks_base + block * ks_sb;
        if constexpr (HEADS == 2) from += lane % 2 == 0 ? 0 : is_v ? vs_next : ks_next;
        load_4(from, uniform(lds_address(s_scale[it % kBuffers][wave][0] + u)));
      }
    };
    if (tiles > 0) fetch(0);
    // a head's groups of rows, and the waves that share one
    const int heads_group = a.group / HEADS, head_rows = n * heads_group, block_row0 = rb * (R / HEADS);
    const int hw = wave / kHeadWaves;  // the wave's head
    const int groups = groups_of(min(head_rows - block_row0, R / HEADS)), sharers = kHeadWaves / groups;
    const int row0 = block_row0 + (wave & (groups - 1)) * kGroupRows;
    const int share = uniform(wave % kHeadWaves / groups);
    // this lane's rows of the head: r = row0 + 16 s + col, token r / G, q head r % G of its G
    // (rows past the last repeat it and are never stored).  Step st of a product takes
    // bytes 8 (st % 2) of the 16 code bytes 64 (st / 2) + 16 quad.
    x8 qop[SUB][kSteps];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int r = min(row0 + 16 * s + col, head_rows - 1);
      const int tok = r / heads_group;
      const T* row = static_cast<const T*>(a.q) + (q0 + tok) * a.q_st +
                     static_cast<int64_t>(g * a.group + hw * heads_group + r - tok * heads_group) * a.q_sh;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        u32x4 w = {0u, 0u, 0u, 0u};
        const int c = 8 * (st / 2) + 2 * quad + st % 2;
        if (8 * c < a.head_dim) w = *((const global_u32x4*)row + c);
        qop[s][st] = __builtin_bit_cast(x8, w);
      }
    }
    f32x4 acc[SUB][kDTiles];
    float neg_m[SUB], l[SUB];  // l: this lane's share of the row's weights
    uint32_t have = 0;         // rows s that have a maximum
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      neg_m[s] = 0.f;
      l[s] = 0.f;
#pragma unroll
      for (int t = 0; t < kDTiles; ++t) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool unset = true;  // some row of the wave has no maximum yet

    // word w of a token's mask row
    auto mask_word = [&](int tok, int w) -> uint64_t {
      if (a.mask) return w < a.mask_words ? a.mask[(q0 + tok) * a.mask_stride + w] : 0;
      const int i = tok - 64 * w;
      return i >= 63 ? ~0ull : i < 0 ? 0 : (2ull << i) - 1;
    };
    auto start_of = [&](int tok) -> int { return a.key_starts ? min(max(a.key_starts[q0 + tok], 0), old) : 0; };
    // what a row sees of the 32 keys from number v0 on: the first ones, those of rank
    // `start` on, and the new tokens' by its words
    auto visible = [&](int v0, int start, auto word) -> uint32_t {
      const int k0 = v0 + gap, base = k0 - old;
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
      const int early = kept - v0;
      if (early >= 32) bits = ~0ull; else if (early > 0) bits |= (1ull << early) - 1;
      return static_cast<uint32_t>(bits);
    };
    if (lane < kGroupRows) {
      const int tok = min(row0 + lane, head_rows - 1) / heads_group;
      s_tok[wave][lane] = tok;
      s_start[wave][lane] = start_of(tok);
#pragma unroll
      for (int w = 0; w < kWordsKept; ++w) s_words[wave][lane][w] = mask_word(tok, w);
    }
    // this lane's operands in part 0: K chunks quad (and 4 + quad) of row col, and the
    // source of its transposed V reads (half a chunk dt of the row of its place in
    // the group); the swizzles are the same in every part
    uint32_t k_at[kSteps / 2], v_at[kDTiles];
    const int vi = col >> 1, vr = 4 * quad + (vi & 3) + 16 * (vi >> 2);
#pragma unroll
    for (int h = 0; h < kSteps / 2; ++h) k_at[h] = col * W + 16 * ((hw * (D / 16) + 4 * h + quad) ^ swz_k<W>(col));
#pragma unroll
    for (int dt = 0; dt < kDTiles; ++dt) v_at[dt] = vr * W + 16 * ((hw * kDTiles + dt) ^ swz_v<W>(vr)) + 8 * (col & 1);
    // products of the 32 keys of a part: S^T[16 j + 4 quad + i][row 16 s + col]
    auto codes_of = [&](const CodeTile<W>& t, int kk, u32x4 (&k)[2][kSteps / 2]) KV8_INLINE {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < kSteps / 2; ++h)
          k[j][h] = *reinterpret_cast<const u32x4*>(t.k + (32 * kk + 16 * j) * W + k_at[h]);
    };
    auto scores = [&](const u32x4 (&k)[2][kSteps / 2], f32x4 (&sc)[2][SUB]) KV8_INLINE {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int h = 0; h < kSteps / 2; ++h) {
          const u32x4 w = k[j][h];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const x8 kop = operand<T, E5>(u32x2{w[2 * half], w[2 * half + 1]});
#pragma unroll
            for (int s = 0; s < SUB; ++s)
              sc[j][s] = product(kop, qop[s][2 * h + half], h + half == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : sc[j][s]);
          }
        }
      }
    };
    // codes V[key][16 dt + col] of keys 4 quad + i (i < 4) of the part, then 16 keys on
    auto v_tile = [&](const CodeTile<W>& t, int kk, int dt) KV8_INLINE -> u32x2 {
      return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(t.v + 32 * kk * W + v_at[dt])));
    };
    // a part's a_j (which 0) or c_j (1) of keys 4 quad + i, and 16 keys on
    auto scales_of = [&](int it, int which, int kk, f32x4 (&x)[2]) KV8_INLINE {
      const float* from = s_scale[it % kBuffers][32 * kk / kWaveKeys][which] + (32 * kk % kWaveKeys + 4 * quad) * HEADS;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (HEADS == 1) {
          x[j] = *reinterpret_cast<const f32x4*>(from + 16 * j);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[j][i] = from[(16 * j + i) * HEADS + hw];
        }
      }
    };
    struct Weights {
      b8 hi, lo;
    };
    // c_j P, rounded
    auto weights = [&](const f32x4 (&e)[2]) KV8_INLINE -> Weights {
      Weights w;
      const b4 h0 = __builtin_convertvector(e[0], b4), h1 = __builtin_convertvector(e[1], b4);
      w.hi = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
      if constexpr (kSplit) {
        const b4 l0 = __builtin_convertvector(e[0] - __builtin_convertvector(h0, f32x4), b4);
        const b4 l1 = __builtin_convertvector(e[1] - __builtin_convertvector(h1, f32x4), b4);
        w.lo = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      return w;
    };
    auto add_values = [&](u32x2 codes, int dt, const Weights (&p)[SUB]) KV8_INLINE {
      const b8 v = operand<__bf16, E5>(codes);
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        acc[s][dt] = product(v, p[s].hi, acc[s][dt]);
        if constexpr (kSplit) acc[s][dt] = product(v, p[s].lo, acc[s][dt]);
      }
    };
    // 32 keys that every row sees, when every row has a maximum; false, with
    // nothing done, where a sum outgrows kHuge
    auto quick = [&](const CodeTile<W>& t, int it, int kk) KV8_INLINE -> bool {
      f32x4 sc[2][SUB], ks[2], vs[2];
      u32x4 k[2][kSteps / 2];
      u32x2 v[kDTiles];
      // all reads first: none of them waits behind a matrix product or the branch
      codes_of(t, kk, k);
      scales_of(it, 0, kk, ks);
      scales_of(it, 1, kk, vs);
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) v[dt] = v_tile(t, kk, dt);
      __builtin_amdgcn_sched_barrier(0);
      // Products before the other wave's vector instructions, which have time while they
      // run (12 requests of up to 20000 keys 149 -> 142 us, 512 tokens over 16000 244 -> 237).
      __builtin_amdgcn_s_setprio(1);
      scores(k, sc);
      __builtin_amdgcn_s_setprio(0);
      ks[0] *= a.scale_log2;
      ks[1] *= a.scale_log2;
      Weights p[SUB];
      float sum[SUB];
      bool huge = false;
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        f32x4 e[2];
        sum[s] = l[s];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[j][i] = __builtin_amdgcn_exp2f(fmaf(sc[j][s][i], ks[j][i], neg_m[s]));
            sum[s] += e[j][i];
          }
          e[j] *= vs[j];
        }
        p[s] = weights(e);
        huge |= sum[s] > 0.25f * kHuge;
      }
      if (__builtin_amdgcn_ballot_w64(huge)) return false;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int s = 0; s < SUB; ++s) l[s] = sum[s];
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) add_values(v[dt], dt, p);
      __builtin_amdgcn_s_setprio(0);
      return true;
    };
    // any 32 keys; v0: the first one's number
    auto part = [&](const CodeTile<W>& t, int it, int kk, int v0, uint32_t dead) KV8_INLINE {
      f32x4 sc[2][SUB], ks[2], vs[2];
      u32x4 k[2][kSteps / 2];
      u32x2 v[kDTiles];
      codes_of(t, kk, k);
      scales_of(it, 0, kk, ks);
      scales_of(it, 1, kk, vs);
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) v[dt] = v_tile(t, kk, dt);
      scores(k, sc);
      uint32_t odd = 0;  // infinities and NaN among the lane's values
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) odd |= odd_bytes<E5>(v[dt][0]) | odd_bytes<E5>(v[dt][1]);
      uint32_t seen[SUB];  // bit 4 j + i: key 16 j + 4 quad + i
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const int in = 16 * s + col;
        const uint32_t bits = ~dead & visible(v0, s_start[wave][in], [&](int w) -> uint64_t {
          return w < kWordsKept ? s_words[wave][in][w] : mask_word(s_tok[wave][in], w);
        });
        seen[s] = (bits >> 4 * quad & 15) | (bits >> (16 + 4 * quad) & 15) << 4;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sc[j][s][i] = seen[s] >> (4 * j + i) & 1 ? sc[j][s][i] * (ks[j][i] * a.scale_log2) : -INFINITY;
      }
      // A row's m is its maximum over the first part it sees a key of, and then
      // stays put: the sum tells when it should not have.  A sum past kHuge takes
      // the part again with exact maxima.
      Weights p[SUB];
      float sum[SUB];
      for (bool exact = unset;; exact = true) {
        if (exact) {
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            const float m0 = max3(sc[0][s][0], sc[0][s][1], sc[0][s][2]);
            const float m1 = max3(sc[0][s][3], sc[1][s][0], sc[1][s][1]);
            const float mx = column_max(max3(m0, m1, max2(sc[1][s][2], sc[1][s][3])));
            const float over = mx + neg_m[s];  // above m
            const bool any = have >> s & 1;
            // (a sum near kHuge whose large weights lie behind moves by 2^16)
            const bool down = any && column_max(l[s]) > 0.125f * kHuge && !(over > 16.f);
            const bool move = any ? over > 0.f : mx > -INFINITY;
            const float alpha = down ? 0x1p-16f : move && any ? __builtin_amdgcn_exp2f(-over) : 1.f;
            l[s] *= alpha;
#pragma unroll
            for (int dt = 0; dt < kDTiles; ++dt) acc[s][dt] *= alpha;
            neg_m[s] = down ? neg_m[s] - 16.f : move ? -mx : neg_m[s];
            if (move) have |= 1u << s;
          }
        }
        bool huge = false;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          f32x4 e[2];
          sum[s] = l[s];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = __builtin_amdgcn_exp2f(sc[j][s][i] + neg_m[s]);
              sum[s] += x;
              // (the scale of a key that is not seen may be anything)
              e[j][i] = seen[s] >> (4 * j + i) & 1 ? x * vs[j][i] : 0.f;
            }
          }
          p[s] = weights(e);
          huge |= sum[s] > 0.25f * kHuge;
        }
        if (exact || !__builtin_amdgcn_ballot_w64(huge)) break;
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) l[s] = sum[s];
      if (unset) {
        bool none = false;
#pragma unroll
        for (int s = 0; s < SUB; ++s) none |= !(have >> s & 1) && l[s] == 0.f;  // (NaN: no maximum will come)
        unset = __builtin_amdgcn_ballot_w64(none) != 0;
      }
      // A weight of 0 does not hide an infinity or NaN from the product: such codes
      // are taken out of it, and the dims of the rows that see them become NaN.
      if (__builtin_amdgcn_ballot_w64(odd != 0)) {
#pragma unroll
        for (int dt = 0; dt < kDTiles; ++dt) {
          const u32x2 here = {odd_bytes<E5>(v[dt][0]), odd_bytes<E5>(v[dt][1])};
          v[dt] &= ~((here >> 7) * 255u);
          const b8 which = operand<__bf16, E5>((here >> 7) * (E5 ? 0x3cu : 0x38u));  // ones
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            b8 sees;
#pragma unroll
            for (int i = 0; i < 8; ++i) sees[i] = static_cast<__bf16>(seen[s] >> i & 1 ? 1.f : 0.f);
            const f32x4 hits = product(which, sees, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[s][dt][i] = hits[i] > 0.f ? __builtin_nanf("") : acc[s][dt][i];
          }
        }
      }
#pragma unroll
      for (int dt = 0; dt < kDTiles; ++dt) add_values(v[dt], dt, p);
    };
    __builtin_amdgcn_s_waitcnt(0);  // (one the compiler sees: Q has arrived)
    __syncthreads();
    if (tiles > 0) stage(0);
    arrive();
    // keys that all of the wave's rows are late enough for
    const int sure = a.mask ? old : old + uniform(min(row0, head_rows - 1) / heads_group) + 1;
    // this wave's parts of a tile
    uint32_t parts = 0;
#pragma unroll
    for (int kk = 0; kk < kParts; ++kk) parts |= (kk & (sharers - 1)) == share ? 1u << kk : 0;
#pragma nounroll
    for (int it = 0; it < tiles; ++it) {
      // into the place that was last read before the barrier
      if (it + 1 < tiles) stage(it + 1);
      const CodeTile<W>& t = buffers[it % kBuffers];
      const int t0 = begin + it * kKeys;
      const uint32_t* dead = s_dead[it % (2 * kEntryTiles)];
      // the parts that all of the wave's rows see: behind their windows' starts or in the
      // first keys, before their tokens, without a hole
      auto below = [&](int at) -> uint32_t {  // parts that end at `at` or before
        const int x = (at - t0) >> 5;
        return x >= kParts ? (2u << (kParts - 1)) - 1 : x <= 0 ? 0 : (1u << x) - 1;
      };
      const uint32_t holes = __builtin_amdgcn_ballot_w64(dead[lane % kParts] != 0);
      uint32_t ready = below(sure - gap) & ~(below(hi_start - gap + 31) & ~below(kept)) & ~holes;
      uint32_t todo = parts & below(end + 31);
#pragma nounroll
      while (todo) {
        if (!unset) {
#pragma nounroll
          for (uint32_t rest = todo & ready; rest; rest &= rest - 1) {
            const int kk = __builtin_ctz(rest);
            if (!quick(t, it, kk)) break;
            todo &= ~(1u << kk);
          }
        }
        if (todo == 0) break;
        const int kk = __builtin_ctz(todo);
        part(t, it, kk, t0 + 32 * kk, uniform(dead[kk]));
        todo &= todo - 1;
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
      l[s] += __shfl_xor(l[s], 16);
      l[s] += __shfl_xor(l[s], 32);
      if (quad == 0) {
        s_m[wave][r] = l[s] == 0.f ? -INFINITY : -neg_m[s];
        s_l[wave][r] = l[s];
      }
    }
    __syncthreads();
    const int here = HEADS == 1 ? min(rows - rb * R, groups * kGroupRows) : min(rows - rb * R, R);
    // where row i of the block is: the first of its waves, a row of theirs
    struct Spot {
      int wave, in;
    };
    auto spot_of = [&](int i) KV8_INLINE -> Spot {
      if constexpr (HEADS == 1) return Spot{i / kGroupRows, i % kGroupRows};
      const int tok = i / a.group, in = i - tok * a.group, second = in >= heads_group;
      const int r = tok * heads_group + in - (second ? heads_group : 0);
      return Spot{second * kHeadWaves + r / kGroupRows, r % kGroupRows};
    };
    // an unfinished piece: a stretch has at most one that continues an earlier
    // stretch's, and one that the next continues
    const int64_t place = 2 * group_id + (first ? 1 : 0);
    float* part_o = a.part_o + place * R * D;
    float* part_ml = a.part_ml + place * R * 2;
    // a thread per row: the sharers' factors, with the sink and the sum when the
    // piece is all of it
    const int mine = here_only(threadIdx.x);
    if (mine < here) {
      const int r = rb * R + mine, token = r / a.group, head = g * a.group + r - token * a.group;
      const int64_t row = q0 + token;
      const auto [w0, in] = spot_of(mine);
      const int w1 = w0 / kHeadWaves * kHeadWaves + kHeadWaves;
      float m = -INFINITY, lt = 0.f;
      for (int w = w0; w < w1; w += groups) m = fmaxf(m, s_m[w][in]);
      // a wave that has seen no key carries m = -inf, l = 0 and O = 0
      float base = m == -INFINITY ? 0.f : m;
      for (int w = w0; w < w1; w += groups) lt += s_l[w][in] * __builtin_amdgcn_exp2f(s_m[w][in] - base);
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
      for (int w = w0; w < w1; w += groups) s_m[w][in] = __builtin_amdgcn_exp2f(s_m[w][in] - base) * scale;
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
    if (d < a.head_dim) {
#pragma unroll 2
      for (int r = mine / (D / 4); r < here; r += kRowsAtOnce) {
        const auto [w0, in] = spot_of(r);
        const int w1 = w0 / kHeadWaves * kHeadWaves + kHeadWaves;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int w = w0; w < w1; w += groups)
          o += *reinterpret_cast<const f32x4*>(result_of(w) + in * D + (d ^ (in & 7) << 2)) * s_m[w][in];
        if (first && last)
          store_four<T>(a, s_out[r] + d, o);
        else
          *reinterpret_cast<f32x4*>(part_o + r * D + d) = o;
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

int tile_dim(int32_t head_dim) { return head_dim <= 64 ? 64 : 128; }

// A wave's row subtiles for requests of up to `rows` rows: two waves' worth, so that
// pairs of waves share the keys (one and four waves' worth, us: 32 requests of 20000 keys,
// 8 heads of 64, 32 rows a head 190 by this rule, 184, 195; 64 rows 225, 234, 271; 12 requests
// of up to 20000, 8 heads of 128, 24 rows 92, 100, 91; 48 rows 108, 110, 117).
int subtiles_for(int d, int64_t rows) {
  const int most = d == 64 ? 4 : 2;
  int sub = 1;
  while (sub < most && rows > 32 * sub) sub *= 2;
  return sub;
}

struct Launch {
  int d, sub, heads;
  bool whole;
  int32_t row_blocks, block_rows;
};

// By the bounds alone, not by the batch's lengths, which the host does not know: a graph
// captured for the longest context cuts its short requests too.
//
// Short requests are not cut: a workgroup has a request and head whole, and nothing is
// merged.  Up to kWholeBytes of K a request always, up to kFullBytes where they are
// kFullGroups (us whole and cut, one token a request of one length, 8 heads of 64: 1 request
// of 800 keys 16.0, 19.5, of 1600 20.9, 21.1; 16 of 1600 22.7, 22.0; 32 of 1600 23.6, 27.0, of
// 6000 69, 56; 8 heads of 128: 1 of 800 18.9, 18.9, of 1200 22.5, 19.0; 32 of 1600 29, 34).
constexpr int64_t kWholeBytes = 96 << 10, kFullBytes = 128 << 10, kFullGroups = 256;

Launch plan(int64_t n_tokens, int64_t n_requests, int64_t q_heads, int64_t kv_heads, int32_t head_dim,
            int64_t max_len, int64_t max_new) {
  Launch p;
  p.d = tile_dim(head_dim);
  const int64_t rows = most_rows(n_tokens, q_heads, kv_heads, max_new);
  p.sub = subtiles_for(p.d, rows);
  auto blocks = [&]() -> int64_t { return (rows + 16 * kWaves * p.sub - 1) / (16 * kWaves * p.sub); };
  p.whole = max_len <= kWholeBytes / p.d ||
            (max_len <= kFullBytes / p.d && n_requests * kv_heads * blocks() >= kFullGroups);
  // (further blocks of rows follow in the same workgroup)
  const int64_t room = std::max<int64_t>(1, kMostBlocks / std::max<int64_t>(1, n_requests * kv_heads));
  p.row_blocks = static_cast<int32_t>(std::min(blocks(), std::min<int64_t>(room, 4096)));
  const int64_t group = q_heads / kv_heads, head_rows = 16 * kWaves / 2 * p.sub;
  // Two heads to a workgroup, as long as their rows are one block and K and V outgrow the
  // last-level cache: their rows of 64 codes share lines of 128 bytes, and their scales one
  // (us of two and one, blocks of 1 and of 16: 32 requests of 20000 keys 156, 200; 135, 148; 16 84, 106;
  // 72, 80; 8 49, 47; 43, 42; 64 of 4000 69, 76; 58, 56; 1 of 4096, 16 tokens, 32, 27).  Never
  // where nothing is cut: the workgroups are few (1 request of 1600 keys 30, 21)
  constexpr double kPairBytes = 192 << 20;
  const double bytes = 2. * p.d * n_requests * kv_heads * max_len;
  p.heads = !p.whole && bytes > kPairBytes && p.d == 64 && kv_heads % 2 == 0 && rows <= head_rows ? 2 : 1;
  p.block_rows = static_cast<int32_t>(p.heads == 2 ? head_rows / group * 2 * group : 16 * kWaves * p.sub);
  return p;
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
  if (max_len <= kWholeBytes / d) return 16;
  return cut_bytes(d, subtiles_for(d, most_rows(n_tokens, q_heads, kv_heads, max_new)), n_tokens, q_heads);
}

template <typename T, bool E5>
int launch(const Kv8Args& a, const Launch& p, hipStream_t st) {
  const int64_t blocks = p.whole ? static_cast<int64_t>(a.t.n_requests) * a.t.kv_heads * a.t.row_blocks : kGroups;
  const dim3 grid(static_cast<unsigned>(blocks)), threads(kThreads);
  auto start = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, threads, 0, st, a); };
  if (p.heads == 2) {
    if (p.sub == 1) start(kv8_attention_kernel<T, E5, 64, 1, 2>);
    else if (p.sub == 2) start(kv8_attention_kernel<T, E5, 64, 2, 2>);
    else start(kv8_attention_kernel<T, E5, 64, 4, 2>);
  } else if (p.d == 64) {
    if (p.sub == 1) start(kv8_attention_kernel<T, E5, 64, 1, 1>);
    else if (p.sub == 2) start(kv8_attention_kernel<T, E5, 64, 2, 1>);
    else start(kv8_attention_kernel<T, E5, 64, 4, 1>);
  } else {
    if (p.sub == 1) start(kv8_attention_kernel<T, E5, 128, 1, 1>);
    else start(kv8_attention_kernel<T, E5, 128, 2, 1>);
  }
  int rc = check_launch("akv_kv8_attention");
  if (rc || p.whole) return rc;
  if (p.d == 64)
    merge<T, 64>(a.t, p.block_rows, st);
  else
    merge<T, 128>(a.t, p.block_rows, st);
  return check_launch("akv_kv8_attention (combine)");
}

bool sizes_ok(int64_t n_tokens, int32_t n_requests, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
              int64_t max_len, int64_t max_new) {
  return n_tokens >= 0 && n_requests >= 0 && q_heads > 0 && kv_heads > 0 && q_heads % kv_heads == 0 &&
         head_dim > 0 && head_dim <= 128 && head_dim % 16 == 0 && max_len >= 0 && max_new >= 0;
}

}  // namespace
}  // namespace akv

extern "C" int64_t akv_kv8_attention_workspace_bytes(int64_t n_tokens, int32_t n_requests, int32_t q_heads,
                                                     int32_t kv_heads, int32_t head_dim, int64_t max_len,
                                                     int64_t max_new) {
  using namespace akv;
  if (!sizes_ok(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len, max_new)) return -1;
  return largest_bytes(n_tokens, q_heads, kv_heads, head_dim, max_len, max_new);
}

extern "C" int akv_kv8_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t dtype,
                                 const void* k_buffer, const void* v_buffer, int32_t format, int64_t k_stride_slot,
                                 int64_t k_stride_head, int64_t v_stride_slot, int64_t v_stride_head,
                                 int64_t pool_slots, const float* k_scales, const float* v_scales,
                                 int32_t scale_block, int64_t ks_stride_block, int64_t ks_stride_head,
                                 int64_t vs_stride_block, int64_t vs_stride_head, int64_t n_tokens,
                                 int32_t n_requests, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                 const void* qo_indptr, const void* kv_indptr, int32_t indptr_dtype,
                                 const int32_t* kv_indices, int64_t table_stride, int64_t table_width,
                                 int32_t page_size, const uint64_t* tree_mask, int64_t mask_stride,
                                 int32_t mask_words, const int32_t* key_starts, int32_t first_keys,
                                 const float* sinks, float scale, void* out, int32_t out_dtype, int64_t out_stride_t,
                                 int64_t out_stride_h, int64_t max_len, int64_t max_new, void* workspace,
                                 int64_t workspace_bytes, const int32_t* status, void* stream) {
  using namespace akv;
  if (n_tokens < 0 || n_requests < 0 || max_len < 0 || max_new < 0 || pool_slots < 0 || table_width < 0 ||
      table_stride < 0 || mask_words < 0 || first_keys < 0)
    return fail(AKV_EINVAL, "akv_kv8_attention: negative size");
  if (n_tokens == 0 || n_requests == 0) return AKV_OK;
  if (head_dim < 16 || head_dim > 128 || head_dim % 16)
    return fail(AKV_EINVAL, "akv_kv8_attention: head_dim %d (multiples of 16 up to 128)", head_dim);
  if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0)
    return fail(AKV_EINVAL, "akv_kv8_attention: %d q heads over %d KV heads", q_heads, kv_heads);
  if (dtype != AKV_BF16 && dtype != AKV_F16) return fail(AKV_EINVAL, "akv_kv8_attention: q must be bf16 or fp16");
  if (format != AKV_E4M3 && format != AKV_E5M2)
    return fail(AKV_EINVAL, "akv_kv8_attention: the cache must be e4m3 or e5m2");
  if (out_dtype != dtype && out_dtype != AKV_F32)
    return fail(AKV_EINVAL, "akv_kv8_attention: the output must have q's type or be f32");
  if (scale_block < 1 || scale_block > 64 || (scale_block & (scale_block - 1)))
    return fail(AKV_EINVAL, "akv_kv8_attention: scale_block %d (powers of two up to 64)", scale_block);
  if (!valid_index_dtype(indptr_dtype)) return fail(AKV_EINVAL, "akv_kv8_attention: indptrs must be int32 or int64");
  if (page_size < 1) return fail(AKV_EINVAL, "akv_kv8_attention: page_size must be positive");
  if (table_stride == 0 && page_size != 1)
    return fail(AKV_EINVAL, "akv_kv8_attention: pages need a block table (a list holds one slot per key)");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(AKV_EINVAL, "akv_kv8_attention: scale must be positive and finite");
  // (an empty pool or list need not have an address: every key is a hole then)
  if (!q || (pool_slots > 0 && (!k_buffer || !v_buffer || !k_scales || !v_scales)) || !qo_indptr || !kv_indptr ||
      (table_width > 0 && !kv_indices) || !out || !workspace)
    return fail(AKV_EINVAL, "akv_kv8_attention: null device pointer");
  if ((q_stride_t | q_stride_h) % 8 != 0 ||
      (k_stride_slot | k_stride_head | v_stride_slot | v_stride_head) % 16 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_buffer) |
        reinterpret_cast<uintptr_t>(v_buffer) | reinterpret_cast<uintptr_t>(workspace)) & 15) != 0)
    return fail(AKV_EINVAL, "akv_kv8_attention: q, K and V rows and the workspace must be 16-byte aligned");
  if (pool_slots > 0xffffffffLL || (k_stride_slot | v_stride_slot) >> 31 || n_tokens > 0x7f000000LL / q_heads ||
      static_cast<int64_t>(n_requests) * kv_heads > 0x7fffffffLL / 4096)
    return fail(AKV_EINVAL, "akv_kv8_attention: batch too large");
  const Launch p = plan(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len, max_new);
  const int64_t need = partial_bytes(p, n_tokens, q_heads);
  if (workspace_bytes < need)
    return fail(AKV_EINVAL, "akv_kv8_attention: workspace holds %lld bytes, needs %lld",
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  Kv8Args a{};
  a.t.q = q;
  a.t.q_st = q_stride_t;
  a.t.q_sh = q_stride_h;
  a.t.k = static_cast<const char*>(k_buffer);
  a.t.v = static_cast<const char*>(v_buffer);
  a.t.k_ss = k_stride_slot;
  a.t.k_sh = k_stride_head;
  a.t.v_ss = v_stride_slot;
  a.t.v_sh = v_stride_head;
  a.t.pool_slots = pool_slots;
  a.t.qo_indptr = qo_indptr;
  a.t.kv_indptr = kv_indptr;
  a.t.kv_indices = kv_indices;
  a.t.table_stride = table_stride;
  a.t.table_width = table_width;
  a.t.mask = tree_mask;
  a.t.mask_stride = mask_stride;
  a.t.mask_words = mask_words;
  a.t.key_starts = key_starts;
  a.t.sinks = sinks;
  a.t.gate = status;
  a.t.scale_log2 = scale * kLog2e;
  a.t.out = out;
  a.t.o_st = out_stride_t;
  a.t.o_sh = out_stride_h;
  a.t.owner = static_cast<int32_t*>(workspace);
  a.t.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + owner_bytes(n_tokens, q_heads));
  a.t.part_ml = a.t.part_o + 2ll * kGroups * p.block_rows * p.d;
  a.t.n_tokens = n_tokens;
  a.t.max_len = max_len;
  a.t.n_requests = n_requests;
  a.t.q_heads = q_heads;
  a.t.kv_heads = kv_heads / p.heads;
  a.t.group = q_heads / kv_heads * p.heads;
  a.t.head_dim = head_dim;
  a.t.page_size = page_size;
  a.t.row_blocks = p.row_blocks;
  a.t.whole = p.whole;
  a.t.indptr64 = indptr_dtype == AKV_I64;
  a.t.out_f32 = out_dtype == AKV_F32;
  a.t.out_vectors = (out_stride_t | out_stride_h) % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(out) % (out_dtype == AKV_F32 ? 16 : 8) == 0;
  a.t.paged = table_stride != 0;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.ks_sb = ks_stride_block;
  a.ks_sh = ks_stride_head;
  a.vs_sb = vs_stride_block;
  a.vs_sh = vs_stride_head;
  a.log2_block = __builtin_ctz(static_cast<uint32_t>(scale_block));
  a.first_keys = first_keys;
  a.block_rows = p.block_rows;
  hipStream_t st = as_stream(stream);
  if (dtype == AKV_F16) return format == AKV_E5M2 ? launch<_Float16, true>(a, p, st) : launch<_Float16, false>(a, p, st);
  return format == AKV_E5M2 ? launch<__bf16, true>(a, p, st) : launch<__bf16, false>(a, p, st);
}
