// Metadata of a forward's new tokens from request lengths (gfx950).
//
// For request b, with L = seq_lens[b] ranks of which the last n = new_lens[b]
// are new, and its registry row (raw_ids, positions, prompt, active, next_pos,
// side row; zeros: an ordinary request), as in decode_meta.hip
//   raw(i)  = i < active ? raw_ids[i] : prompt + i - active      (ordinary: i)
//   slot(i) = row[raw(i)]
//   pos(i)  = i < active ? positions[i] : next_pos + i - active  (ordinary: i)
// the call writes
//   qo_indptr, kv_indptr   cumulative sums of n and L
//   slot_map[qo + i]       slot(L - n + i), -1 behind the last token
//   positions[qo + i]      pos(L - n) + depth(i), without parents pos(L - n + i);
//                          0 behind the last token
//   block_tables[b][j]     slot(j P) / P for j P < L, -1 behind
//   tree_mask[qo + i]      bits of the request's new tokens: i and its ancestors
//   window_mask[qo + i]    those whose position is at least positions[qo + i] - window
//   window_starts[qo + i]  first rank of [0, L - n) whose position is at least
//                          positions[qo + i] - window
// where depth(i) is the length of i's path through `parents` (so an ancestor's
// position is as many less as it is levels up).  Without them token i follows
// i - 1; behind the registry's active ranks its position is one more, among them
// (a chunk of a prompt with dropped spans) it may be further.
//
// One launch.  Grid (token blocks + table blocks, B + 1): the first workgroups
// of request b share its tokens, the others its block table; row B fills what
// lies behind the last token.  A table entry is two dependent loads (raw id,
// row entry), four chains of them in flight per thread.  Bound by such round trips:
// one request of 4096 ranks 3.6 us, 32 of 20k with a page per rank, trees of 16 and
// a window 8.4 us (7.7 MB), 64 of 2k to 64k with pages of 16 8.0 us.  A token walks
// to its root by itself, so a tree's masks cost the sum of its depths.
#include "common.h"

namespace akv {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
// Most workgroups of a request, four times as many in batches of up to kSmallBatch
// (us: one request of 65536 tokens, 16 groups 8.0, 64 4.5; 64 of 2048 tokens, 4.9 and
// 8.4, most of them idle; a table of one request of 10^6 ranks, 64 groups 11.8, 256
// 5.5; of 64 requests of 65536, 10.3 and 10.8).
constexpr int kMaxTokenBlocks = 16, kMaxTableBlocks = 64, kSmallBatch = 16;
constexpr int kStagedParents = 2048;  // nodes of a tree kept in LDS; later ones read global memory

struct MapArgs {
  const int64_t* registry;
  const int32_t* table;
  int64_t row_stride, table_width;
  const void* rows;
  const void* seq_lens;
  const void* new_lens;
  void* qo_indptr;
  void* kv_indptr;
  void* slot_map;
  void* positions;
  int32_t* block_tables;
  int64_t block_stride, block_width;
  const int32_t* parents;
  uint64_t* tree_mask;
  uint64_t* window_mask;
  int64_t tree_stride, near_stride;  // words between two tokens' masks
  int32_t* window_starts;
  int64_t window;
  const int32_t* gate;
  int64_t n_tokens;
  int32_t n_requests, page_size, tree_words, near_words, token_blocks;
  bool rows64, lens64, indptr64, slots64, pos64;
};

// One request's row, positions and ranks.
struct Request {
  const int32_t* raw_ids;  // nullptr: an ordinary request
  const int32_t* positions;
  const int32_t* row;
  int64_t width;  // entries of the row (of a side row: not known, no bound)
  int32_t prompt, active, next_pos;
  int64_t len, fresh;  // ranks, and how many of them are new

  __device__ __forceinline__ int64_t raw_of(int64_t i) const {
    if (!raw_ids) return i;
    return i < active ? raw_ids[i] : prompt + i - active;
  }
  __device__ __forceinline__ int32_t slot_at(int64_t raw) const { return raw >= 0 && raw < width ? row[raw] : -1; }
  __device__ __forceinline__ int64_t pos_of(int64_t i) const {
    if (!raw_ids) return i;
    return i < active ? positions[i] : next_pos + i - active;
  }
};

__device__ __forceinline__ void lengths_of(const MapArgs& a, int64_t b, int64_t* len, int64_t* fresh) {
  const int64_t l = load_index(a.seq_lens, a.lens64, b), n = load_index(a.new_lens, a.lens64, b);
  *len = l > 0 ? l : 0;
  *fresh = n > 0 ? (n < *len ? n : *len) : 0;
}

__device__ __forceinline__ Request request_of(const MapArgs& a, int b) {
  Request r;
  lengths_of(a, b, &r.len, &r.fresh);
  // (a request without ranks, as a padded batch's last ones, may name any row)
  const int64_t row = load_index(a.rows, a.rows64, b), id = r.len > 0 ? row : 0;
  const int64_t* entry = a.registry + id * 6;
  r.raw_ids = reinterpret_cast<const int32_t*>(entry[0]);
  r.positions = reinterpret_cast<const int32_t*>(entry[1]);
  r.prompt = static_cast<int32_t>(entry[2]);
  r.active = static_cast<int32_t>(entry[3]);
  r.next_pos = static_cast<int32_t>(entry[4]);
  const int64_t side = entry[5];
  r.row = side ? reinterpret_cast<const int32_t*>(side) : a.table + id * a.row_stride;
  r.width = side ? INT64_MAX : a.table_width;
  return r;
}

// Sums of L and n over the requests before `end`, in every thread.
__device__ __forceinline__ void sums_before(const MapArgs& a, int end, int64_t* len, int64_t* fresh) {
  __shared__ int64_t part[2][kThreads / 64];
  int64_t l = 0, n = 0;
  for (int i = threadIdx.x; i < end; i += kThreads) {
    int64_t li, ni;
    lengths_of(a, i, &li, &ni);
    l += li;
    n += ni;
  }
  for (int off = 32; off; off >>= 1) {
    l += __shfl_xor(l, off);
    n += __shfl_xor(n, off);
  }
  if ((threadIdx.x & 63) == 0) {
    part[0][threadIdx.x >> 6] = l;
    part[1][threadIdx.x >> 6] = n;
  }
  __syncthreads();
  *len = *fresh = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    *len += part[0][w];
    *fresh += part[1][w];
  }
}

// Bits lo .. hi of word w of a bit row.
__device__ __forceinline__ uint64_t bits_of(int64_t lo, int64_t hi, int64_t w) {
  const int64_t a = lo - 64 * w, b = hi - 64 * w;
  if (a > 63 || b < 0) return 0;
  const uint64_t up = b >= 63 ? ~0ull : (2ull << b) - 1;
  return a <= 0 ? up : up & ~((1ull << a) - 1);
}

__device__ __forceinline__ void token_maps(const MapArgs& a, int b) {
  __shared__ int32_t staged[kStagedParents];
  __shared__ int64_t keys[kThreads];  // positions from the first key inside a root's window on
  const Request r = request_of(a, b);
  int64_t len0, tok0;
  sums_before(a, b, &len0, &tok0);
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0 && blockIdx.x == 0) {
    if (b == 0) {
      store_index(a.qo_indptr, a.indptr64, 0, 0);
      store_index(a.kv_indptr, a.indptr64, 0, 0);
    }
    store_index(a.qo_indptr, a.indptr64, b + 1, tok0 + r.fresh);
    store_index(a.kv_indptr, a.indptr64, b + 1, len0 + r.len);
  }
  // tokens past the outputs' capacity (a caller error) are left out
  const int64_t room = a.n_tokens > tok0 ? a.n_tokens - tok0 : 0;
  const int64_t n = r.fresh < room ? r.fresh : room;
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * kThreads;
  if (begin >= n) return;
  const int64_t old = r.len - r.fresh;
  if (a.parents) {
    for (int64_t i = tid; i < n && i < kStagedParents; i += kThreads) staged[i] = a.parents[tok0 + i];
    __syncthreads();
  }
  // the path upwards; a parent that is no earlier node is none
  auto parent_of = [&](int64_t i) -> int64_t {
    const int64_t p = i < kStagedParents ? staged[i] : a.parents[tok0 + i];
    return p >= 0 && p < i ? p : -1;
  };
  const int64_t root = r.pos_of(old);
  int64_t first = 0;  // first key inside the window of a token of depth 0
  if (a.window_starts && r.raw_ids) {
    first = first_at_least([&](int32_t i) -> int64_t { return r.pos_of(i); }, static_cast<int32_t>(old),
                           root - a.window, lane);
    if (first + tid < old) keys[tid] = r.pos_of(first + tid);
    __syncthreads();
  }
  for (int64_t i = begin + tid; i < n; i += static_cast<int64_t>(a.token_blocks) * kThreads) {
    const int64_t t = tok0 + i;
    store_index(a.slot_map, a.slots64, t, r.slot_at(r.raw_of(old + i)));
    uint64_t* tree = a.tree_mask ? a.tree_mask + t * a.tree_stride : nullptr;
    uint64_t* near = a.window_mask ? a.window_mask + t * a.near_stride : nullptr;
    int64_t pos;
    if (!a.parents) {
      pos = r.pos_of(old + i);
      int64_t lo = i - a.window;
      if (near && r.raw_ids && old < r.active) {
        // among active ranks: positions ascend, maybe by more than one
        int64_t hi = i;
        lo = lo < 0 ? 0 : lo;
        while (lo < hi) {
          const int64_t mid = (lo + hi) >> 1;
          if (r.pos_of(old + mid) < pos - a.window) lo = mid + 1; else hi = mid;
        }
      }
      for (int w = 0; tree && w < a.tree_words; ++w) tree[w] = bits_of(0, i, w);
      for (int w = 0; near && w < a.near_words; ++w) near[w] = bits_of(lo, i, w);
    } else {
      // ancestors have smaller numbers, so the words fill from the last one down
      int64_t w = i >> 6, at = i, depth = 0;
      uint64_t all = 0, close = 0;
      for (int64_t u = w + 1; tree && u < a.tree_words; ++u) tree[u] = 0;
      for (int64_t u = w + 1; near && u < a.near_words; ++u) near[u] = 0;
      for (;;) {
        const uint64_t bit = 1ull << (at & 63);
        all |= bit;
        if (depth <= a.window) close |= bit;
        const int64_t up = parent_of(at);
        const int64_t below = up < 0 ? -1 : up >> 6;
        for (; w > below; --w) {
          if (tree && w < a.tree_words) tree[w] = all;
          if (near && w < a.near_words) near[w] = close;
          all = close = 0;
        }
        if (up < 0) break;
        at = up;
        ++depth;
      }
      pos = root + depth;
    }
    store_index(a.positions, a.pos64, t, pos);
    if (a.window_starts) {
      const int64_t lower = pos - a.window;
      int64_t lo;
      if (!r.raw_ids) {
        lo = lower < 0 ? 0 : (lower < old ? lower : old);
      } else {
        // positions ascend, so the first key is at most pos - root ranks on
        lo = first;
        int64_t hi = first + (pos - root) < old ? first + (pos - root) : old;
        while (lo < hi) {
          const int64_t mid = (lo + hi) >> 1;
          const int64_t at = mid - first < kThreads ? keys[mid - first] : r.pos_of(mid);
          if (at < lower) lo = mid + 1; else hi = mid;
        }
      }
      a.window_starts[t] = static_cast<int32_t>(lo);
    }
  }
}

__device__ __forceinline__ void block_table(const MapArgs& a, int b) {
  const Request r = request_of(a, b);
  const int64_t step = static_cast<int64_t>(gridDim.x - a.token_blocks) * kThreads;
  int32_t* out = a.block_tables + b * a.block_stride;
  const uint32_t page = a.page_size;
  auto emit = [&](int64_t j, int32_t slot) { out[j] = slot < 0 ? -1 : static_cast<int32_t>(slot / page); };
  int64_t j = static_cast<int64_t>(blockIdx.x - a.token_blocks) * kThreads + threadIdx.x;
  int64_t pages = (r.len + page - 1) / page;
  if (pages > a.block_width) pages = a.block_width;
  for (; j + (kUnroll - 1) * step < pages; j += kUnroll * step) {
    int64_t raw[kUnroll];
    int32_t slot[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = r.raw_of((j + u * step) * page);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) slot[u] = r.slot_at(raw[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) emit(j + u * step, slot[u]);
  }
  for (; j < pages; j += step) emit(j, r.slot_at(r.raw_of(j * page)));
  for (; j < a.block_width; j += step) out[j] = -1;
}

// Behind the last token: no slot, position 0, masks that see nothing.
__device__ __forceinline__ void padding(const MapArgs& a) {
  int64_t len, tokens;
  sums_before(a, a.n_requests, &len, &tokens);
  if (a.n_requests == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
    store_index(a.qo_indptr, a.indptr64, 0, 0);
    store_index(a.kv_indptr, a.indptr64, 0, 0);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t t = tokens + static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; t < a.n_tokens; t += step) {
    store_index(a.slot_map, a.slots64, t, -1);
    store_index(a.positions, a.pos64, t, 0);
    if (a.window_starts) a.window_starts[t] = 0;
    for (int w = 0; a.tree_mask && w < a.tree_words; ++w) a.tree_mask[t * a.tree_stride + w] = 0;
    for (int w = 0; a.window_mask && w < a.near_words; ++w) a.window_mask[t * a.near_stride + w] = 0;
  }
}

__global__ void __launch_bounds__(kThreads) step_maps_kernel(const MapArgs a) {
  if (gated(a.gate)) return;
  const int b = blockIdx.y;
  if (b == a.n_requests)
    padding(a);
  else if (static_cast<int>(blockIdx.x) < a.token_blocks)
    token_maps(a, b);
  else
    block_table(a, b);
}

}  // namespace
}  // namespace akv

extern "C" int akv_step_maps(const int64_t* registry, const int32_t* table, int64_t row_stride, int64_t table_width,
                             const void* rows, int32_t rows_dtype, const void* seq_lens, const void* new_lens,
                             int32_t lens_dtype, int32_t n_requests, void* qo_indptr, void* kv_indptr,
                             int32_t indptr_dtype, int64_t n_tokens, void* slot_map, int32_t slots_dtype,
                             void* positions, int32_t positions_dtype, int32_t* block_tables, int64_t block_stride,
                             int64_t block_width, int32_t page_size, const int32_t* parents, uint64_t* tree_mask,
                             int64_t tree_stride, int32_t tree_words, int64_t window, uint64_t* window_mask,
                             int64_t window_stride, int32_t window_words, int32_t* window_starts,
                             const int32_t* status, void* stream) {
  using namespace akv;
  if (n_requests < 0 || n_tokens < 0 || block_width < 0 || tree_words < 0 || window_words < 0 || table_width < 0)
    return fail(AKV_EINVAL, "akv_step_maps: negative size");
  if (n_requests > 65534) return fail(AKV_EINVAL, "akv_step_maps: batch of %d requests exceeds one launch", n_requests);
  if (page_size < 1) return fail(AKV_EINVAL, "akv_step_maps: page_size must be positive");
  if (!valid_index_dtype(rows_dtype) || !valid_index_dtype(lens_dtype) || !valid_index_dtype(indptr_dtype) ||
      !valid_index_dtype(slots_dtype) || !valid_index_dtype(positions_dtype))
    return fail(AKV_EINVAL, "akv_step_maps: index vectors must be int32 or int64");
  if ((window_mask || window_starts) && (window < 0 || window >= (1ll << 31)))
    return fail(AKV_EINVAL, "akv_step_maps: the window's outputs need a window of [0, 2^31)");
  if (!qo_indptr || !kv_indptr || (n_tokens > 0 && (!slot_map || !positions)) ||
      (n_requests > 0 && (!registry || (table_width > 0 && !table) || !rows || !seq_lens || !new_lens)))
    return fail(AKV_EINVAL, "akv_step_maps: null device pointer");
  MapArgs a{};
  a.registry = registry;
  a.table = table;
  a.row_stride = row_stride;
  a.table_width = table_width;
  a.rows = rows;
  a.seq_lens = seq_lens;
  a.new_lens = new_lens;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.slot_map = slot_map;
  a.positions = positions;
  a.block_tables = block_width > 0 ? block_tables : nullptr;
  a.block_stride = block_stride;
  a.block_width = block_width;
  a.parents = parents;
  a.tree_mask = tree_words > 0 ? tree_mask : nullptr;
  a.window_mask = window_words > 0 ? window_mask : nullptr;
  a.tree_stride = tree_stride;
  a.near_stride = window_stride;
  a.window_starts = window_starts;
  a.window = window;
  a.gate = status;
  a.n_tokens = n_tokens;
  a.n_requests = n_requests;
  a.page_size = page_size;
  a.tree_words = tree_words;
  a.near_words = window_words;
  a.rows64 = rows_dtype == AKV_I64;
  a.lens64 = lens_dtype == AKV_I64;
  a.indptr64 = indptr_dtype == AKV_I64;
  a.slots64 = slots_dtype == AKV_I64;
  a.pos64 = positions_dtype == AKV_I64;
  const int more = n_requests <= kSmallBatch ? 4 : 1;
  unsigned blocks = 0;
  if (a.block_tables) {
    const int64_t want = (block_width + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    blocks = static_cast<unsigned>(want < more * kMaxTableBlocks ? want : more * kMaxTableBlocks);
  }
  // a thread's tokens follow each other: four of them where a request has most
  const int64_t shares = (n_tokens + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  const int64_t most = more * kMaxTokenBlocks;
  a.token_blocks = static_cast<int32_t>(shares < 1 ? 1 : shares < most ? shares : most);
  const dim3 grid(a.token_blocks + blocks, static_cast<unsigned>(n_requests) + 1);
  hipLaunchKernelGGL(step_maps_kernel, grid, dim3(kThreads), 0, as_stream(stream), a);
  return check_launch("akv_step_maps");
}
