// The glue of a round over a tree of drafted tokens: where its nodes go and what they see, and, once the model has answered, the
// walk along the nodes it agreed with and the move of their cache rows.
//
//   kern_tree_rows   depth_i = depth_parent + 1, mask_i = mask_parent | 1 << i; position base + depth_i, slot of place base + i
//   kern_tree_keep   node <- the lowest child of node with ids[child] == verify[node], from node 0, while there is one; then in
//                    every layer's pool the rows of path[i] move from place base + path[i] to base + i
//
// Both are bound by latency: a few hundred bytes a sequence, and the rows of a handful of nodes. One block holds a whole tree (up
// to 256 nodes) in shared memory. Ancestors come by doubling: every thread follows its node's jump pointer and takes over its
// mask and its pointer, so a chain of n nodes takes log2 n steps, not n. The walk asks all nodes at once, one vote a step. Every
// (sequence, layer) has a block of its own that walks again rather than wait for another launch to have walked.
//
// Measured: the walk and the move for 128 trees of up to 32 nodes in 12 layers of a bf16 cache (8 kv heads of 128) 15.4 us, where
// their bytes take 5.8 at the copy bandwidth; for three trees 7 us.
//
// The move is in place. path[i] >= i, so the place that row i is written to is never read for a later row; a thread moves the
// same bytes of every row, in the path's order, so no row is written by one thread before another has read it.
#include "common.cuh"

using namespace kern;

namespace kern {

constexpr int kMaxNodes = 256, kMaxPools = 128;
constexpr long long kFar = 1ll << 62;                       // a place that no table holds, and that its nodes can be added to
struct PoolTable {
  unsigned long long at[kMaxPools];
};

// The rows of a sequence, cu[s] to cu[s + 1] - 1; `lie`: whether they are rows of the call. If not, the bounds cut to the call's.
struct Span {
  int from, to;
  bool lie;
};
KERN_DEVICE Span span_of(const int* cu, int s, int nodes) {
  const int from = cu[s], to = cu[s + 1];
  return {min(max(from, 0), nodes), min(max(to, 0), nodes), from >= 0 && to >= from && to <= nodes};
}

// the cache slot of a sequence's token place, or -1
KERN_DEVICE long long place_slot(long long place, const int* pages, int max_pages, int page_size) {
  const long long pi = place / page_size;
  return pi < max_pages ? (long long)pages[pi] * page_size + place % page_size : -1;
}

}  // namespace kern

// grid seqs, block 256; `most` nodes of a tree (up to 256, 64 to a word). Nodes that no tree holds (of padding sequences, before the first
// sequence and behind the last, over the limit, between bounds that are none) get position 0, slot -1 and no mask.
extern "C" __global__ void __launch_bounds__(256)
    kern_tree_rows(const int* parents, const int* cu, const long long* base, const int* block_table, long long* positions, long long* slots,
                   int* seq_lens, long long* masks, int nodes, int most, int words, int max_pages, int page_size, int* err) {
  __shared__ unsigned long long mask_s[kMaxNodes][4];
  __shared__ int jump_s[kMaxNodes], depth_s[kMaxNodes];
  pdl_wait();
  const int s = blockIdx.x, i = threadIdx.x;
  const Span mine = span_of(cu, s, nodes);
  const int row0 = mine.from, all = mine.lie ? mine.to - mine.from : 0;
  if (!mine.lie && i == 0) set_error(err, ERR_BOUNDS);
  const long long b = min(base[s], kFar);
  const int n = b < 0 ? 0 : min(all, most);
  auto none = [&](int from, int to) {
    for (int x = from + i; x < to; x += blockDim.x) {
      positions[x] = 0;
      slots[x] = -1;
      for (int w = 0; w < words; ++w) masks[(size_t)x * words + w] = 0;
    }
  };
  if (i == 0) {
    if (b >= 0 && all > n) set_error(err, ERR_BOUNDS);
    seq_lens[s] = b < 0 ? 0 : (int)min(b + all, (long long)INT_MAX);
  }
  none(row0 + n, mine.to);
  if (s == 0) none(0, row0);
  if (s == (int)gridDim.x - 1) none(mine.to, nodes);
  if (n == 0) return;
  int jump = -1, depth = 0;
  unsigned long long m[4] = {0, 0, 0, 0};
  if (i < n) {
    jump = parents[row0 + i];
    if (jump < -1 || jump >= i) {
      set_error(err, ERR_BOUNDS);
      jump = -1;
    }
    depth = jump >= 0 ? 1 : 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) m[w] = (i >> 6) == w ? 1ull << (i & 63) : 0ull;
  }
  // `jump`: an ancestor, or -1 past the first; depth: steps to it; m: the nodes passed, that one not among them
  for (int span = 1; span < n; span <<= 1) {
    if (i < n) {
      jump_s[i] = jump;
      depth_s[i] = depth;
#pragma unroll
      for (int w = 0; w < 4; ++w) mask_s[i][w] = m[w];
    }
    __syncthreads();
    if (i < n && jump >= 0) {
      const int p = jump;
#pragma unroll
      for (int w = 0; w < 4; ++w) m[w] |= mask_s[p][w];
      depth += depth_s[p];
      jump = jump_s[p];
    }
    __syncthreads();
  }
  if (i < n) {
    const long long slot = place_slot(b + i, block_table + (size_t)s * max_pages, max_pages, page_size);
    if (slot < 0) set_error(err, ERR_BOUNDS);
    positions[row0 + i] = b + depth;
    slots[row0 + i] = slot < 0 ? -1 : slot;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (w < words) masks[(size_t)(row0 + i) * words + w] = (long long)m[w];
  }
}

// grid (seqs, layers), block 128; `most` as above
extern "C" __global__ void __launch_bounds__(128)
    kern_tree_keep(const __grid_constant__ PoolTable pools, const long long* ids, const int* parents, const long long* verify, const int* cu,
                   const long long* base, const int* block_table, int* count, int* path, long long* emitted, int nodes, int most, int layers,
                   int max_pages, int page_size, int hk, int d, int e4m3, int pool_pages, int* err) {
  __shared__ int path_s[kMaxNodes];
  __shared__ long long slot_s[2][kMaxNodes];
  __shared__ int len_s;
  pdl_wait();
  const int s = blockIdx.x, t = threadIdx.x;
  const Span mine = span_of(cu, s, nodes);
  const int row0 = mine.from, all = mine.lie ? mine.to - mine.from : 0;
  if (!mine.lie && t == 0) set_error(err, ERR_BOUNDS);
  const int n = min(all, most);
  const long long b = min(base[s], kFar);
  if (t < 32) {
    // lane holds nodes t, t + 32, ..: the edge into each, and whether the model agrees with it
    int par[8];
    bool hit[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = t + 32 * k;
      par[k] = i < n ? parents[row0 + i] : -1;
      hit[k] = i > 0 && i < n && par[k] >= 0 && par[k] < i && ids[row0 + i] == verify[row0 + par[k]];
    }
    int at = 0, len = n > 0 && b >= 0 ? 1 : 0;
    if (len && t == 0) path_s[0] = 0;
    while (len) {
      int next = kMaxNodes;
#pragma unroll
      for (int k = 7; k >= 0; --k)
        if (hit[k] && par[k] == at) next = t + 32 * k;
      next = __reduce_min_sync(0xffffffffu, next);
      if (next >= kMaxNodes) break;               // (next > at: the walk ends)
      if (t == 0) path_s[len] = next;
      at = next;
      ++len;
    }
    if (t == 0) len_s = len;
  }
  __syncthreads();
  const int len = len_s;
  if (blockIdx.y == 0) {
    if (t == 0) {
      count[s] = len;
      if (all > n) set_error(err, ERR_BOUNDS);
    }
    for (int i = t; i < all; i += blockDim.x) {
      path[row0 + i] = i < len ? path_s[i] : -1;
      emitted[row0 + i] = i < len ? verify[row0 + path_s[i]] : 0;
    }
    auto none = [&](int from, int to) {
      for (int i = from + t; i < to; i += blockDim.x) {
        path[i] = -1;
        emitted[i] = 0;
      }
    };
    none(row0 + all, mine.to);
    if (s == 0) none(0, row0);
    if (s == (int)gridDim.x - 1) none(mine.to, nodes);
  }
  if ((int)blockIdx.y >= layers) return;
  const int* pages = block_table + (size_t)s * max_pages;
  for (int i = t; i < len; i += blockDim.x) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long slot = place_slot(b + (k ? i : path_s[i]), pages, max_pages, page_size);
      const bool ok = slot >= 0 && slot < (long long)pool_pages * page_size;
      if (!ok) set_error(err, ERR_BOUNDS);
      slot_s[k][i] = ok ? slot : -1;
    }
  }
  __syncthreads();
  uint8_t* pool = reinterpret_cast<uint8_t*>(pools.at[blockIdx.y]);
  const int row_bytes = d * (e4m3 ? 1 : 2), pieces = row_bytes / 16, rows = 2 * hk;
  const size_t codes = (size_t)rows * page_size * row_bytes, page_bytes = codes + (e4m3 ? rows * page_size : 0);
  auto row_at = [&](long long slot, int r) { return pool + (size_t)(slot / page_size) * page_bytes + ((size_t)r * page_size + slot % page_size) * row_bytes; };
  // nodes at the head of the path that are in place already need no move
  int first = 0;
  while (first < len && path_s[first] == first) ++first;
  for (int x = t; x < rows * pieces; x += blockDim.x) {
    const int r = x / pieces, piece = x % pieces;
    for (int i0 = first; i0 < len; i0 += 4) {     // four rows in flight
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k < len && slot_s[0][i0 + k] >= 0 && KERN_CHECK(row_at(slot_s[0][i0 + k], r), row_bytes, SITE_KV_ROW))
          v[k] = *reinterpret_cast<const uint4*>(row_at(slot_s[0][i0 + k], r) + piece * 16);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k < len && slot_s[0][i0 + k] >= 0 && slot_s[1][i0 + k] >= 0 && KERN_CHECK(row_at(slot_s[1][i0 + k], r), row_bytes, SITE_KV_APPEND))
          *reinterpret_cast<uint4*>(row_at(slot_s[1][i0 + k], r) + piece * 16) = v[k];
    }
  }
  if (e4m3) {
    auto byte_at = [&](long long slot, int r) { return pool + (size_t)(slot / page_size) * page_bytes + codes + (size_t)r * page_size + slot % page_size; };
    for (int r = t; r < rows; r += blockDim.x)
      for (int i = first; i < len; ++i)
        if (slot_s[0][i] >= 0 && slot_s[1][i] >= 0) *byte_at(slot_s[1][i], r) = *byte_at(slot_s[0][i], r);
  }
}
