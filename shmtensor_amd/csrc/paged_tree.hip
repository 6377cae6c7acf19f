// Trees of drafted tokens over the paged key/value cache: a step's trees numbered for the attention (shmt_page_tree), and the
// path that the model agrees with kept, its rows moved to where they would lie without the rest (shmt_page_keep).
#include "common.h"
#include "paged_dev.h"
#include "paged_host.h"
#include "wave.h"

#include <algorithm>

namespace shmt {

// Rows in front of the first request's and behind the last one's, as two ranges [0, lo) and [hi, tokens).
struct NoRequest {
  int64_t lo, hi;
};
__device__ __forceinline__ NoRequest rows_of_no_request(const void *starts, int len_bytes, int64_t requests, int64_t tokens) {
  if (requests == 0) return {tokens, tokens};
  const int64_t lo = min(max(load_int(starts, 0, len_bytes), int64_t{0}), tokens);
  return {lo, min(max(load_int(starts, requests, len_bytes), lo), tokens)};
}

// ---- page_tree ------------------------------------------------------------------
// A node's four words: its number in preorder (a node before its children, siblings and roots in ascending order), the size of
// its subtree, its depth, the least depth from it to the request's last node. Node j is i or above it if and only if
// 0 <= number[i] - number[j] < size[j]: two words a token and one a row say what a row of the attention sees, however large the
// tree is.
struct TreeArgs {
  const int32_t *parents;
  const void *starts, *kv_lens;
  int len_bytes;
  int64_t requests, tokens;
  int4 *nodes;
  int32_t *positions;
};

// A parent that is not in front of its child is none.
__device__ __forceinline__ int parent_of(const TreeArgs &a, int64_t first_row, int i, int n) {
  if (i >= n) return -1;
  const int p = a.parents[first_row + i];
  return p >= 0 && p < i ? p : -1;
}

__device__ __forceinline__ void put_node(const TreeArgs &a, const Request &r, int i, int number, int size, int depth, int least) {
  a.nodes[r.first_row + i] = make_int4(number, size, depth, least);
  a.positions[r.first_row + i] = r.before + depth;
}

// Of 64 nodes, one a lane: which of them are the lane's own or above it, `p` being the parent's lane or -1.
__device__ __forceinline__ uint64_t lanes_above(int p, bool there) {
  const int lane = lane_id();
  uint64_t above = there ? uint64_t{1} << lane : 0;
  int jump = p;
  while (__ballot(jump >= 0)) {  // twice as many generations a turn
    const int at = jump >= 0 ? jump : lane;
    const uint64_t more = static_cast<uint64_t>(shfl64(static_cast<int64_t>(above), at));
    const int next = __shfl(jump, at, kWave);
    above |= jump >= 0 ? more : 0;
    jump = jump >= 0 ? next : -1;
  }
  return above;
}

// The sum of x over the lane's own and those above it.
__device__ __forceinline__ int sum_above(int p, int x) {
  const int lane = lane_id();
  int jump = p;
  while (__ballot(jump >= 0)) {
    const int at = jump >= 0 ? jump : lane;
    const int more = __shfl(x, at, kWave), next = __shfl(jump, at, kWave);
    x += jump >= 0 ? more : 0;
    jump = jump >= 0 ? next : -1;
  }
  return x;
}

// The sum of `size` over the lanes in front that have the same parent.
__device__ __forceinline__ int earlier_siblings(int p, int size, int lanes) {
  const int lane = lane_id();
  int sum = 0;
  for (int s = 0; s < lanes; ++s) {
    const int p_s = __builtin_amdgcn_readlane(p, s), size_s = __builtin_amdgcn_readlane(size, s);
    sum += p_s == p && s < lane ? size_s : 0;
  }
  return sum;
}

// The least x from the lane on.
__device__ __forceinline__ int least_from(int x) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int y = __shfl_down(x, d, kWave);
    x = lane_id() + d < kWave ? min(x, y) : x;
  }
  return x;
}

constexpr int kNoDepth = 0x7fffffff;

// A tree of up to 64 nodes, a lane each.
__device__ __forceinline__ void small_tree(const TreeArgs &a, const Request &r, int p) {
  const int lane = lane_id(), n = r.queries;
  const uint64_t above = lanes_above(p, lane < n);
  int size = 0;
  for (int j = 0; j < n; ++j) {
    const int below = __popcll(__ballot(above >> j & 1));
    size = lane == j ? below : size;
  }
  const int depth = __popcll(above) - 1;
  const int number = sum_above(p, earlier_siblings(p, size, n)) + depth;
  const int least = least_from(lane < n ? depth : kNoDepth);
  if (lane < n) put_node(a, r, lane, number, size, depth, least);
}

// Four words a node that the lanes of one wave hand to each other: in LDS, or in the result itself, past the first-level cache.
struct TreeInLds {
  int (*word)[4];
  __device__ int get(int i, int w) const { return word[i][w]; }
  __device__ void put(int i, int w, int v) const { word[i][w] = v; }
  __device__ void add(int i, int w, int v) const { atomicAdd(&word[i][w], v); }
  __device__ void fence() const { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"), __builtin_amdgcn_wave_barrier(); }
};
struct TreeInMemory {
  int *word;
  __device__ int get(int i, int w) const {
    return __hip_atomic_load(word + int64_t{4} * i + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ void put(int i, int w, int v) const {
    __hip_atomic_store(word + int64_t{4} * i + w, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ void add(int i, int w, int v) const {
    __hip_atomic_fetch_add(word + int64_t{4} * i + w, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ void fence() const { __threadfence(); }
};
enum : int { kNumber, kSize, kDepth, kTaken };  // kTaken: nodes below the earlier children

// A larger tree, by one wave, 64 nodes at a time: parents lie in front, so sizes come from the last nodes to the first, numbers
// and depths from the first to the last. What crosses the 64 goes through `m`.
template <typename Memory>
__device__ void large_tree(const TreeArgs &a, const Request &r, Memory m) {
  const int lane = lane_id(), n = r.queries;
  const int last = (n - 1) / kWave * kWave;
  for (int i = lane; i < n; i += kWave) m.put(i, kSize, 0), m.put(i, kTaken, 0);
  m.fence();
  for (int base = last; base >= 0; base -= kWave) {
    const int i = base + lane, p = parent_of(a, r.first_row, i, n);
    const uint64_t above = lanes_above(p >= base ? p - base : -1, i < n);
    const int weight = i < n ? 1 + m.get(i, kSize) : 0;  // itself and what later nodes brought
    int size = 0;
    for (int j = 0; j < kWave; ++j) {
      const uint64_t above_j = static_cast<uint64_t>(lane64(static_cast<int64_t>(above), j));
      const int weight_j = __builtin_amdgcn_readlane(weight, j);
      size += above_j >> lane & 1 ? weight_j : 0;
    }
    if (i < n) m.put(i, kSize, size);
    if (p >= 0 && p < base) m.add(p, kSize, size);
    m.fence();
  }
  int roots = 0;  // nodes below earlier roots
  for (int base = 0; base < n; base += kWave) {
    const int i = base + lane, p = parent_of(a, r.first_row, i, n), near = p >= base ? p - base : -1;
    const int size = i < n ? m.get(i, kSize) : 0;
    const int before = (p >= 0 ? m.get(p, kTaken) : roots) + earlier_siblings(p, size, kWave);
    int number = before + (p >= 0 ? 1 : 0), depth = p >= 0 ? 1 : 0;
    if (p >= 0 && p < base) number += m.get(p, kNumber), depth += m.get(p, kDepth);
    number = sum_above(near, number);
    depth = sum_above(near, depth);
    int all = p < 0 ? size : 0;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) all += __shfl_xor(all, d, kWave);
    roots += all;
    m.fence();  // kTaken has been read
    if (i < n) m.put(i, kNumber, number), m.put(i, kDepth, depth);
    if (p >= 0) m.add(p, kTaken, size);
    m.fence();
  }
  int least = kNoDepth;
  for (int base = last; base >= 0; base -= kWave) {
    const int i = base + lane;
    int number = 0, size = 0, depth = 0;
    if (i < n) number = m.get(i, kNumber), size = m.get(i, kSize), depth = m.get(i, kDepth);
    const int mine = min(least_from(i < n ? depth : kNoDepth), least);
    least = __builtin_amdgcn_readfirstlane(mine);
    if (i < n) put_node(a, r, i, number, size, depth, mine);
  }
}

constexpr int kTreeLds = 1024;  // nodes

// A wave takes a request of up to 64 nodes; the larger ones of a workgroup's four are done by all of it (a chain, as a prompt
// is one), or by its first wave.
__global__ __launch_bounds__(256) void page_tree_kernel(TreeArgs a) {
  __shared__ int words[kTreeLds][4];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const NoRequest none = rows_of_no_request(a.starts, a.len_bytes, a.requests, a.tokens);
  for (int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x; i < none.lo + a.tokens - none.hi; i += int64_t{gridDim.x} * 256) {
    const int64_t row = i < none.lo ? i : i - none.lo + none.hi;
    a.nodes[row] = make_int4(-1, -1, -1, -1);
    a.positions[row] = -1;
  }
  for (int64_t b0 = int64_t{blockIdx.x} * 4; b0 < a.requests; b0 += int64_t{gridDim.x} * 4) {
    bool large = false;
    if (b0 + wave < a.requests) {
      const Request r = load_request(a.starts, a.kv_lens, a.len_bytes, a.tokens, b0 + wave);
      large = r.queries > kWave;
      if (!large && r.queries > 0) small_tree(a, r, parent_of(a, r.first_row, lane, r.queries));
    }
    if (!__syncthreads_or(large)) continue;
    for (int w = 0; w < 4 && b0 + w < a.requests; ++w) {
      const Request r = load_request(a.starts, a.kv_lens, a.len_bytes, a.tokens, b0 + w);
      const int n = r.queries;
      if (n <= kWave) continue;
      bool other = false;
      for (int i = threadIdx.x; i < n; i += 256) other |= parent_of(a, r.first_row, i, n) != i - 1;
      if (!__syncthreads_or(other)) {
        for (int i = threadIdx.x; i < n; i += 256) put_node(a, r, i, i, n - i, i, i);
      } else if (wave == 0) {
        if (n <= kTreeLds) large_tree(a, r, TreeInLds{words});
        else large_tree(a, r, TreeInMemory{reinterpret_cast<int *>(a.nodes + r.first_row)});
      }
      __syncthreads();
    }
  }
}

// ---- page_keep ------------------------------------------------------------------

struct KeepArgs {
  PagedView v;
  int64_t layers, cache_layer, scales_layer;  // strides in bytes
  int log2_pieces;                            // pieces of 16 bytes in a row's codes
  int blocks;                                 // of 32 values in a row
  const int32_t *table;
  int64_t width, table_stride;
  const void *starts, *kv_lens;
  int len_bytes;
  int64_t requests, rows;
  const int32_t *parents;
  const void *tokens, *picked;
  int token_bytes;
  const int32_t *given;
  int32_t *counts, *path;
  void *next;
  int splits;  // workgroups of a request
};

__device__ __forceinline__ int64_t slot_of(const KeepArgs &a, int64_t b, int64_t token) {
  const int64_t at = token >> a.v.log2_page;
  if (token < 0 || at >= a.width) return -1;
  const int64_t page = a.table[b * a.table_stride + at];
  return page >= 0 && page < a.v.pages ? (page << a.v.log2_page) + (token & ((1 << a.v.log2_page) - 1)) : -1;
}

constexpr int kMoves = 256;  // of a round

// A request's path and moves are found by the first wave of each of its workgroups, 64 nodes at a time in one sweep: children lie
// behind their parents, and the first that fits is taken. All rows of a layer's keys (or values) of one head are moved by one
// wave, places ascending: place k is written after the rows for places up to k have been read, which lie at k or behind it.
__global__ __launch_bounds__(256) void page_keep_kernel(KeepArgs a) {
  __shared__ int64_t src[kMoves], dst[kMoves];
  __shared__ int moves, done;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const NoRequest none = rows_of_no_request(a.starts, a.len_bytes, a.requests, a.rows);
  for (int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x; i < none.lo + a.rows - none.hi; i += int64_t{gridDim.x} * 256)
    a.path[i < none.lo ? i : i - none.lo + none.hi] = -1;
  const int64_t b = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  if (b >= a.requests) return;
  const Request r = load_request(a.starts, a.kv_lens, a.len_bytes, a.rows, b);
  const int n = r.queries;
  if (n == 0) {
    if (split == 0 && threadIdx.x == 0) a.counts[b] = 0, store_int(a.next, b, a.token_bytes, -1);
    return;
  }
  const int given = a.given ? min(max(a.given[b], 1), n) : 1;
  if (split == 0)
    for (int i = threadIdx.x; i < given; i += 256) a.path[r.first_row + i] = i;
  int at = given - 1, count = given, base = given;
  int64_t want = load_int(a.picked, r.first_row + at, a.token_bytes);
  for (;;) {
    if (wave == 0) {
      int listed = 0;
      while (base < n && listed < kMoves) {
        const int i = base + lane;
        int p = -1;
        int64_t token = 0, pick = 0;
        if (i < n) {
          p = a.parents[r.first_row + i];
          token = load_int(a.tokens, r.first_row + i, a.token_bytes);
          pick = load_int(a.picked, r.first_row + i, a.token_bytes);
        }
        while (listed < kMoves) {
          const uint64_t fits = __ballot(i < n && i > at && p == at && token == want);
          if (!fits) {
            base += kWave;
            break;
          }
          const int l = __builtin_ctzll(fits);
          at = base + l;
          want = lane64(pick, l);
          if (lane == 0) {
            if (split == 0) a.path[r.first_row + count] = at;
            if (at != count) {
              src[listed] = slot_of(a, b, int64_t{r.before} + at);
              dst[listed] = slot_of(a, b, int64_t{r.before} + count);
            }
          }
          listed += at != count;
          ++count;
        }
      }
      if (lane == 0) moves = listed, done = base >= n;
    }
    __syncthreads();
    const int m = moves;
    const bool last = done;
    const int64_t tiles = a.layers * a.v.kv_heads * 2;
    const int page = 1 << a.v.log2_page;
    for (int64_t t = split * 4 + wave; m > 0 && t < tiles; t += a.splits * 4) {
      const int64_t layer = t / (2 * a.v.kv_heads), part = t % (2 * a.v.kv_heads);  // head and keys or values
      uint8_t *codes = a.v.cache + layer * a.cache_layer + ((part << a.v.log2_page << a.log2_pieces) << 4);
      uint8_t *scales = a.v.scales + layer * a.scales_layer + (part * a.blocks << a.v.log2_page);
      const int rows = kWave >> a.log2_pieces, piece = lane & ((1 << a.log2_pieces) - 1);
      for (int k0 = 0; k0 < m; k0 += rows) {
        const int k = k0 + (lane >> a.log2_pieces);
        const int64_t s = k < m ? src[k] : -1, d = k < m ? dst[k] : -1;
        if (s < 0 || d < 0) continue;
        const int64_t from = (s >> a.v.log2_page) * a.v.cache_stride + ((s & (page - 1)) << a.log2_pieces << 4) + 16 * piece;
        const int64_t to = (d >> a.v.log2_page) * a.v.cache_stride + ((d & (page - 1)) << a.log2_pieces << 4) + 16 * piece;
        *reinterpret_cast<uint4 *>(codes + to) = *reinterpret_cast<const uint4 *>(codes + from);
      }
      const int each = kWave / a.blocks, block = lane % a.blocks;
      for (int k0 = 0; k0 < m; k0 += each) {
        const int k = k0 + lane / a.blocks;
        const int64_t s = k < m ? src[k] : -1, d = k < m ? dst[k] : -1;
        if (s < 0 || d < 0) continue;
        scales[(d >> a.v.log2_page) * a.v.scales_stride + block * page + (d & (page - 1))] =
            scales[(s >> a.v.log2_page) * a.v.scales_stride + block * page + (s & (page - 1))];
      }
    }
    __syncthreads();
    if (last) break;
  }
  if (split != 0 || wave != 0) return;
  if (lane == 0) a.counts[b] = count, store_int(a.next, b, a.token_bytes, want);
  for (int i = count + lane; i < n; i += kWave) a.path[r.first_row + i] = -1;
}

}  // namespace shmt

using namespace shmt;

extern "C" {

int shmt_page_tree(const int32_t *parents, const void *query_starts, const void *kv_lens, int len_bytes, int64_t requests,
                   int64_t tokens, int32_t *nodes, int32_t *positions, void *stream) {
  SHMT_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 31), "the number of nodes must be in [0, 2^31)");
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(width_ok(len_bytes), "query_starts and kv_lens can only be int32 or int64");
  if (tokens == 0) return SHMT_OK;
  SHMT_REQUIRE(parents && nodes && positions, "parents, nodes or positions is null");
  SHMT_REQUIRE(requests == 0 || (query_starts && kv_lens), "query_starts or kv_lens is null");
  SHMT_REQUIRE((reinterpret_cast<int64_t>(nodes) & 15) == 0, "nodes has to begin on 16 bytes");
  const TreeArgs a{parents, query_starts, kv_lens, len_bytes, requests, tokens, reinterpret_cast<int4 *>(nodes), positions};
  hipLaunchKernelGGL(page_tree_kernel, dim3(grid_for(std::max<int64_t>(requests, 1), 4, 65536)), dim3(256), 0, as_stream(stream), a);
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

int shmt_page_keep(const shmt_paged_cache *cache, int bits, int64_t layers, int64_t cache_layer_stride,
                   int64_t scales_layer_stride, const int32_t *block_table, int64_t width, int64_t table_stride,
                   const void *query_starts, const void *kv_lens, int len_bytes, int64_t requests, int64_t rows,
                   const int32_t *parents, const void *tokens, const void *picked, int token_bytes, const int32_t *given,
                   int32_t *counts, int32_t *path, void *next, void *stream) {
  PagedView v;
  const int rc = paged_view(cache, bits, &v);
  if (rc != SHMT_OK) return rc;
  SHMT_REQUIRE(layers >= 0 && layers <= 65535, "the number of layers must be in [0, 65535]");
  SHMT_REQUIRE(((cache_layer_stride | scales_layer_stride) & 15) == 0, "every layer has to begin on 16 bytes");
  const int64_t values = int64_t{cache->kv_heads} * 2 * cache->page * cache->dim;  // of a page
  SHMT_REQUIRE(layers <= 1 || cache->pages == 0 || (cache_layer_stride >= values * bits / 8 && scales_layer_stride >= values / 32),
               "layers overlap");
  SHMT_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), "the number of nodes must be in [0, 2^31)");
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(width >= 0 && width <= (int64_t{1} << 30) / cache->page,
               "the block table holds too many tokens: more than 2^30 a request");
  SHMT_REQUIRE(width_ok(len_bytes), "query_starts and kv_lens can only be int32 or int64");
  SHMT_REQUIRE(width_ok(token_bytes), "tokens and picked can only be int32 or int64");
  SHMT_REQUIRE(requests == 0 || (query_starts && kv_lens && counts && next), "query_starts, kv_lens, counts or next is null");
  SHMT_REQUIRE(requests == 0 || width == 0 || (block_table && table_stride >= width), "block_table is null or narrow");
  SHMT_REQUIRE(rows == 0 || (parents && tokens && picked && path), "parents, tokens, picked or path is null");
  if (requests == 0 && rows == 0) return SHMT_OK;
  KeepArgs a{v, layers, cache_layer_stride, scales_layer_stride, 0, cache->dim / 32, block_table, width, table_stride,
             query_starts, kv_lens, len_bytes, requests, rows, parents, tokens, picked, token_bytes, given, counts, path, next, 1};
  while (16 << a.log2_pieces < cache->dim * bits / 8) ++a.log2_pieces;
  if (v.pages == 0) a.width = 0;
  // workgroups of a request: each has to find the path first, so no more than fill the card, and four tiles for each wave
  const int64_t tiles = layers * cache->kv_heads * 2;
  a.splits = static_cast<int>(std::max<int64_t>(1, std::min((tiles + 15) / 16, 2048 / std::max<int64_t>(requests, 1))));
  const int64_t groups = std::max<int64_t>(requests, 1) * a.splits;
  SHMT_REQUIRE(groups < (int64_t{1} << 24), "too many requests in one call");
  hipLaunchKernelGGL(page_keep_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, as_stream(stream), a);
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
