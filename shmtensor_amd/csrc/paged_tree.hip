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

// Of 64 nodes, one a lane, `p` being the parent's lane or -1: x (and y) become their sums over the lane's own and those above it.
__device__ __forceinline__ void sum_above(int p, int &x, int *y = nullptr) {
  const int lane = lane_id();
  int jump = p;
  while (__ballot(jump >= 0)) {  // twice as many generations a turn
    const int at = jump >= 0 ? jump : lane;
    const int more = __shfl(x, at, kWave), more_y = y ? __shfl(*y, at, kWave) : 0, next = __shfl(jump, at, kWave);
    x += jump >= 0 ? more : 0;
    if (y) *y += jump >= 0 ? more_y : 0;
    jump = jump >= 0 ? next : -1;
  }
}

// From the last of 64 nodes to the first: each gives its size to its parent, the lane p - base, and to the siblings in front of it.
__device__ __forceinline__ void give_sizes(int p, int base, int lanes, int &size, int &later) {
  const int lane = lane_id();
  for (int s = lanes - 1; s >= 0; --s) {
    const int p_s = __builtin_amdgcn_readlane(p, s), size_s = __builtin_amdgcn_readlane(size, s);
    size += lane == p_s - base ? size_s : 0;
    later += p == p_s && lane < s ? size_s : 0;
  }
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

// A tree of up to 64 nodes, a lane each. A node's number is what lies in front of it: below its parent, in front of that, ...
__device__ __forceinline__ void small_tree(const TreeArgs &a, const Request &r, int p) {
  const int lane = lane_id(), n = r.queries;
  int size = lane < n ? 1 : 0, later = 0;
  give_sizes(p, 0, n, size, later);
  const int of_parent = __shfl(size, max(p, 0), kWave);
  const int before = (p >= 0 ? of_parent - 1 : n) - size - later;  // earlier children of the same parent
  int both = (before + (p >= 0 ? 1 : 0)) | 1 << 16;  // number and depth, which are below 64
  sum_above(p, both);
  const int depth = (both >> 16) - 1;
  const int least = least_from(lane < n ? depth : kNoDepth);
  if (lane < n) put_node(a, r, lane, both & 0xffff, size, depth, least);
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
enum : int { kNumber, kSize, kDepth, kLater };  // kLater: what is below the later children of the same parent

// A larger tree, by one wave, 64 nodes at a time: parents lie in front, so sizes come from the last nodes to the first, numbers
// and depths from the first to the last. What crosses the 64 goes through `m`; until a node's turn comes, its size there is what
// its children have brought so far, and its number its parent.
//
// Requests whose rows overlap, where starts descend, write into each other's words: what is read as a parent is made one again
// before it is used, so that they reach nobody else's and every loop ends.
__device__ __forceinline__ int parent_again(int p, int i, int n) { return i < n && p >= 0 && p < i ? p : -1; }

template <typename Memory>
__device__ void large_tree(const TreeArgs &a, const Request &r, Memory m) {
  const int lane = lane_id(), n = r.queries;
  const int last = (n - 1) / kWave * kWave;
  for (int i = lane; i < n; i += kWave) m.put(i, kSize, 0), m.put(i, kNumber, parent_of(a, r.first_row, i, n));
  m.fence();
  int roots = 0;  // nodes below later roots
  for (int base = last; base >= 0; base -= kWave) {
    const int i = base + lane, p = parent_again(i < n ? m.get(i, kNumber) : -1, i, n);
    int size = i < n ? 1 + m.get(i, kSize) : 0, later = p >= 0 ? m.get(p, kSize) : roots;
    give_sizes(p, base, kWave, size, later);
    roots += static_cast<int>(wave_last(wave_inclusive_scan(static_cast<uint32_t>(p < 0 ? size : 0))));
    m.fence();  // sizes have been read
    if (i < n) m.put(i, kSize, size), m.put(i, kLater, later);
    if (p >= 0 && p < base) m.add(p, kSize, size);
    m.fence();
  }
  for (int base = 0; base < n; base += kWave) {
    const int i = base + lane, p = parent_again(i < n ? m.get(i, kNumber) : -1, i, n), near = p >= base ? p - base : -1;
    int number = 0, depth = 0;
    if (i < n) {
      const int before = (p >= 0 ? m.get(p, kSize) - 1 : n) - m.get(i, kSize) - m.get(i, kLater);
      number = before + (p >= 0 ? 1 : 0), depth = p >= 0 ? 1 : 0;
      if (p >= 0 && p < base) number += m.get(p, kNumber), depth += m.get(p, kDepth);
    }
    sum_above(near, number, &depth);
    if (i < n) m.put(i, kNumber, number), m.put(i, kDepth, depth);
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

// Whether a request's nodes are one chain, as a prompt's are: node i's parent is i - 1.
__device__ __forceinline__ bool is_chain(const TreeArgs &a, const Request &r) {
  constexpr int kEach = 8;  // loads on their way
  const int n = r.queries;
  for (int base = 0; base < n; base += kEach * kWave) {
    int p[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) p[k] = a.parents[r.first_row + min(base + k * kWave + lane_id(), n - 1)];
    bool other = false;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = min(base + k * kWave + lane_id(), n - 1);
      other |= (p[k] >= 0 && p[k] < i ? p[k] : -1) != i - 1;
    }
    if (__ballot(other)) return false;
  }
  return true;
}

// A wave a request, a workgroup a wave: what there is to do is two dependent reads and some 400 instructions, so a launch is
// quickest when no wave waits for another. Four requests to a workgroup, the larger ones one after the other by all of it, took
// 8.8 us instead of 6.5 for 481 trees of up to 64 nodes and 20 prompts of 400; 6 requests of up to 16 nodes 4.3 and 3.8.
__global__ __launch_bounds__(kWave) void page_tree_kernel(TreeArgs a) {
  __shared__ int words[kTreeLds][4];
  const int lane = lane_id();
  const NoRequest none = rows_of_no_request(a.starts, a.len_bytes, a.requests, a.tokens);
  for (int64_t i = int64_t{blockIdx.x} * kWave + lane; i < none.lo + a.tokens - none.hi; i += int64_t{gridDim.x} * kWave) {
    const int64_t row = i < none.lo ? i : i - none.lo + none.hi;
    a.nodes[row] = make_int4(-1, -1, -1, -1);
    a.positions[row] = -1;
  }
  for (int64_t b = blockIdx.x; b < a.requests; b += gridDim.x) {
    const Request r = load_request(a.starts, a.kv_lens, a.len_bytes, a.tokens, b);
    const int n = r.queries;
    if (n <= kWave) {
      if (n > 0) small_tree(a, r, parent_of(a, r.first_row, lane, n));
    } else if (is_chain(a, r)) {
      for (int i = lane; i < n; i += kWave) put_node(a, r, i, i, n - i, i, i);
    } else if (n <= kTreeLds) {
      large_tree(a, r, TreeInLds{words});
    } else {
      large_tree(a, r, TreeInMemory{reinterpret_cast<int *>(a.nodes + r.first_row)});
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

// Where tile t begins, a layer's keys or values of one head: the codes and the scales of page 0.
struct KeepTile {
  uint8_t *codes, *scales;
};
__device__ __forceinline__ KeepTile keep_tile(const KeepArgs &a, uint32_t t) {
  const uint32_t parts = 2 * a.v.kv_heads, layer = t / parts, part = t - layer * parts;
  return {a.v.cache + layer * a.cache_layer + (int64_t{part} << a.v.log2_page << a.log2_pieces << 4),
          a.v.scales + layer * a.scales_layer + (int64_t{part} * a.blocks << a.v.log2_page)};
}

// x[i] and y[i], on their way together.
__device__ __forceinline__ void load_both(const void *x, const void *y, int64_t i, int bytes, int64_t *a, int64_t *b) {
  if (bytes == 8) {
    const int64_t u = static_cast<const int64_t *>(x)[i], v = static_cast<const int64_t *>(y)[i];
    *a = u, *b = v;
  } else {
    const int32_t u = static_cast<const int32_t *>(x)[i], v = static_cast<const int32_t *>(y)[i];
    *a = u, *b = v;
  }
}

constexpr int kMoves = 256;  // of a round

// A request's path and moves are found by the first wave of each of its workgroups, 64 nodes at a time in one sweep: children lie
// behind their parents, and the first that fits is taken. All rows of a layer's keys (or values) of one head are moved by one
// wave, places ascending: place k is written after the rows for places up to k have been read, which lie at k or behind it.
// Bound by five dependent reads (lengths, nodes, table, rows, and their writes), so nothing is moved one after the other that
// can be on its way together: 120 requests of 24 to 64 nodes, 16 layers of 8 heads of 128 in 8 bits, 10 us on the GPU; a tile at
// a time 14.4, with a wave's lane 0 looking up the slots 12, with twice as many workgroups, that do not all fit, 11.3.
__global__ __launch_bounds__(256) void page_keep_kernel(KeepArgs a) {
  __shared__ int64_t src[kMoves], dst[kMoves];
  __shared__ int moves, done;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  auto clear_rows_of_no_request = [&] {
    if (split != 0) return;
    const NoRequest none = rows_of_no_request(a.starts, a.len_bytes, a.requests, a.rows);
    const int64_t groups = gridDim.x / a.splits;
    for (int64_t i = b * 256 + threadIdx.x; i < none.lo + a.rows - none.hi; i += groups * 256)
      a.path[i < none.lo ? i : i - none.lo + none.hi] = -1;
  };
  if (b >= a.requests) return clear_rows_of_no_request();
  const Request r = load_request(a.starts, a.kv_lens, a.len_bytes, a.rows, b);
  const int n = r.queries;
  if (n == 0) {
    if (split == 0 && threadIdx.x == 0) a.counts[b] = 0, store_int(a.next, b, a.token_bytes, -1);
    return clear_rows_of_no_request();
  }
  const int given = a.given ? min(max(a.given[b], 1), n) : 1;
  if (split == 0)
    for (int i = threadIdx.x; i < given; i += 256) a.path[r.first_row + i] = i;
  int at = given - 1, count = given, base = at;  // the path's end; its nodes; the 64 that are looked at
  int64_t want = 0;
  for (;;) {
    if (wave == 0) {
      int listed = 0;
      while (base < n && listed < kMoves) {
        const int i = base + lane;
        int p = -1;
        int64_t token = 0, pick = 0;
        if (i < n) {
          p = a.parents[r.first_row + i];
          load_both(a.tokens, a.picked, r.first_row + i, a.token_bytes, &token, &pick);
        }
        if (base == given - 1) want = lane64(pick, 0);  // the first 64 begin with the path's end, and fill no list
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
            if (at != count) src[listed] = at, dst[listed] = count;
          }
          listed += at != count;
          ++count;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int k = lane; k < listed; k += kWave) {  // tokens to slots
        const int64_t from = slot_of(a, b, r.before + src[k]), to = slot_of(a, b, r.before + dst[k]);
        src[k] = from, dst[k] = to;
      }
      if (lane == 0) moves = listed, done = base >= n;
    }
    __syncthreads();
    const int m = moves;
    const bool last = done;
    const uint32_t tiles = static_cast<uint32_t>(a.layers * a.v.kv_heads * 2);
    // As many rows at a time as a wave has lanes for their codes and for their scales; four tiles' are on their way together.
    const int rows = min(kWave >> a.log2_pieces, kWave / a.blocks), l = a.v.log2_page, in_page = (1 << l) - 1;
    const int piece = lane & ((1 << a.log2_pieces) - 1), block = lane % a.blocks;
    const uint32_t stride = a.splits * 4;
    for (uint32_t t0 = split * 4 + wave; m > 0 && t0 < tiles; t0 += 4 * stride) {
      KeepTile tile[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) tile[j] = keep_tile(a, t0 + j * stride < tiles ? t0 + j * stride : t0);  // or the first again
      for (int k0 = 0; k0 < m; k0 += rows) {
        const int k = k0 + (lane >> a.log2_pieces), k_scale = k0 + lane / a.blocks;
        const int64_t s = src[min(k, m - 1)], d = dst[min(k, m - 1)];
        const int64_t s_scale = src[min(k_scale, m - 1)], d_scale = dst[min(k_scale, m - 1)];
        const bool move = lane >> a.log2_pieces < rows && k < m && s >= 0 && d >= 0;
        const bool move_scale = lane / a.blocks < rows && k_scale < m && s_scale >= 0 && d_scale >= 0;
        const int64_t from = (s >> l) * a.v.cache_stride + ((s & in_page) << a.log2_pieces << 4) + 16 * piece;
        const int64_t to = (d >> l) * a.v.cache_stride + ((d & in_page) << a.log2_pieces << 4) + 16 * piece;
        const int64_t from_scale = (s_scale >> l) * a.v.scales_stride + (block << l) + (s_scale & in_page);
        const int64_t to_scale = (d_scale >> l) * a.v.scales_stride + (block << l) + (d_scale & in_page);
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        u32x4 codes[4];
        uint8_t scale[4];
        if (move) {
#pragma unroll
          for (int j = 0; j < 4; ++j) codes[j] = *reinterpret_cast<const u32x4 *>(tile[j].codes + from);
        }
        if (move_scale) {
#pragma unroll
          for (int j = 0; j < 4; ++j) scale[j] = tile[j].scales[from_scale];
        }
        if (move) {
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4 *>(tile[j].codes + to) = codes[j];
        }
        if (move_scale) {
#pragma unroll
          for (int j = 0; j < 4; ++j) tile[j].scales[to_scale] = scale[j];
        }
      }
    }
    __syncthreads();
    if (last) break;
  }
  clear_rows_of_no_request();
  if (split != 0 || wave != 0) return;
  if (lane == 0) a.counts[b] = count, store_int(a.next, b, a.token_bytes, want);
  for (int i = count + lane; i < n; i += kWave) a.path[r.first_row + i] = -1;
}

}  // namespace shmt

using namespace shmt;

extern "C" {

int shmt_page_tree(const int32_t *parents, const void *query_starts, const void *kv_lens, int len_bytes, int64_t requests,
                   int64_t tokens, int32_t *nodes, int32_t *positions, void *stream) {
  SHMT_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 30), "the number of nodes must be in [0, 2^30)");
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(width_ok(len_bytes), "query_starts and kv_lens can only be int32 or int64");
  if (tokens == 0) return SHMT_OK;
  SHMT_REQUIRE(parents && nodes && positions, "parents, nodes or positions is null");
  SHMT_REQUIRE(requests == 0 || (query_starts && kv_lens), "query_starts or kv_lens is null");
  SHMT_REQUIRE((reinterpret_cast<int64_t>(nodes) & 15) == 0, "nodes has to begin on 16 bytes");
  const TreeArgs a{parents, query_starts, kv_lens, len_bytes, requests, tokens, reinterpret_cast<int4 *>(nodes), positions};
  hipLaunchKernelGGL(page_tree_kernel, dim3(grid_for(std::max<int64_t>(requests, 1), 1, 65536)), dim3(kWave), 0, as_stream(stream), a);
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
  SHMT_REQUIRE(layers >= 0 && layers < (int64_t{1} << 28) / cache->kv_heads, "too many layers and heads: 2^28 or more");
  SHMT_REQUIRE(((cache_layer_stride | scales_layer_stride) & 15) == 0, "every layer has to begin on 16 bytes");
  const int64_t values = int64_t{cache->kv_heads} * 2 * cache->page * cache->dim;  // of a page
  SHMT_REQUIRE(layers <= 1 || cache->pages == 0 || (cache_layer_stride >= values * bits / 8 && scales_layer_stride >= values / 32),
               "layers overlap");
  SHMT_REQUIRE(rows >= 0 && rows < (int64_t{1} << 30), "the number of nodes must be in [0, 2^30)");
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(requests < (int64_t{1} << 24), "too many requests in one call: 2^24 or more");  // a workgroup each
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
  // workgroups of a request: each has to find the path first, so no more than the card holds, and four tiles for each wave
  const int64_t tiles = layers * cache->kv_heads * 2;
  a.splits = static_cast<int>(std::max<int64_t>(1, std::min((tiles + 15) / 16, 1024 / std::max<int64_t>(requests, 1))));
  const int64_t groups = std::max<int64_t>(requests, 1) * a.splits;
  hipLaunchKernelGGL(page_keep_kernel, dim3(static_cast<unsigned>(groups)), dim3(256), 0, as_stream(stream), a);
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
