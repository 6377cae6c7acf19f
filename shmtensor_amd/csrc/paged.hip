// The paged key/value cache held in 4 bits: block tables and slot maps from
// request lengths (shmt_page_plan), rows into the cache (shmt_page_set) and
// out of it (shmt_page_fetch). The attention that reads it is in
// paged_attention.hip.
#include "common.h"
#include "paged_dev.h"
#include "paged_host.h"
#include "wave.h"

#include <algorithm>

namespace shmt {

// ---- plan ---------------------------------------------------------------------

struct PlanArgs {
  const void *cached, *fresh;
  int len_bytes;
  int64_t requests;
  int32_t *table;
  int64_t width, table_stride;
  const int32_t *free_pages;
  int64_t n_free;
  int log2_page;
  int64_t max_tokens;
  int32_t *starts, *kv_lens, *positions;
  int64_t *slots, *counts;
};

// A request: its tokens, and what lies in front of it in the step.
struct PlanRequest {
  int64_t cached, fresh;
  int64_t start, first_free;  // new tokens and pages needed by the requests before it
};

__device__ __forceinline__ int64_t plan_pages(const PlanArgs &a, int64_t tokens) {
  return (tokens + (int64_t{1} << a.log2_page) - 1) >> a.log2_page;
}

__device__ __forceinline__ void plan_lens(const PlanArgs &a, int64_t i, int64_t *cached, int64_t *fresh) {
  const int64_t at[1] = {i};
  const bool ok[1] = {true};
  int64_t c[1], n[1];
  load_ints(a.cached, at, ok, a.len_bytes, c);
  load_ints(a.fresh, at, ok, a.len_bytes, n);
  *cached = max(c[0], int64_t{0});
  *fresh = max(n[0], int64_t{0});
}

// Page p of a request after the step; -1 where there is none.
__device__ __forceinline__ int64_t planned_page(const PlanArgs &a, int64_t b, int64_t p, int64_t have,
                                                int64_t first_free) {
  if (p >= a.width) return -1;
  if (p < have) return a.table[b * a.table_stride + p];
  const int64_t f = first_free + p - have;
  return f < a.n_free ? a.free_pages[f] : -1;
}

// Positions and slots of new tokens t .. t + N - 1, as far as there is room; `start_of(b)` and `first_free_of(b)` are the sums in
// front of request b, `cached_of(b)` its length. N = 4 for prompts, whose tokens in a row are mostly one request's, on one
// page; N = 1 where requests have a few tokens each.
template <int N, typename Start, typename Free, typename Cached>
__device__ __forceinline__ void plan_tokens(const PlanArgs &a, int64_t t, int64_t total, bool wide, Start start_of,
                                            Free first_free_of, Cached cached_of) {
  const int64_t page = int64_t{1} << a.log2_page;
  int32_t position[N];
  int64_t slot[N];
  int64_t b = 0, last = a.requests - 1;  // the last request that starts at t or before
  while (b < last) {
    const int64_t mid = (b + last + 1) >> 1;
    if (start_of(mid) <= t) b = mid; else last = mid - 1;
  }
  int64_t at = -1, at_page = -1;  // the page of the token before, and its number in the request
#pragma unroll
  for (int i = 0; i < N; ++i) {
    position[i] = -1, slot[i] = -1;
    if (t + i >= total) continue;
    while (i > 0 && b + 1 < a.requests && start_of(b + 1) <= t + i) ++b, at_page = -1;
    const int64_t c = cached_of(b), pos = c + t + i - start_of(b);
    if (pos >> a.log2_page != at_page) {
      at_page = pos >> a.log2_page;
      at = planned_page(a, b, at_page, plan_pages(a, c), first_free_of(b));
    }
    position[i] = static_cast<int32_t>(pos);
    slot[i] = at < 0 ? -1 : (at << a.log2_page) + (pos & (page - 1));
  }
  if constexpr (N == 4)
    if (wide && t + 4 <= a.max_tokens) {
      *reinterpret_cast<int4 *>(a.positions + t) = make_int4(position[0], position[1], position[2], position[3]);
      reinterpret_cast<longlong2 *>(a.slots + t)[0] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2 *>(a.slots + t)[1] = make_longlong2(slot[2], slot[3]);
      return;
    }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (t + i < a.max_tokens) a.positions[t + i] = position[i], a.slots[t + i] = slot[i];
}

// The new table entries of request b, by `lanes` lanes.
__device__ __forceinline__ void plan_entries(const PlanArgs &a, int64_t b, const PlanRequest &r, int lane, int lanes) {
  const int64_t have = plan_pages(a, r.cached), end = min(plan_pages(a, r.cached + r.fresh), a.width);
  for (int64_t p = have + lane; p < end; p += lanes)
    a.table[b * a.table_stride + p] = static_cast<int32_t>(planned_page(a, b, p, have, r.first_free));
}

// Up to kPlanOne requests, in one launch: every workgroup adds up all lengths for itself (they are few, and it costs less than
// a second launch: 7 / 1,024 / 301 requests 3.6 / 6.5 / 7.6 us on the GPU, with sums, table and tokens in three launches 6 / 11
// / 13 us), keeps the sums in LDS and takes its share of the tokens and of the requests' table rows. No workgroup
// reads a table entry that another writes: tokens on new pages take them from the list of free pages.
constexpr int kPlanOne = 2048;

template <int N>
__global__ __launch_bounds__(256) void page_plan_one_kernel(PlanArgs a, bool wide) {
  __shared__ int64_t cached[kPlanOne], start[kPlanOne + 1], first_free[kPlanOne];
  __shared__ uint64_t scan[4];
  const int n = static_cast<int>(a.requests);
  // lengths, all in flight at once; counts to where the sums will be
  constexpr int kEach = kPlanOne / 256;
  int64_t at[kEach], c[kEach] = {}, f[kEach] = {};
  bool ok[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) at[k] = threadIdx.x + 256 * k, ok[k] = at[k] < n;
  load_ints(a.cached, at, ok, a.len_bytes, c);
  load_ints(a.fresh, at, ok, a.len_bytes, f);
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (ok[k]) {
      c[k] = max(c[k], int64_t{0}), f[k] = max(f[k], int64_t{0});
      cached[at[k]] = c[k];
      start[at[k]] = f[k];
      first_free[at[k]] = plan_pages(a, c[k] + f[k]) - plan_pages(a, c[k]);
      if (blockIdx.x == 0) a.kv_lens[at[k]] = static_cast<int32_t>(c[k] + f[k]);
    }
  __syncthreads();
  const int each = (n + 255) / 256, lo = min(static_cast<int>(threadIdx.x) * each, n), hi = min(lo + each, n);
  uint64_t tokens = 0, pages = 0;
  for (int b = lo; b < hi; ++b) tokens += start[b], pages += first_free[b];
  uint64_t all_tokens, all_pages;
  uint64_t at_token = block_exclusive_scan<uint64_t, 256>(tokens, scan, &all_tokens);
  uint64_t at_page = block_exclusive_scan<uint64_t, 256>(pages, scan, &all_pages);
  for (int b = lo; b < hi; ++b) {
    const uint64_t t = start[b], p = first_free[b];
    start[b] = at_token;
    first_free[b] = at_page;
    if (blockIdx.x == 0) a.starts[b] = static_cast<int32_t>(at_token);
    at_token += t;
    at_page += p;
  }
  if (threadIdx.x == 0) {
    start[n] = all_tokens;
    if (blockIdx.x == 0) {
      a.starts[n] = static_cast<int32_t>(all_tokens);
      a.counts[0] = static_cast<int64_t>(all_tokens);
      a.counts[1] = static_cast<int64_t>(all_pages);
    }
  }
  __syncthreads();
  const int64_t total = static_cast<int64_t>(all_tokens);
  for (int64_t t = (int64_t{blockIdx.x} * 256 + threadIdx.x) * N; t < a.max_tokens; t += int64_t{gridDim.x} * 256 * N)
    plan_tokens<N>(a, t, total, wide, [&](int64_t b) { return start[b]; }, [&](int64_t b) { return first_free[b]; },
                [&](int64_t b) { return cached[b]; });
  // 16 lanes a request
  for (int64_t b = int64_t{blockIdx.x} * 16 + threadIdx.x / 16; b < n; b += int64_t{gridDim.x} * 16)
    plan_entries(a, b, PlanRequest{cached[b], start[b + 1] - start[b], start[b], first_free[b]}, threadIdx.x % 16, 16);
}

// More requests: the sums by one workgroup, 1024 requests a step ...
__global__ __launch_bounds__(1024) void page_plan_scan_kernel(PlanArgs a, int64_t *first_free) {
  __shared__ uint64_t lds[16];
  uint64_t tokens = 0, taken = 0;
  for (int64_t base = 0; base < a.requests; base += 1024) {
    const int64_t i = base + threadIdx.x;
    int64_t c = 0, n = 0;
    if (i < a.requests) plan_lens(a, i, &c, &n);
    uint64_t sum_n, sum_need;
    const uint64_t at_n = block_exclusive_scan<uint64_t, 1024>(n, lds, &sum_n);
    const uint64_t at_need =
        block_exclusive_scan<uint64_t, 1024>(plan_pages(a, c + n) - plan_pages(a, c), lds, &sum_need);
    if (i < a.requests) {
      a.starts[i] = static_cast<int32_t>(tokens + at_n);
      a.kv_lens[i] = static_cast<int32_t>(c + n);
      first_free[i] = static_cast<int64_t>(taken + at_need);
    }
    tokens += sum_n;
    taken += sum_need;
  }
  if (threadIdx.x == 0) {
    a.starts[a.requests] = static_cast<int32_t>(tokens);
    a.counts[0] = static_cast<int64_t>(tokens);
    a.counts[1] = static_cast<int64_t>(taken);
  }
}

// ... then tokens and table rows by all.
__global__ __launch_bounds__(256) void page_plan_rest_kernel(PlanArgs a, const int64_t *first_free) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256, me = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t total = a.counts[0];
  for (int64_t t = me; t < a.max_tokens; t += stride)
    plan_tokens<1>(a, t, total, false, [&](int64_t b) { return static_cast<int64_t>(a.starts[b]); },
                   [&](int64_t b) { return first_free[b]; },
                   [&](int64_t b) { return max(load_int(a.cached, b, a.len_bytes), int64_t{0}); });
  for (int64_t b = me / 16; b < a.requests; b += stride / 16) {
    PlanRequest r;
    plan_lens(a, b, &r.cached, &r.fresh);
    r.first_free = first_free[b];
    plan_entries(a, b, r, threadIdx.x % 16, 16);
  }
}

// ---- set / fetch ----------------------------------------------------------------

struct RowsArgs {
  PagedView v;
  const void *slots;
  int slot_bytes;
  int64_t tokens;
  const void *keys, *values;  // fetch: written
  int64_t key_token, key_head, value_token, value_head;  // strides in elements
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p)),
                b = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p) + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    const vec a = __builtin_nontemporal_load(reinterpret_cast<const vec *>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4 *>(p));
    __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4 *>(p) + 1);
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    vec a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = static_cast<T>(x[i]);
    __builtin_nontemporal_store(a, reinterpret_cast<vec *>(p));
  }
}

// A workgroup takes PASSES * 2048 / DIM tokens in a row of one head's keys or values: DIM / 8 lanes a token, eight values a
// lane, four lanes a block of 32 that shares a scale. Tokens in a row mostly lie in a row in their page too, so the codes
// leave (or come) as one piece, and the scale bytes, which lie token by token, meet in one L2. All of a lane's rows are in
// flight together. Bound by HBM: 65,536 tokens of 8 heads x 128 in bfloat16 (268 MB in, 71 MB out, or the reverse) take 70 us
// to set and 55 us to fetch, 4.8 and 6.2 TB/s; a copy of 2 GiB moves 4.9. Rows are read and written past the caches, which a
// row is not read from again: without that, 81 and 90 us. With a lane for 8 values of any token in turn, and 64-bit divisions
// for its place, 90 and 94 us.
template <int DIM, int PASSES>
struct RowPlace {
  static constexpr int kLanes = DIM / 8;
  static constexpr int kPasses = PASSES;
  int head, which, piece;
  int64_t token0;  // of pass 0; 256 / kLanes tokens a pass
  int64_t slot[kPasses];  // -1: nowhere

  __device__ __forceinline__ explicit RowPlace(const RowsArgs &a) {
    const uint32_t tiles = 2 * a.v.kv_heads;
    const uint32_t tile = blockIdx.x % tiles;
    which = tile / a.v.kv_heads;
    head = tile % a.v.kv_heads;
    piece = threadIdx.x % kLanes;
    token0 = int64_t{blockIdx.x / tiles} * (PASSES * 256 / kLanes) + threadIdx.x / kLanes;
    int64_t at[kPasses];
    bool ok[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      at[p] = token0 + p * (256 / kLanes);
      ok[p] = at[p] < a.tokens;
      slot[p] = -1;
    }
    load_ints(a.slots, at, ok, a.slot_bytes, slot);
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
      if (slot[p] < 0 || slot[p] >> a.v.log2_page >= a.v.pages) slot[p] = -1;
  }
  __device__ __forceinline__ int64_t token(int p) const { return token0 + p * (256 / kLanes); }
  __device__ __forceinline__ uint32_t *codes(const RowsArgs &a, int p) const {
    const int64_t at = slot[p] >> a.v.log2_page, off = slot[p] & ((1 << a.v.log2_page) - 1);
    return reinterpret_cast<uint32_t *>(a.v.cache + at * a.v.cache_stride +
                                        (((int64_t{2} * head + which) << a.v.log2_page) + off) * (DIM / 2) + piece * 4);
  }
  __device__ __forceinline__ uint8_t *scale(const RowsArgs &a, int p) const {
    const int64_t at = slot[p] >> a.v.log2_page, off = slot[p] & ((1 << a.v.log2_page) - 1);
    return a.v.scales + at * a.v.scales_stride +
           (((int64_t{2} * head + which) * (DIM / 32) + piece / 4) << a.v.log2_page) + off;
  }
};

template <typename T, int DIM, int PASSES>
__global__ __launch_bounds__(256) void page_set_kernel(RowsArgs a) {
  const RowPlace<DIM, PASSES> r(a);
  constexpr int kPasses = PASSES;
  const T *src = r.which ? static_cast<const T *>(a.values) + r.head * a.value_head
                         : static_cast<const T *>(a.keys) + r.head * a.key_head;
  const int64_t token_stride = r.which ? a.value_token : a.key_token;
  float x[kPasses][8];
#pragma unroll
  for (int p = 0; p < kPasses; ++p)
    if (r.slot[p] >= 0) load8(src + r.token(p) * token_stride + r.piece * 8, x[p]);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    if (r.slot[p] < 0) continue;  // the same for all lanes of a row
    // the largest magnitude, compared as bits, so that "not a number" comes out on top
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[p][j]) & 0x7fffffffu);
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2)));
    // The smallest power of two with most < 7 * 2^e: nothing is cut by more than half the step at its place (6 is
    // the largest code, 7 the middle between it and the 8 that there is not).
    const bool broken = most >= 0x7f800000u;
    const int e = max(static_cast<int>((most + 0x200000u) >> 23) - 2, 0);
    const float s = scale_operand(static_cast<uint32_t>(e));
    uint32_t codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[p][0], x[p][1], s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[p][2], x[p][3], s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[p][4], x[p][5], s, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[p][6], x[p][7], s, 3);
    *r.codes(a, p) = broken ? 0u : codes;
    if ((r.piece & 3) == 0) *r.scale(a, p) = static_cast<uint8_t>(broken ? 255 : e);
  }
}

template <typename T, int DIM, int PASSES>
__global__ __launch_bounds__(256) void page_fetch_kernel(RowsArgs a) {
  const RowPlace<DIM, PASSES> r(a);
  constexpr int kPasses = PASSES;
  uint32_t codes[kPasses], scale[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    codes[p] = scale[p] = 0;
    if (r.slot[p] >= 0) codes[p] = *r.codes(a, p), scale[p] = *r.scale(a, p);
  }
  T *dst = static_cast<T *>(const_cast<void *>(r.which ? a.values : a.keys)) + r.head * a.key_head + r.piece * 8;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    if (r.token(p) >= a.tokens) continue;
    const float s = scale_operand(scale[p]);
    const f32x2 y[4] = {decode2_f32<0>(codes[p], s), decode2_f32<1>(codes[p], s), decode2_f32<2>(codes[p], s),
                        decode2_f32<3>(codes[p], s)};
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = y[j / 2][j % 2];
    store8(dst + r.token(p) * a.key_token, x);
  }
}

// 64 tokens a workgroup where that makes enough of them to fill the card, else as few as its lanes can hold. Measured, set /
// fetch, 8 heads of 128 in bfloat16, with 64 and with 16 tokens: 2,048 tokens (512 workgroups of 64) 4.3 / 4.2 and 4.1 / 4.1
// us, 4,096 tokens 5.6 / 5.0 and 6.0 / 5.3 us, 16,384 tokens 17 / 12.7 and 21 / 12.5 us; 2 heads of 256, 8,192 tokens (512)
// 7.0 / 5.4 and 6.1 / 5.2 us.
template <typename T, int DIM>
void launch_some_rows(const RowsArgs &a, bool set, hipStream_t s) {
  constexpr int kMany = DIM / 32, kOne = 2048 / DIM;  // passes for 64 tokens; tokens of one pass
  const int64_t tiles = 2 * a.v.kv_heads, many = (a.tokens + 63) / 64 * tiles, few = (a.tokens + kOne - 1) / kOne * tiles;
  const dim3 block(256);
  if (many >= 1024) {
    const dim3 grid(static_cast<unsigned>(many));
    if (set) hipLaunchKernelGGL((page_set_kernel<T, DIM, kMany>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((page_fetch_kernel<T, DIM, kMany>), grid, block, 0, s, a);
  } else {
    const dim3 grid(static_cast<unsigned>(few));
    if (set) hipLaunchKernelGGL((page_set_kernel<T, DIM, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((page_fetch_kernel<T, DIM, 1>), grid, block, 0, s, a);
  }
}

// A launch has less than 2^32 threads; more rows are more launches.
template <typename T, int DIM>
void launch_rows(const RowsArgs &all, bool set, hipStream_t s) {
  const int64_t each = ((int64_t{1} << 24) - 1) / (2 * all.v.kv_heads) * 64;
  RowsArgs a = all;
  for (int64_t t0 = 0; t0 < all.tokens; t0 += each) {
    a.tokens = std::min(each, all.tokens - t0);
    a.slots = static_cast<const char *>(all.slots) + t0 * all.slot_bytes;
    a.keys = static_cast<const T *>(all.keys) + t0 * all.key_token;
    a.values = static_cast<const T *>(all.values) + t0 * all.value_token;
    launch_some_rows<T, DIM>(a, set, s);
  }
}

template <typename T>
int launch_rows(const RowsArgs &a, int dim, bool set, hipStream_t s) {
  if (dim == 64) launch_rows<T, 64>(a, set, s);
  else if (dim == 128) launch_rows<T, 128>(a, set, s);
  else launch_rows<T, 256>(a, set, s);
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

int rows_entry(const shmt_paged_cache *c, const void *slots, int slot_bytes, int64_t n, const void *keys,
               int64_t key_token, int64_t key_head, const void *values, int64_t value_token, int64_t value_head,
               int elem_type, bool set, hipStream_t s) {
  PagedView v;
  const int rc = paged_view(c, &v);
  if (rc != SHMT_OK) return rc;
  SHMT_REQUIRE(n >= 0, "the number of rows must be >= 0");
  SHMT_REQUIRE(width_ok(slot_bytes), "slots can only be int32 or int64");
  SHMT_REQUIRE(elem_type == SHMT_F32 || elem_type == SHMT_F16 || elem_type == SHMT_BF16, "unknown element type %d",
               elem_type);
  if (n == 0) return SHMT_OK;
  SHMT_REQUIRE(slots && keys && values, "slots, keys or values is null");
  SHMT_REQUIRE(n / 64 < (int64_t{1} << 30) / c->kv_heads, "too many rows in one call");
  const int64_t esize = elem_type == SHMT_F32 ? 4 : 2;
  const int64_t bits = reinterpret_cast<int64_t>(keys) | reinterpret_cast<int64_t>(values) |
                       (key_token | key_head | value_token | value_head) * esize;
  SHMT_REQUIRE((bits & 15) == 0, "every row of keys and values has to begin on 16 bytes");
  const RowsArgs a{v, slots, slot_bytes, n, keys, values, key_token, key_head, value_token, value_head};
  if (elem_type == SHMT_F32) return launch_rows<float>(a, c->dim, set, s);
  if (elem_type == SHMT_F16) return launch_rows<_Float16>(a, c->dim, set, s);
  return launch_rows<__bf16>(a, c->dim, set, s);
}

}  // namespace shmt

using namespace shmt;

extern "C" {

int64_t shmt_page_plan_scratch_bytes(int64_t requests) { return requests > kPlanOne ? requests * 8 : 0; }

int shmt_page_plan(const void *cached_lens, const void *new_lens, int len_bytes, int64_t requests,
                   int32_t *block_table, int64_t width, int64_t table_stride, const int32_t *free_pages,
                   int64_t n_free, int page, int64_t max_tokens, int32_t *query_starts, int32_t *kv_lens,
                   int32_t *positions, int64_t *slots, int64_t *counts, void *scratch, int64_t scratch_bytes,
                   void *stream) {
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(max_tokens >= 0 && max_tokens < (int64_t{1} << 31), "max_tokens must be in [0, 2^31)");
  SHMT_REQUIRE(width >= 0 && n_free >= 0, "width and the number of free pages must be >= 0");
  SHMT_REQUIRE(width_ok(len_bytes), "lengths can only be int32 or int64");
  const int log2_page = paged_log2(page);
  SHMT_REQUIRE(log2_page >= 0, "a page must hold 16, 32, 64, 128 or 256 tokens, not %d", page);
  SHMT_REQUIRE(query_starts && counts, "query_starts or counts is null");
  SHMT_REQUIRE(requests == 0 || (cached_lens && new_lens && kv_lens), "a length array is null");
  SHMT_REQUIRE(requests == 0 || width == 0 || (block_table && table_stride >= width), "block_table is null or narrow");
  SHMT_REQUIRE(n_free == 0 || free_pages, "free_pages is null");
  SHMT_REQUIRE(max_tokens == 0 || (positions && slots), "positions or slots is null");
  if (scratch_bytes < shmt_page_plan_scratch_bytes(requests) || (requests > kPlanOne && !scratch)) {
    set_error("scratch too small: %lld bytes", static_cast<long long>(scratch_bytes));
    return SHMT_ENOMEM;
  }
  const PlanArgs a{cached_lens, new_lens, len_bytes, requests, block_table, width, table_stride,
                   free_pages, n_free, log2_page, max_tokens, query_starts, kv_lens, positions,
                   slots, counts};
  hipStream_t s = as_stream(stream);
  const bool wide = ((reinterpret_cast<int64_t>(positions) | reinterpret_cast<int64_t>(slots)) & 15) == 0;  // stores of 16 bytes
  if (requests <= kPlanOne) {
    // Measured: 1,024 requests, 2,500 tokens: 6.1 us with a token a thread, 7.7 us with four; 301 requests, 440 K tokens: 8.6
    // us and 7.2 us.
    if (max_tokens > 65536 && max_tokens / 32 > requests)
      hipLaunchKernelGGL(page_plan_one_kernel<4>, dim3(grid_for(max_tokens, 1024, 512)), dim3(256), 0, s, a, wide);
    else
      hipLaunchKernelGGL(page_plan_one_kernel<1>, dim3(grid_for(std::max(max_tokens, requests * 16), 256, 512)), dim3(256),
                         0, s, a, false);
  } else {
    int64_t *first_free = static_cast<int64_t *>(scratch);
    hipLaunchKernelGGL(page_plan_scan_kernel, dim3(1), dim3(1024), 0, s, a, first_free);
    hipLaunchKernelGGL(page_plan_rest_kernel, dim3(grid_for(std::max(max_tokens, requests * 16), 256)), dim3(256), 0, s, a,
                       first_free);
  }
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

int shmt_page_set(const shmt_paged_cache *cache, const void *slots, int slot_bytes, int64_t n, const void *keys,
                  int64_t key_token_stride, int64_t key_head_stride, const void *values, int64_t value_token_stride,
                  int64_t value_head_stride, int elem_type, void *stream) {
  return rows_entry(cache, slots, slot_bytes, n, keys, key_token_stride, key_head_stride, values, value_token_stride,
                    value_head_stride, elem_type, true, as_stream(stream));
}

int shmt_page_fetch(const shmt_paged_cache *cache, const void *slots, int slot_bytes, int64_t n, void *keys,
                    void *values, int elem_type, void *stream) {
  const int64_t head = cache ? cache->dim : 0, token = cache ? int64_t{cache->kv_heads} * cache->dim : 0;
  return rows_entry(cache, slots, slot_bytes, n, keys, token, head, values, token, head, elem_type, false,
                    as_stream(stream));
}

}  // extern "C"
