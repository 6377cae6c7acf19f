// The paged key/value cache held in 4 bits: block tables and slot maps from
// request lengths (shmt_page_plan), rows into the cache (shmt_page_set) and
// out of it (shmt_page_fetch). The attention that reads it is in
// paged_attention.hip.
#include "common.h"
#include "paged_dev.h"
#include "paged_host.h"
#include "wave.h"

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
  int64_t *first_free;  // scratch: [requests]
};

__device__ __forceinline__ int64_t plan_len(const void *p, int64_t i, int bytes) {
  const int64_t v = load_int(p, i, bytes);
  return v < 0 ? 0 : v;
}

// Token counts and page needs of all requests, summed in front of each: one workgroup, 1024 requests a step.
__global__ __launch_bounds__(1024) void page_plan_scan_kernel(PlanArgs a) {
  __shared__ uint64_t lds[32];
  const int64_t page = int64_t{1} << a.log2_page;
  uint64_t tokens = 0, taken = 0;
  for (int64_t base = 0; base < a.requests; base += 1024) {
    const int64_t i = base + threadIdx.x;
    int64_t c = 0, n = 0;
    if (i < a.requests) {
      c = plan_len(a.cached, i, a.len_bytes);
      n = plan_len(a.fresh, i, a.len_bytes);
    }
    const int64_t need = ((c + n + page - 1) >> a.log2_page) - ((c + page - 1) >> a.log2_page);
    uint64_t sum_n, sum_need;
    const uint64_t at_n = block_exclusive_scan<uint64_t, 1024>(n, lds, &sum_n);
    __syncthreads();
    const uint64_t at_need = block_exclusive_scan<uint64_t, 1024>(need, lds, &sum_need);
    __syncthreads();
    if (i < a.requests) {
      a.starts[i] = static_cast<int32_t>(tokens + at_n);
      a.kv_lens[i] = static_cast<int32_t>(c + n);
      a.first_free[i] = static_cast<int64_t>(taken + at_need);
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

// Page p of request b after the step; -1 where there is none.
__device__ __forceinline__ int64_t planned_page(const PlanArgs &a, int64_t b, int64_t p, int64_t have) {
  if (p >= a.width) return -1;
  if (p < have) return a.table[b * a.table_stride + p];
  const int64_t f = a.first_free[b] + p - have;
  return f < a.n_free ? a.free_pages[f] : -1;
}

__global__ __launch_bounds__(256) void page_plan_tokens_kernel(PlanArgs a) {
  const int64_t page = int64_t{1} << a.log2_page;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  const int64_t total = a.counts[0];
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < a.max_tokens; t += stride) {
    int64_t pos = -1, slot = -1;
    if (t < total) {
      int64_t lo = 0, hi = a.requests - 1;  // the last request that starts at t or before
      while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (a.starts[mid] <= t) lo = mid; else hi = mid - 1;
      }
      const int64_t c = plan_len(a.cached, lo, a.len_bytes);
      pos = c + t - a.starts[lo];
      const int64_t at = planned_page(a, lo, pos >> a.log2_page, (c + page - 1) >> a.log2_page);
      slot = at < 0 ? -1 : (at << a.log2_page) + (pos & (page - 1));
    }
    a.positions[t] = static_cast<int32_t>(pos);
    a.slots[t] = slot;
  }
}

// The new entries of the block table, a wave per request.
__global__ __launch_bounds__(256) void page_plan_table_kernel(PlanArgs a) {
  const int64_t page = int64_t{1} << a.log2_page;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 4;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave; b < a.requests; b += stride) {
    const int64_t c = plan_len(a.cached, b, a.len_bytes), n = plan_len(a.fresh, b, a.len_bytes);
    const int64_t have = (c + page - 1) >> a.log2_page;
    int64_t end = (c + n + page - 1) >> a.log2_page;
    if (end > a.width) end = a.width;
    for (int64_t p = have + lane_id(); p < end; p += kWave)
      a.table[b * a.table_stride + p] = static_cast<int32_t>(planned_page(a, b, p, have));
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
    const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    const vec a = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4 *>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<f32x4 *>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    vec a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = static_cast<T>(x[i]);
    *reinterpret_cast<vec *>(p) = a;
  }
}

// Eight values a lane, DIM / 8 lanes a row, four lanes a block of 32 that shares a scale.
template <typename T, int DIM>
__global__ __launch_bounds__(256) void page_set_kernel(RowsArgs a) {
  constexpr int kLanes = DIM / 8;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  const int64_t all = a.tokens * a.v.kv_heads * 2 * kLanes;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += stride) {
    const int piece = static_cast<int>(i % kLanes);
    const int64_t row = i / kLanes;
    const int head = static_cast<int>(row % a.v.kv_heads);
    const int64_t th = row / a.v.kv_heads;
    const int which = static_cast<int>(th & 1);
    const int64_t token = th >> 1;
    const int64_t slot = load_int(a.slots, token, a.slot_bytes);
    if (slot < 0 || slot >> a.v.log2_page >= a.v.pages) continue;  // the same for all lanes of a row
    const T *src = which ? static_cast<const T *>(a.values) + token * a.value_token + head * a.value_head
                         : static_cast<const T *>(a.keys) + token * a.key_token + head * a.key_head;
    float x[8];
    load8(src + piece * 8, x);
    // the largest magnitude, compared as bits, so that "not a number" comes out on top
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1)));
    most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2)));
    // The smallest power of two with most < 7 * 2^e: nothing is cut by more than half the step at its place (6 is
    // the largest code, 7 the middle between it and the 8 that there is not).
    const bool broken = most >= 0x7f800000u;
    const int e = max(static_cast<int>((most + 0x200000u) >> 23) - 2, 0);
    const float s = scale_operand(static_cast<uint32_t>(e));
    uint32_t codes = 0;
    if (!broken) {
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], s, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], s, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], s, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], s, 3);
    }
    const int64_t at = slot >> a.v.log2_page, page = int64_t{1} << a.v.log2_page, off = slot & (page - 1);
    const int64_t tile = head * 2 + which;
    *reinterpret_cast<uint32_t *>(a.v.cache + at * a.v.cache_stride + (tile * page + off) * (DIM / 2) + piece * 4) =
        codes;
    if ((piece & 3) == 0)
      a.v.scales[at * a.v.scales_stride + (tile * (DIM / 32) + piece / 4) * page + off] =
          static_cast<uint8_t>(broken ? 255 : e);
  }
}

template <typename T, int DIM>
__global__ __launch_bounds__(256) void page_fetch_kernel(RowsArgs a) {
  constexpr int kLanes = DIM / 8;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256;
  const int64_t all = a.tokens * a.v.kv_heads * 2 * kLanes;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += stride) {
    const int piece = static_cast<int>(i % kLanes);
    const int64_t row = i / kLanes;
    const int head = static_cast<int>(row % a.v.kv_heads);
    const int64_t th = row / a.v.kv_heads;
    const int which = static_cast<int>(th & 1);
    const int64_t token = th >> 1;
    const int64_t slot = load_int(a.slots, token, a.slot_bytes);
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (slot >= 0 && slot >> a.v.log2_page < a.v.pages) {
      const int64_t at = slot >> a.v.log2_page, page = int64_t{1} << a.v.log2_page, off = slot & (page - 1);
      const int64_t tile = head * 2 + which;
      const uint32_t codes = *reinterpret_cast<const uint32_t *>(
          a.v.cache + at * a.v.cache_stride + (tile * page + off) * (DIM / 2) + piece * 4);
      const float s =
          scale_operand(a.v.scales[at * a.v.scales_stride + (tile * (DIM / 32) + piece / 4) * page + off]);
      const f32x2 p0 = decode2_f32<0>(codes, s), p1 = decode2_f32<1>(codes, s), p2 = decode2_f32<2>(codes, s),
                  p3 = decode2_f32<3>(codes, s);
      x[0] = p0[0], x[1] = p0[1], x[2] = p1[0], x[3] = p1[1], x[4] = p2[0], x[5] = p2[1], x[6] = p3[0], x[7] = p3[1];
    }
    T *dst = which ? static_cast<T *>(const_cast<void *>(a.values)) + token * a.value_token + head * a.value_head
                   : static_cast<T *>(const_cast<void *>(a.keys)) + token * a.key_token + head * a.key_head;
    store8(dst + piece * 8, x);
  }
}

template <typename T>
int launch_rows(const RowsArgs &a, int dim, bool set, hipStream_t s) {
  const int64_t lanes = a.tokens * a.v.kv_heads * 2 * (dim / 8);
  const dim3 grid(grid_for(lanes, 256, 256 * 32)), block(256);
  switch (dim) {
    case 64:
      if (set) hipLaunchKernelGGL((page_set_kernel<T, 64>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((page_fetch_kernel<T, 64>), grid, block, 0, s, a);
      break;
    case 128:
      if (set) hipLaunchKernelGGL((page_set_kernel<T, 128>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((page_fetch_kernel<T, 128>), grid, block, 0, s, a);
      break;
    default:
      if (set) hipLaunchKernelGGL((page_set_kernel<T, 256>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((page_fetch_kernel<T, 256>), grid, block, 0, s, a);
  }
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
  SHMT_REQUIRE(n <= (int64_t{1} << 40) / (int64_t{c->kv_heads} * c->dim), "too many rows in one call");
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

int64_t shmt_page_plan_scratch_bytes(int64_t requests) { return requests > 0 ? requests * 8 : 0; }

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
  if (scratch_bytes < shmt_page_plan_scratch_bytes(requests) || (requests > 0 && !scratch)) {
    set_error("scratch too small: %lld bytes", static_cast<long long>(scratch_bytes));
    return SHMT_ENOMEM;
  }
  const PlanArgs a{cached_lens, new_lens, len_bytes, requests, block_table, width, table_stride,
                   free_pages, n_free, log2_page, max_tokens, query_starts, kv_lens, positions,
                   slots, counts, static_cast<int64_t *>(scratch)};
  hipStream_t s = as_stream(stream);
  hipLaunchKernelGGL(page_plan_scan_kernel, dim3(1), dim3(1024), 0, s, a);
  if (requests > 0 && width > 0)
    hipLaunchKernelGGL(page_plan_table_kernel, dim3(grid_for(requests, 4)), dim3(256), 0, s, a);
  if (max_tokens > 0)
    hipLaunchKernelGGL(page_plan_tokens_kernel, dim3(grid_for(max_tokens, 256)), dim3(256), 0, s, a);
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
