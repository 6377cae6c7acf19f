// Attention over the paged key/value cache held in 4 bits
// (shmt_page_attention).
#include "common.h"
#include "paged_dev.h"
#include "paged_host.h"
#include "wave.h"

namespace shmt {

struct AttnArgs {
  PagedView v;
  const void *query;
  int64_t query_token, query_head;
  int64_t tokens;
  int heads, group;
  const int32_t *table;
  int64_t width, table_stride;
  const void *starts, *kv_lens;
  int len_bytes;
  int64_t requests;
  float scale;
  int64_t window, sinks;
  void *out;
  float *lse;
};

// One wave for each query row and head. Scores: a token a lane, 64 at a time, with the softmax's running maximum and
// sum; the weighted values: DIM / 64 dimensions a lane.
template <typename T, int DIM>
__global__ __launch_bounds__(64) void page_attention_rows_kernel(AttnArgs a) {
  constexpr int kOwn = DIM / 64;
  __shared__ float q[DIM];
  __shared__ float weight[kWave];
  __shared__ int64_t place[kWave];
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, kvh = h / a.group;
  for (int d = lane; d < DIM; d += kWave)
    q[d] = static_cast<float>(static_cast<const T *>(a.query)[t * a.query_token + h * a.query_head + d]);
  int64_t lo = 0, hi = a.requests - 1;  // the last request that starts at t or before
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (load_int(a.starts, mid, a.len_bytes) <= t) lo = mid; else hi = mid - 1;
  }
  int64_t pos = -1;
  if (a.requests > 0) {
    const int64_t begin = load_int(a.starts, lo, a.len_bytes), end = load_int(a.starts, lo + 1, a.len_bytes);
    if (begin <= t && t < end) pos = load_int(a.kv_lens, lo, a.len_bytes) - (end - begin) + (t - begin);
  }
  const int64_t page = int64_t{1} << a.v.log2_page;
  const int64_t limit = min(pos + 1, a.width << a.v.log2_page);
  const int64_t first = a.window ? max(pos - a.window + 1, int64_t{0}) : 0;
  const int64_t sinks = min(a.sinks, first);
  float m = -__builtin_inff(), l = 0;
  float acc[kOwn] = {};
  __syncthreads();
  int64_t base = sinks > 0 ? 0 : first;
  while (base < limit) {
    const int64_t j = base + lane;
    const bool inside = base < first ? j < sinks : j < limit;
    int64_t at = -1;
    if (inside) at = a.table[lo * a.table_stride + (j >> a.v.log2_page)];
    const bool sees = at >= 0 && at < a.v.pages;
    const int64_t off = j & (page - 1);
    float s = -__builtin_inff();
    if (sees) {
      const uint8_t *row = a.v.cache + at * a.v.cache_stride + (2 * kvh * page + off) * (DIM / 2);
      const uint8_t *sc = a.v.scales + at * a.v.scales_stride + 2 * kvh * (DIM / 32) * page + off;
      s = 0;
      for (int p = 0; p < DIM / 8; ++p) {
        const uint32_t codes = reinterpret_cast<const uint32_t *>(row)[p];
        const float f = scale_operand(sc[(p / 4) * page]);
        const f32x2 x0 = decode2_f32<0>(codes, f), x1 = decode2_f32<1>(codes, f), x2 = decode2_f32<2>(codes, f),
                    x3 = decode2_f32<3>(codes, f);
        s += q[8 * p] * x0[0] + q[8 * p + 1] * x0[1] + q[8 * p + 2] * x1[0] + q[8 * p + 3] * x1[1] +
             q[8 * p + 4] * x2[0] + q[8 * p + 5] * x2[1] + q[8 * p + 6] * x3[0] + q[8 * p + 7] * x3[1];
      }
      s *= a.scale;
    }
    float top = s;
    for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float next = fmaxf(m, top);
    if (__ballot(sees)) {
      const float old = expf(m - fmaxf(next, -3.0e38f));
      const float w = sees ? expf(s - fmaxf(next, -3.0e38f)) : 0;
      float sum = w;
      for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
      l = l * old + sum;
      m = next;
      weight[lane] = w;
      place[lane] = sees ? at : -1;
      __syncthreads();
#pragma unroll
      for (int o = 0; o < kOwn; ++o) acc[o] *= old;
      for (int i = 0; i < kWave; ++i) {
        if (place[i] < 0) continue;
        const int64_t off_i = (base + i) & (page - 1);
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
          const int d = o * 64 + lane;
          const uint32_t byte =
              a.v.cache[place[i] * a.v.cache_stride + ((2 * kvh + 1) * page + off_i) * (DIM / 2) + d / 2];
          const float f =
              scale_operand(a.v.scales[place[i] * a.v.scales_stride +
                                       ((2 * kvh + 1) * (DIM / 32) + d / 32) * page + off_i]);
          const f32x2 x = decode2_f32<0>(byte, f);
          acc[o] += weight[i] * ((d & 1) ? x[1] : x[0]);
        }
      }
      __syncthreads();
    }
    base = base < first && base + kWave >= sinks ? first : base + kWave;
  }
  T *out = static_cast<T *>(a.out) + (t * a.heads + h) * DIM;
#pragma unroll
  for (int o = 0; o < kOwn; ++o) out[o * 64 + lane] = static_cast<T>(l == 0 ? 0 : acc[o] / l);
  if (a.lse && lane == 0) a.lse[t * a.heads + h] = l == 0 ? -__builtin_inff() : m + logf(l);
}

template <typename T>
void launch_attention(const AttnArgs &a, int dim, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.tokens), a.heads), block(64);
  if (dim == 64) hipLaunchKernelGGL((page_attention_rows_kernel<T, 64>), grid, block, 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL((page_attention_rows_kernel<T, 128>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((page_attention_rows_kernel<T, 256>), grid, block, 0, s, a);
}

}  // namespace shmt

using namespace shmt;

extern "C" {

int64_t shmt_page_attention_scratch_bytes(int64_t tokens, int heads, int kv_heads, int dim, int64_t requests,
                                          int64_t max_query_len) {
  (void)tokens, (void)heads, (void)kv_heads, (void)dim, (void)requests, (void)max_query_len;
  return 0;
}

int shmt_page_attention(const shmt_paged_cache *cache, const void *query, int64_t query_token_stride,
                        int64_t query_head_stride, int elem_type, int64_t tokens, int heads,
                        const int32_t *block_table, int64_t width, int64_t table_stride, const void *query_starts,
                        const void *kv_lens, int len_bytes, int64_t requests, float softmax_scale, int64_t window,
                        int64_t sinks, int64_t max_query_len, void *out, float *lse, void *scratch,
                        int64_t scratch_bytes, void *stream) {
  PagedView v;
  const int rc = paged_view(cache, &v);
  if (rc != SHMT_OK) return rc;
  SHMT_REQUIRE(elem_type == SHMT_F16 || elem_type == SHMT_BF16, "queries can only be float16 or bfloat16");
  SHMT_REQUIRE(tokens >= 0 && tokens < (int64_t{1} << 31), "the number of query rows must be in [0, 2^31)");
  SHMT_REQUIRE(heads >= 1 && heads <= 65535 && heads % cache->kv_heads == 0,
               "%d query heads do not share %d heads of the cache evenly", heads, cache->kv_heads);
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(width >= 0 && width < (int64_t{1} << 31) / cache->page, "the block table holds too many tokens");
  SHMT_REQUIRE(width_ok(len_bytes), "query_starts and kv_lens can only be int32 or int64");
  SHMT_REQUIRE(window >= 0 && sinks >= 0 && max_query_len >= 0, "window, sinks and max_query_len must be >= 0");
  SHMT_REQUIRE(softmax_scale == softmax_scale && softmax_scale - softmax_scale == 0, "softmax_scale must be finite");
  if (tokens == 0) return SHMT_OK;
  SHMT_REQUIRE(query && out, "query or out is null");
  SHMT_REQUIRE(requests == 0 || (query_starts && kv_lens), "query_starts or kv_lens is null");
  SHMT_REQUIRE(requests == 0 || width == 0 || (block_table && table_stride >= width), "block_table is null or narrow");
  SHMT_REQUIRE(((reinterpret_cast<int64_t>(query) | query_token_stride * 2 | query_head_stride * 2) & 15) == 0,
               "every row of query has to begin on 16 bytes");
  SHMT_REQUIRE((reinterpret_cast<int64_t>(out) & 15) == 0, "out has to begin on 16 bytes");
  (void)scratch, (void)scratch_bytes;
  const AttnArgs a{v, query, query_token_stride, query_head_stride, tokens, heads, heads / cache->kv_heads,
                   block_table, width, table_stride, query_starts, kv_lens, len_bytes, requests, softmax_scale,
                   window, sinks, out, lse};
  if (elem_type == SHMT_F16) launch_attention<_Float16>(a, cache->dim, as_stream(stream));
  else launch_attention<__bf16>(a, cache->dim, as_stream(stream));
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
