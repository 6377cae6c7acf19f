// Attention over the paged key/value cache held in 4 bits
// (shmt_page_attention).
#include "common.h"
#include "paged_dev.h"
#include "paged_host.h"
#include "wave.h"

#include <algorithm>
#include <type_traits>

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

// What a workgroup left for the join: the item it finished that other workgroups had begun.
struct JoinRecord {
  int32_t first;  // the workgroup that began the item; -1: nothing to join
  int32_t head;   // of the cache
  int32_t rows;
  int32_t row0;       // the item's first row, counted (token, head of the group) from the request's first query
  int64_t first_row;  // the request's first row of `query`
};

// ---- items and units -------------------------------------------------------------
// An item is kRows rows (queries of one request, all heads of one group: row r is token r / group, head r % group) against one head of
// the cache. Its tokens are cut at multiples of kUnit: the tiles that hold first tokens ("sinks") that are seen,
// then those from the window's begin to the last row's own place. Units are numbered request by request, head by
// head, row tile by row tile; workgroup w of G takes units floor(w U / G) up to floor((w + 1) U / G), so all end at
// the same time whatever the lengths are, and an item may be shared by several workgroups, each of which leaves a
// part (maximum, sum, weighted values) that page_attention_join_kernel puts together.
constexpr int kUnit = 128;      // tokens: four waves of 32
constexpr int kWaveTokens = 32;

struct Request {
  int64_t first_row;  // of `query`
  int32_t queries;
  int32_t before;     // tokens in front of the first query (may be negative: then the first rows see nothing)
  int32_t limit;      // tokens that the table has room for
};

struct Span {
  int32_t sink_tiles;  // tiles 0 .. sink_tiles
  int32_t tile0;       // then tiles from here
  int32_t units;
  int32_t sink_end;    // tokens below this are seen as sinks by every row that has them outside of its window
  int32_t begin, end;  // tokens [begin, end) and [0, sink_end) are all that any row of the item sees
};

__device__ __forceinline__ Request attn_request(const AttnArgs &a, int64_t b) {
  int64_t lo, hi;
  load_int_pair(a.starts, b, a.len_bytes, &lo, &hi);
  const int64_t len = load_int(a.kv_lens, b, a.len_bytes);
  lo = min(max(lo, int64_t{0}), a.tokens);
  hi = min(max(hi, lo), a.tokens);
  Request r;
  r.first_row = lo;
  r.queries = static_cast<int32_t>(hi - lo);
  r.before = static_cast<int32_t>(min(max(len, int64_t{0}), int64_t{0x7fffffff}) - (hi - lo));
  r.limit = a.v.pages > 0 ? static_cast<int32_t>(a.width << a.v.log2_page) : 0;
  return r;
}

template <int ROWS>
__device__ __forceinline__ Span attn_span(const AttnArgs &a, const Request &r, int64_t row0) {
  const int64_t all = static_cast<int64_t>(r.queries) * a.group;
  const int32_t t_first = static_cast<int32_t>(row0 / a.group);
  const int32_t t_last = static_cast<int32_t>((min(row0 + ROWS, all) - 1) / a.group);
  Span s;
  s.end = max(min(r.before + t_last + 1, r.limit), 0);
  s.begin = 0;
  if (a.window > 0) s.begin = static_cast<int32_t>(max(min(int64_t{r.before} + t_first + 1 - a.window, int64_t{s.end}), int64_t{0}));
  s.tile0 = s.begin / kUnit;
  s.sink_end = static_cast<int32_t>(min(a.sinks, int64_t{s.begin}));
  s.sink_tiles = min((s.sink_end + kUnit - 1) / kUnit, s.tile0);
  s.units = max(s.sink_tiles + (s.end + kUnit - 1) / kUnit - s.tile0, 1);
  return s;
}

// Units of request b for one head.
template <int ROWS>
__device__ __forceinline__ int64_t attn_units(const AttnArgs &a, const Request &r) {
  int64_t n = 0;
  const int64_t all = static_cast<int64_t>(r.queries) * a.group;
  for (int64_t row0 = 0; row0 < all; row0 += ROWS) n += attn_span<ROWS>(a, r, row0).units;
  return n;
}

// x of this lane and of the lane 32 (16) further on: the swap instructions exchange halves (odd and even quarters) of two
// registers.
struct Both {
  float a, b;
};
__device__ __forceinline__ Both swap32(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const uint32_t a = p[0], b = p[1];
  return {__uint_as_float(a), __uint_as_float(b)};
}
__device__ __forceinline__ Both swap16(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const uint32_t a = p[0], b = p[1];
  return {__uint_as_float(a), __uint_as_float(b)};
}
// The maximum / sum of a value over the four lanes that hold one column of a 16 x 16 product.
__device__ __forceinline__ float across_max(float x) {
  const Both p = swap32(x);
  const Both q = swap16(fmaxf(p.a, p.b));
  return fmaxf(q.a, q.b);
}
__device__ __forceinline__ float across_sum(float x) {
  const Both p = swap32(x);
  const Both q = swap16(p.a + p.b);
  return q.a + q.b;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  bf16x2 p;
  p[0] = static_cast<__bf16>(a);
  p[1] = static_cast<__bf16>(b);
  return __builtin_bit_cast(uint32_t, p);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 32 tokens of one head as a wave holds them: lane (m, g) = (lane % 16, lane / 16) has, of the key of token m of each
// 16, the quarter g; of the values of tokens 4g .. 4g + 3 of each 16, the sixteenth m.
template <int DIM>
struct KvTile {
  static constexpr int kKeyWords = DIM / 32;                       // of 8 codes
  static constexpr int kKeyScales = DIM / 128 > 0 ? DIM / 128 : 1;
  static constexpr int kValueWords = DIM / 128 > 0 ? DIM / 128 : 1;  // at 64 dimensions: half a word
  uint32_t key[2][kKeyWords];
  uint32_t key_scale[2][kKeyScales];
  uint32_t value[2][4][kValueWords];
  uint32_t value_scale[2];  // a byte for each of the four tokens
};

// Loads the 16 tokens at place `off` of page `at`.
template <int DIM>
__device__ __forceinline__ void load_half(const PagedView &v, int head, int64_t at, int off, int lane, int half,
                                          KvTile<DIM> &t) {
  const int m = lane & 15, g = lane >> 4;
  const int page = 1 << v.log2_page;
  const uint8_t *tile = v.cache + at * v.cache_stride + (static_cast<int64_t>(head) * 2 << v.log2_page) * (DIM / 2);
  const uint8_t *sc = v.scales + at * v.scales_stride + (static_cast<int64_t>(head) * 2 << v.log2_page) * (DIM / 32);
  const uint8_t *k = tile + (off + m) * (DIM / 2) + g * (DIM / 8);
  if constexpr (DIM == 64) {
    const uint2 x = *reinterpret_cast<const uint2 *>(k);
    t.key[half][0] = x.x, t.key[half][1] = x.y;
    t.key_scale[half][0] = sc[(g >> 1) * page + off + m];
  } else {
#pragma unroll
    for (int i = 0; i < DIM / 128; ++i) {
      const uint4 x = reinterpret_cast<const uint4 *>(k)[i];
      t.key[half][4 * i] = x.x, t.key[half][4 * i + 1] = x.y, t.key[half][4 * i + 2] = x.z, t.key[half][4 * i + 3] = x.w;
      t.key_scale[half][i] = sc[(g * (DIM / 128) + i) * page + off + m];
    }
  }
  const uint8_t *val = tile + (page + off + 4 * g) * (DIM / 2) + m * (DIM / 32);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint8_t *p = val + r * (DIM / 2);
    if constexpr (DIM == 64) t.value[half][r][0] = *reinterpret_cast<const uint16_t *>(p);
    else if constexpr (DIM == 128) t.value[half][r][0] = *reinterpret_cast<const uint32_t *>(p);
    else {
      const uint2 x = *reinterpret_cast<const uint2 *>(p);
      t.value[half][r][0] = x.x, t.value[half][r][1] = x.y;
    }
  }
  t.value_scale[half] =
      *reinterpret_cast<const uint32_t *>(sc + (DIM / 32 + m * (DIM / 16) / 32) * page + off + 4 * g);
}

// Softmax state and weighted values of NT x 16 rows: lane (n, g) has row n of each 16, and the dimensions
// (4 g + r) * DIM / 16 + i in acc[.][i][r].
template <int DIM, int NT>
struct RowState {
  float top[NT], sum[NT];  // of scores in powers of two; the sum over this lane's tokens only
  f32x4 acc[NT][DIM / 16];
};

constexpr float kNothing = -__builtin_inff();

// One wave's step over 32 tokens.
//   S^T = K Q^T, 16 tokens x 16 rows at a time: lane (n, g) gets the scores of row n with tokens 4g .. 4g + 3, which is
//   the place that the weights need to have as the right operand of O^T += V^T P^T (contraction over tokens, which may be
//   numbered in any order as long as both operands agree): nothing crosses lanes but the maximum.
// Keys and values become bfloat16 exactly. The weights of float16 queries are held as the sum of two bfloat16 (16 bits), as
// are the queries themselves; with bfloat16 queries the weights are rounded to bfloat16, an error of the size of the
// result's own rounding.
template <int DIM, int NT, int PARTS, bool MASKED>
__device__ __forceinline__ void attend_tile(const AttnArgs &a, const KvTile<DIM> &t, const u32x4 (&q)[PARTS][NT][DIM / 32],
                                            RowState<DIM, NT> &st, float scale2, int lane, int token0, const bool (&there)[2],
                                            const int (&pos)[NT], int limit) {
  const int g = lane >> 4;
  f32x4 s[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) {
      const float f = scale_operand(t.key_scale[half][i / 4]);
      const uint32_t c = t.key[half][i];
      const u32x4 k = {decode2_bf16<0>(c, f), decode2_bf16<1>(c, f), decode2_bf16<2>(c, f), decode2_bf16<3>(c, f)};
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) s[n][half] = mfma(k, q[p][n][i], s[n][half]);
    }
  }
  u32x4 w[PARTS][NT];
  float seen[NT][8];  // MASKED: the weights, -1 where the row does not see the token
  bool grows = false;
  float most[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float x = kNothing;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = s[n][half][r] * scale2;
        if constexpr (MASKED) {
          const int j = token0 + 16 * half + 4 * g + r;
          const bool sees = there[half] && j <= pos[n] && j < limit &&
                            (a.window == 0 || int64_t{j} > int64_t{pos[n]} - a.window || j < a.sinks);
          v = sees ? v : kNothing;
          seen[n][4 * half + r] = sees ? 0.0f : -1.0f;
        }
        s[n][half][r] = v;
        x = fmaxf(x, v);
      }
    most[n] = across_max(x);
    grows |= most[n] > st.top[n] + 8.0f;
  }
  // The running maximum moves only where a weight would pass 2^8 (the first one always does).
  if (__ballot(grows)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float next = fmaxf(st.top[n], most[n]);
      const float f = __builtin_amdgcn_exp2f(st.top[n] - fmaxf(next, -3.0e38f));
      st.top[n] = next;
      st.sum[n] *= f;
#pragma unroll
      for (int i = 0; i < DIM / 16; ++i) st.acc[n][i] *= f;
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float base = fmaxf(st.top[n], -3.0e38f);
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(s[n][j / 4][j % 4] - base);
      st.sum[n] += e[j];
      if constexpr (MASKED) seen[n][j] = seen[n][j] < 0 ? -1.0f : e[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t hi = pack_bf16(e[2 * j], e[2 * j + 1]);
      w[0][n][j] = hi;
      if constexpr (PARTS == 2)
        w[1][n][j] = pack_bf16(e[2 * j] - __builtin_bit_cast(float, hi << 16),
                               e[2 * j + 1] - __builtin_bit_cast(float, hi & 0xffff0000u));
    }
  }
  uint32_t vs[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) vs[j] = (t.value_scale[j / 4] >> (8 * (j % 4))) & 255u;
  if constexpr (MASKED) {
    // Values that are not finite in bfloat16 must not meet the weight 0 of a row that does not see them: they are taken
    // out of the product (their scale becomes the smallest) and added for the rows that do see them, one token at a time.
    bool wild = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) wild |= vs[j] >= 253u;
    if (__ballot(wild)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        for (int gt = 0; gt < 4; ++gt) {
          if (!(__ballot(vs[j] >= 253u) >> (16 * gt) & 0xffffull)) continue;
          float p[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) p[n] = __shfl(seen[n][j], (lane & 15) + 16 * gt);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int from = 4 * g + r + 16 * gt;
            const uint32_t byte = static_cast<uint32_t>(__shfl(static_cast<int>(vs[j]), from));
#pragma unroll
            for (int word = 0; word < KvTile<DIM>::kValueWords; ++word) {
              const uint32_t c = static_cast<uint32_t>(__shfl(static_cast<int>(t.value[j / 4][j % 4][word]), from));
              const float f = scale_operand(byte);
              const f32x2 x[4] = {decode2_f32<0>(c, f), decode2_f32<1>(c, f), decode2_f32<2>(c, f), decode2_f32<3>(c, f)};
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < (DIM == 64 ? 4 : 8); ++i)
                  if (byte >= 253u && p[n] >= 0) st.acc[n][8 * word + i][r] += p[n] * x[i / 2][i % 2];
            }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) vs[j] = vs[j] >= 253u ? 0u : vs[j];
    }
  }
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = scale_operand(vs[j]);
#pragma unroll
  for (int word = 0; word < KvTile<DIM>::kValueWords; ++word) {
    auto two = [&](auto byte) {  // dimensions 2 B and 2 B + 1 of this lane's
      constexpr int B = decltype(byte)::value;
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = decode2_bf16<B>(t.value[j / 4][j % 4][word], f[j]);
      u32x4 lo, hi;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        lo[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
        hi[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          st.acc[n][8 * word + 2 * B] = mfma(lo, w[p][n], st.acc[n][8 * word + 2 * B]);
          st.acc[n][8 * word + 2 * B + 1] = mfma(hi, w[p][n], st.acc[n][8 * word + 2 * B + 1]);
        }
    };
    two(std::integral_constant<int, 0>{});
    two(std::integral_constant<int, 1>{});
    if constexpr (DIM > 64) {
      two(std::integral_constant<int, 2>{});
      two(std::integral_constant<int, 3>{});
    }
  }
}

// What the waves of a workgroup exchange at the end of an item.
template <int DIM>
struct JoinShared {
  static constexpr int kStride = DIM + 4;  // rows shifted against each other over the banks
  alignas(16) float acc[4][16 * kStride];
  float top[4][16], sum[4][16];
};

template <typename T, int DIM, int NT>
__global__ __launch_bounds__(256, NT * DIM <= 128 ? 4 : NT * DIM <= 256 ? 2 : 1) void page_attention_kernel(
    AttnArgs a, float *parts, float *part_stats, JoinRecord *records) {
  constexpr int kRows = 16 * NT;
  constexpr int kParts = sizeof(T) == 2 && std::is_same<T, _Float16>::value ? 2 : 1;
  __shared__ JoinShared<DIM> shared;
  __shared__ int64_t scan[4];
  __shared__ int64_t found[2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n_lane = lane & 15, g = lane >> 4;
  const int kv_heads = a.v.kv_heads;

  // rows of no request
  {
    int64_t row_lo = a.tokens, row_hi = a.tokens;
    if (a.requests > 0) {
      row_lo = min(max(load_int(a.starts, 0, a.len_bytes), int64_t{0}), a.tokens);
      row_hi = min(max(load_int(a.starts, a.requests, a.len_bytes), row_lo), a.tokens);
    }
    const int64_t row16 = static_cast<int64_t>(a.heads) * DIM / 8;  // pieces of 16 bytes
    const int64_t none = row_lo + a.tokens - row_hi;
    for (int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x; i < none * row16; i += int64_t{gridDim.x} * 256) {
      const int64_t row = i / row16;
      reinterpret_cast<uint4 *>(a.out)[(row < row_lo ? row : row - row_lo + row_hi) * row16 + i % row16] = uint4{0, 0, 0, 0};
    }
    if (a.lse)
      for (int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x; i < none * a.heads; i += int64_t{gridDim.x} * 256) {
        const int64_t row = i / a.heads;
        a.lse[(row < row_lo ? row : row - row_lo + row_hi) * a.heads + i % a.heads] = kNothing;
      }
  }

  // This workgroup's units: each thread counts a run of requests.
  const int64_t each = (a.requests + 255) / 256;
  const int64_t b_lo = min(threadIdx.x * each, a.requests), b_hi = min(b_lo + each, a.requests);
  int64_t mine = 0;
  for (int64_t b = b_lo; b < b_hi; ++b) mine += attn_units<kRows>(a, attn_request(a, b)) * kv_heads;
  uint64_t total;
  const int64_t at = static_cast<int64_t>(
      block_exclusive_scan<uint64_t, 256>(static_cast<uint64_t>(mine), reinterpret_cast<uint64_t *>(scan), &total));
  const int64_t U = static_cast<int64_t>(total);
  // With a unit for everyone, neighbours in the numbering of units are on one XCD: they read the same pages. With fewer
  // units than workgroups each has one, on all XCDs.
  const int64_t G = min(int64_t{gridDim.x}, U);
  const int64_t wg = G == gridDim.x && G % 8 == 0 ? (blockIdx.x & 7) * (G / 8) + (blockIdx.x >> 3) : blockIdx.x;
  if (threadIdx.x == 0) records[wg].first = -1;
  if (wg >= G) return;
  const int64_t u_begin = wg * U / G, u_end = (wg + 1) * U / G;
  if (at <= u_begin && u_begin < at + mine) {
    int64_t b = b_lo, before = at;
    for (;; ++b) {
      const int64_t n = attn_units<kRows>(a, attn_request(a, b)) * kv_heads;
      if (u_begin < before + n) break;
      before += n;
    }
    found[0] = b, found[1] = before;
  }
  __syncthreads();
  int64_t b = found[0], u_request = found[1];  // units in front of request b
  Request req = attn_request(a, b);
  int64_t per_head = attn_units<kRows>(a, req);
  int head = static_cast<int>((u_begin - u_request) / per_head);
  int64_t u_item = u_request + head * per_head, row0 = 0;
  Span span = attn_span<kRows>(a, req, 0);
  while (u_item + span.units <= u_begin) {
    u_item += span.units;
    row0 += kRows;
    span = attn_span<kRows>(a, req, row0);
  }

  const float scale2 = a.scale * 1.44269504088896340736f;  // scores in powers of two
  for (int64_t u = u_begin; u < u_end;) {
    const int64_t stop = min(u_item + span.units, u_end);
    const int rows = static_cast<int>(min(int64_t{kRows}, static_cast<int64_t>(req.queries) * a.group - row0));
    // queries: row n of each 16, quarter g of the dimensions, as the right operand
    u32x4 q[kParts][NT][DIM / 32];
    int pos[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 16 * n + n_lane;
      const int64_t row = row0 + min(r, rows - 1);
      const int64_t token = row / a.group;
      const int64_t h = head * a.group + row % a.group;
      pos[n] = r < rows ? req.before + static_cast<int>(token) : -1;
      const T *src = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head + g * (DIM / 4);
#pragma unroll
      for (int i = 0; i < DIM / 32; ++i) {
        const u32x4 x = reinterpret_cast<const u32x4 *>(src)[i];
        if constexpr (kParts == 1) {
          q[0][n][i] = x;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 y = __builtin_bit_cast(f16x2, static_cast<uint32_t>(x[j]));
            const float y0 = static_cast<float>(y[0]), y1 = static_cast<float>(y[1]);
            const uint32_t hi = pack_bf16(y0, y1);
            q[0][n][i][j] = hi;
            q[kParts - 1][n][i][j] = pack_bf16(y0 - __builtin_bit_cast(float, hi << 16),
                                               y1 - __builtin_bit_cast(float, hi & 0xffff0000u));
          }
        }
      }
    }
    RowState<DIM, NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      st.top[n] = kNothing;
      st.sum[n] = 0;
#pragma unroll
      for (int i = 0; i < DIM / 16; ++i) st.acc[n][i] = f32x4{0, 0, 0, 0};
    }
    const int pos_first = req.before + static_cast<int>(row0 / a.group);
    const int pos_last = req.before + static_cast<int>((row0 + rows - 1) / a.group);
    const int32_t *table = a.table + b * a.table_stride;
    for (; u < stop; ++u) {
      const int k = static_cast<int>(u - u_item);
      const int tile = k < span.sink_tiles ? k : span.tile0 + k - span.sink_tiles;
      const int token0 = __builtin_amdgcn_readfirstlane(tile * kUnit + wave * kWaveTokens);
      bool there[2];
      int64_t page_at[2];
      int off[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j = token0 + 16 * half;
        there[half] = j < span.end && (j + 15 >= span.begin || j < span.sink_end);
        const int p = there[half] ? table[j >> a.v.log2_page] : 0;
        there[half] = there[half] && p >= 0 && p < a.v.pages;
        page_at[half] = there[half] ? p : 0;
        off[half] = j & ((1 << a.v.log2_page) - 1);
      }
      if (!there[0] && !there[1]) continue;
      KvTile<DIM> t;
      load_half<DIM>(a.v, head, page_at[0], off[0], lane, 0, t);
      load_half<DIM>(a.v, head, page_at[1], off[1], lane, 1, t);
      const bool whole = there[0] && there[1] && token0 + kWaveTokens - 1 <= pos_first && token0 + kWaveTokens <= span.end &&
                         (a.window == 0 || int64_t{token0} > int64_t{pos_last} - a.window || token0 + kWaveTokens <= a.sinks);
      if (whole) attend_tile<DIM, NT, kParts, false>(a, t, q, st, scale2, lane, token0, there, pos, span.end);
      else attend_tile<DIM, NT, kParts, true>(a, t, q, st, scale2, lane, token0, there, pos, span.end);
    }

    // The four waves' states, 16 rows at a time, into the result or into a part.
    const bool begins = u_item >= u_begin, ends = stop == u_item + span.units;
    const int64_t slot = 2 * wg + (begins ? 1 : 0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (16 * n < rows) {
        const float sum = across_sum(st.sum[n]);
        if (g == 0) {
          shared.top[wave][n_lane] = st.top[n];
          shared.sum[wave][n_lane] = sum;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < DIM / 16; i += 4)
            *reinterpret_cast<f32x4 *>(&shared.acc[wave][n_lane * JoinShared<DIM>::kStride + (4 * g + r) * (DIM / 16) + i]) =
                f32x4{st.acc[n][i][r], st.acc[n][i + 1][r], st.acc[n][i + 2][r], st.acc[n][i + 3][r]};
        __syncthreads();
        const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (DIM / 16);
        if (16 * n + r < rows) {
          float top = kNothing;
#pragma unroll
          for (int v = 0; v < 4; ++v) top = fmaxf(top, shared.top[v][r]);
          const float base = fmaxf(top, -3.0e38f);
          float f[4], total_sum = 0;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            f[v] = __builtin_amdgcn_exp2f(shared.top[v][r] - base);
            total_sum += f[v] * shared.sum[v][r];
          }
          float o[DIM / 16];
#pragma unroll
          for (int i = 0; i < DIM / 16; ++i) {
            o[i] = 0;
#pragma unroll
            for (int v = 0; v < 4; ++v) o[i] += f[v] * shared.acc[v][r * JoinShared<DIM>::kStride + d0 + i];
          }
          if (begins && ends) {
            const int64_t row = row0 + 16 * n + r;
            const int64_t line = (req.first_row + row / a.group) * a.heads + head * a.group + row % a.group;
            const float inv = total_sum == 0 ? 0 : 1 / total_sum;
            T *out = static_cast<T *>(a.out) + line * DIM + d0;
            typedef T out_vec __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int i = 0; i < DIM / 16; i += 4)
              *reinterpret_cast<out_vec *>(out + i) =
                  out_vec{static_cast<T>(o[i] * inv), static_cast<T>(o[i + 1] * inv), static_cast<T>(o[i + 2] * inv),
                          static_cast<T>(o[i + 3] * inv)};
            if (a.lse && (threadIdx.x & 15) == 0)
              a.lse[line] = total_sum == 0 ? kNothing : (top + __builtin_log2f(total_sum)) * 0.69314718055994530942f;
          } else {
            float *out = parts + (slot * kRows + 16 * n + r) * DIM + d0;
#pragma unroll
            for (int i = 0; i < DIM / 16; i += 4) *reinterpret_cast<f32x4 *>(out + i) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
            if ((threadIdx.x & 15) == 0) {
              part_stats[(slot * kRows + 16 * n + r) * 2] = top;
              part_stats[(slot * kRows + 16 * n + r) * 2 + 1] = total_sum;
            }
          }
        }
        __syncthreads();
      }
    }
    if (!begins && ends && threadIdx.x == 0) {
      // the last workgroup whose units begin at the item's first unit or before it
      records[wg] = JoinRecord{static_cast<int32_t>(((u_item + 1) * G - 1) / U), head, rows, static_cast<int32_t>(row0),
                               req.first_row};
    }
    if (u >= u_end) break;
    // the next item
    u_item += span.units;
    row0 += kRows;
    if (row0 >= static_cast<int64_t>(req.queries) * a.group) {
      row0 = 0;
      if (++head == kv_heads) {
        head = 0;
        do {
          req = attn_request(a, ++b);
        } while (req.queries == 0);
      }
    }
    span = attn_span<kRows>(a, req, row0);
  }
}

// Puts the parts of an item together; a workgroup for each 4 rows of each record.
template <typename T, int DIM, int ROWS>
__global__ __launch_bounds__(256) void page_attention_join_kernel(AttnArgs a, const float *parts, const float *part_stats,
                                                                  const JoinRecord *records) {
  const int64_t wg = blockIdx.x;
  const JoinRecord rec = records[wg];
  const int r = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (rec.first < 0 || r >= rec.rows) return;
  const int lane = threadIdx.x & 63;
  constexpr int kOwn = DIM / 64;
  float top = kNothing, sum = 0, acc[kOwn] = {};
  for (int64_t w = rec.first; w <= wg; ++w) {
    const int64_t line = (2 * w + (w == rec.first ? 1 : 0)) * ROWS + r;
    const float m = part_stats[line * 2], l = part_stats[line * 2 + 1];
    const float next = fmaxf(top, m), base = fmaxf(next, -3.0e38f);
    const float f = __builtin_amdgcn_exp2f(top - base), e = __builtin_amdgcn_exp2f(m - base);
    sum = sum * f + l * e;
#pragma unroll
    for (int o = 0; o < kOwn; ++o) acc[o] = acc[o] * f + parts[line * DIM + lane * kOwn + o] * e;
    top = next;
  }
  const int64_t row = rec.row0 + r;
  const int64_t line = (rec.first_row + row / a.group) * a.heads + rec.head * a.group + row % a.group;
  T *out = static_cast<T *>(a.out) + line * DIM + lane * kOwn;
#pragma unroll
  for (int o = 0; o < kOwn; ++o) out[o] = static_cast<T>(sum == 0 ? 0 : acc[o] / sum);
  if (a.lse && lane == 0) a.lse[line] = sum == 0 ? kNothing : (top + __builtin_log2f(sum)) * 0.69314718055994530942f;
}

// ---- launch ------------------------------------------------------------------------

struct AttnShape {
  int tiles;       // of 16 rows an item
  int64_t groups;  // workgroups
  int64_t parts_bytes, stats_bytes, record_bytes;
  int64_t bytes() const { return parts_bytes + stats_bytes + record_bytes; }
};

// How many rows an item has, and how many workgroups share the units: what the card holds at once, or the most units that
// there can be.
inline AttnShape attn_shape(int64_t tokens, int heads, int kv_heads, int dim, int elem_type, int64_t requests,
                            int64_t max_query_len) {
  const int64_t longest = max_query_len > 0 ? std::min(max_query_len, tokens) : std::max<int64_t>(tokens - requests + 1, 1);
  const int64_t rows = longest * (heads / kv_heads);
  const int most = (elem_type == SHMT_F16 ? 2 : 4) / (dim == 256 ? 2 : 1);
  AttnShape s;
  s.tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  s.tiles = std::min(s.tiles, most);
  s.groups = s.tiles * dim <= 128 ? 1024 : s.tiles * dim <= 256 ? 512 : 256;
  const int64_t lines = 2 * s.groups * 16 * s.tiles;
  s.parts_bytes = lines * dim * 4;
  s.stats_bytes = lines * 8;
  s.record_bytes = s.groups * static_cast<int64_t>(sizeof(JoinRecord));
  return s;
}

template <typename T, int DIM, int NT>
void launch_tiles(const AttnArgs &a, const AttnShape &s, void *scratch, hipStream_t stream) {
  float *parts = static_cast<float *>(scratch);
  float *stats = reinterpret_cast<float *>(static_cast<char *>(scratch) + s.parts_bytes);
  JoinRecord *records = reinterpret_cast<JoinRecord *>(static_cast<char *>(scratch) + s.parts_bytes + s.stats_bytes);
  const unsigned groups = static_cast<unsigned>(s.groups);
  hipLaunchKernelGGL((page_attention_kernel<T, DIM, NT>), dim3(groups), dim3(256), 0, stream, a, parts, stats, records);
  hipLaunchKernelGGL((page_attention_join_kernel<T, DIM, 16 * NT>), dim3(groups, 4 * NT), dim3(256), 0, stream, a, parts,
                     stats, records);
}

template <typename T, int DIM>
void launch_dim(const AttnArgs &a, const AttnShape &s, void *scratch, hipStream_t stream) {
  constexpr int kMost = (std::is_same<T, _Float16>::value ? 2 : 4) / (DIM == 256 ? 2 : 1);
  if (s.tiles == 1) return launch_tiles<T, DIM, 1>(a, s, scratch, stream);
  if constexpr (kMost >= 2)
    if (s.tiles == 2) return launch_tiles<T, DIM, 2>(a, s, scratch, stream);
  if constexpr (kMost >= 4) launch_tiles<T, DIM, 4>(a, s, scratch, stream);
}

template <typename T>
void launch_attention(const AttnArgs &a, int dim, const AttnShape &s, void *scratch, hipStream_t stream) {
  if (dim == 64) launch_dim<T, 64>(a, s, scratch, stream);
  else if (dim == 128) launch_dim<T, 128>(a, s, scratch, stream);
  else launch_dim<T, 256>(a, s, scratch, stream);
}

}  // namespace shmt

using namespace shmt;

extern "C" {

int64_t shmt_page_attention_scratch_bytes(int64_t tokens, int heads, int kv_heads, int dim, int elem_type,
                                          int64_t requests, int64_t max_query_len) {
  if (tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || (dim != 64 && dim != 128 && dim != 256) ||
      (elem_type != SHMT_F16 && elem_type != SHMT_BF16) || requests < 0 || max_query_len < 0) {
    set_error("bad arguments for the attention's scratch size");
    return -1;
  }
  return attn_shape(tokens, heads, kv_heads, dim, elem_type, requests, max_query_len).bytes();
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
  const AttnShape shape = attn_shape(tokens, heads, cache->kv_heads, cache->dim, elem_type, requests, max_query_len);
  if (scratch_bytes < shape.bytes() || !scratch) {
    set_error("scratch too small: %lld bytes, needed %lld", static_cast<long long>(scratch_bytes),
              static_cast<long long>(shape.bytes()));
    return SHMT_ENOMEM;
  }
  SHMT_REQUIRE((reinterpret_cast<int64_t>(scratch) & 15) == 0, "scratch has to begin on 16 bytes");
  const AttnArgs a{v, query, query_token_stride, query_head_stride, tokens, heads, heads / cache->kv_heads,
                   block_table, width, table_stride, query_starts, kv_lens, len_bytes, requests, softmax_scale,
                   window, sinks, out, lse};
  if (elem_type == SHMT_F16) launch_attention<_Float16>(a, cache->dim, shape, scratch, as_stream(stream));
  else launch_attention<__bf16>(a, cache->dim, shape, scratch, as_stream(stream));
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
