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
  int64_t table_stride;
  const void *starts, *kv_lens;
  int len_bytes;
  int64_t requests;
  float scale;
  int32_t window, sinks;
  int32_t limit;  // tokens that a row of the table has room for
  void *out;
  float *lse;
};

// ---- items and units -------------------------------------------------------------
// An item is up to kRows rows against one head of the cache: a row is a query token and a head of the group that shares the
// cache's head, row r of a request being token r / group, head r % group. The tokens that an item's rows see are cut at
// multiples of kUnit: the tiles that hold first tokens ("sinks"), then those from the window's begin to the last row's own
// place. Units are numbered head by head, request by request, row tile by row tile; workgroup w of G takes units
// floor(w U / G) up to floor((w + 1) U / G), so all end at about the same time whatever the lengths are. An item may be
// shared by several workgroups; each leaves a part (maximum, sum, weighted values), which page_attention_join_kernel puts
// together.
constexpr int kUnit = 128;  // tokens: four waves of 32
constexpr int kWaveTokens = 32;
constexpr float kNothing = -__builtin_inff();
constexpr float kLowest = -3.0e38f;  // subtracted instead of kNothing, so that nothing stays nothing

struct AttnItem {
  int64_t unit;  // units of one head in front of it
  int32_t request, row0;
};

// What a workgroup left for the join: the item that it finished and others had begun.
struct JoinRecord {
  int32_t first;  // the workgroup that began the item; -1: nothing to join
  int32_t head;   // of the cache
  int32_t rows;
  int32_t row0;
  int64_t first_row;  // the request's first row of `query`
};

struct Request {
  int64_t first_row;  // of `query`
  int32_t queries;
  int32_t before;  // tokens in front of the first query; negative: the first rows see nothing
};

struct Span {
  int32_t sink_tiles;  // tiles 0 .. sink_tiles
  int32_t tile0;       // then tiles from here
  int32_t units;
  int32_t sink_end;    // tokens [0, sink_end) and [begin, end) are all that any row of the item sees
  int32_t begin, end;
};

// A value that is the same for the whole wave, as the compiler cannot tell of what came from memory: held once, not per lane.
__device__ __forceinline__ int same(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t same(int64_t v) {
  const uint32_t lo = same(static_cast<int>(v)), hi = same(static_cast<int>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ Request same(Request r) { return {same(r.first_row), same(r.queries), same(r.before)}; }
__device__ __forceinline__ Span same(Span s) {
  return {same(s.sink_tiles), same(s.tile0), same(s.units), same(s.sink_end), same(s.begin), same(s.end)};
}

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
  return r;
}

template <int ROWS>
__device__ __forceinline__ Span attn_span(const AttnArgs &a, const Request &r, int row0) {
  const int all = r.queries * a.group;
  const int t_first = static_cast<int>(static_cast<uint32_t>(row0) / static_cast<uint32_t>(a.group));
  const int t_last =
      static_cast<int>(static_cast<uint32_t>(min(row0 + ROWS, all) - 1) / static_cast<uint32_t>(a.group));
  Span s;
  s.end = max(min(r.before + t_last + 1, a.limit), 0);
  s.begin = a.window > 0 ? max(min(max(r.before + t_first, -1) - a.window + 1, s.end), 0) : 0;
  s.tile0 = s.begin / kUnit;
  s.sink_end = min(a.sinks, s.begin);
  s.sink_tiles = min((s.sink_end + kUnit - 1) / kUnit, s.tile0);
  s.units = max(s.sink_tiles + (s.end + kUnit - 1) / kUnit - s.tile0, 1);
  return s;
}

// Units of a request for one head.
template <int ROWS>
__device__ __forceinline__ int64_t attn_units(const AttnArgs &a, const Request &r) {
  int64_t n = 0;
  const int all = r.queries * a.group;
  for (int row0 = 0; row0 < all; row0 += ROWS) n += attn_span<ROWS>(a, r, row0).units;
  return n;
}

// Items of all requests with the units in front of each, for calls in which a request has many row tiles: one workgroup.
// items[0 .. n) and, behind the last, the number of units; *count = n. (Only starts that descend could make more items than
// there is room for.)
template <int ROWS>
__global__ __launch_bounds__(1024) void page_attention_items_kernel(AttnArgs a, int32_t *first_item, AttnItem *items,
                                                                    int64_t room, int32_t *count) {
  __shared__ uint64_t lds[16];
  int64_t n = 0;
  for (int64_t base = 0; base < a.requests; base += 1024) {
    const int64_t b = base + threadIdx.x;
    int64_t mine = 0;
    if (b < a.requests) mine = (attn_request(a, b).queries * a.group + ROWS - 1) / ROWS;
    uint64_t sum;
    const int64_t at = block_exclusive_scan<uint64_t, 1024>(mine, lds, &sum);
    if (b < a.requests) first_item[b] = static_cast<int32_t>(n + at);
    n += sum;
  }
  n = min(n, room);
  __syncthreads();
  int64_t units = 0;
  for (int64_t base = 0; base < n; base += 1024) {
    const int64_t i = base + threadIdx.x;
    int64_t mine = 0, lo = 0;
    int row0 = 0;
    if (i < n) {
      int64_t hi = a.requests - 1;  // the last request whose first item is i or before it
      while (lo < hi) {
        const int64_t mid = (lo + hi + 1) >> 1;
        if (first_item[mid] <= i) lo = mid; else hi = mid - 1;
      }
      row0 = static_cast<int>(i - first_item[lo]) * ROWS;
      mine = attn_span<ROWS>(a, attn_request(a, lo), row0).units;
    }
    uint64_t sum;
    const int64_t at = block_exclusive_scan<uint64_t, 1024>(mine, lds, &sum);
    if (i < n) items[i] = AttnItem{units + at, static_cast<int32_t>(lo), row0};
    units += sum;
  }
  if (threadIdx.x == 0) {
    items[n] = AttnItem{units, 0, 0};
    *count = static_cast<int32_t>(n);
  }
}

// ---- arithmetic of a tile ------------------------------------------------------------

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

// Where a lane's pieces lie behind the first of 16 tokens of a page; the rest of an address is the same for the wave.
struct LaneOffsets {
  uint32_t key, key_scale, value, value_scale;
};
template <int DIM>
__device__ __forceinline__ LaneOffsets lane_offsets(int lane, int page) {
  const int m = lane & 15, g = lane >> 4;
  LaneOffsets o;
  o.key = m * (DIM / 2) + g * (DIM / 8);
  o.key_scale = (DIM == 64 ? g >> 1 : g * (DIM / 128)) * page + m;
  o.value = (page + 4 * g) * (DIM / 2) + m * (DIM / 32);
  o.value_scale = (DIM / 32 + m * (DIM / 16) / 32) * page + 4 * g;
  return o;
}

// Loads the 16 tokens at place `off` of page `at` (both the same for the wave).
template <int DIM>
__device__ __forceinline__ void load_half(const PagedView &v, int head, int at, int off, const LaneOffsets &o, int half,
                                          KvTile<DIM> &t) {
  const int64_t tile = int64_t{2} * head << v.log2_page;
  const uint8_t *rows = v.cache + at * v.cache_stride + (tile + off) * (DIM / 2);
  const uint8_t *sc = v.scales + at * v.scales_stride + tile * (DIM / 32) + off;
  if constexpr (DIM == 64) {
    const uint2 x = *reinterpret_cast<const uint2 *>(rows + o.key);
    t.key[half][0] = x.x, t.key[half][1] = x.y;
    t.key_scale[half][0] = sc[o.key_scale];
  } else {
#pragma unroll
    for (int i = 0; i < DIM / 128; ++i) {
      const uint4 x = reinterpret_cast<const uint4 *>(rows + o.key)[i];
      t.key[half][4 * i] = x.x, t.key[half][4 * i + 1] = x.y, t.key[half][4 * i + 2] = x.z, t.key[half][4 * i + 3] = x.w;
      t.key_scale[half][i] = sc[o.key_scale + (i << v.log2_page)];
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint8_t *p = rows + o.value + r * (DIM / 2);
    if constexpr (DIM == 64) t.value[half][r][0] = *reinterpret_cast<const uint16_t *>(p);
    else if constexpr (DIM == 128) t.value[half][r][0] = *reinterpret_cast<const uint32_t *>(p);
    else {
      const uint2 x = *reinterpret_cast<const uint2 *>(p);
      t.value[half][r][0] = x.x, t.value[half][r][1] = x.y;
    }
  }
  t.value_scale[half] = *reinterpret_cast<const uint32_t *>(sc + o.value_scale);
}

// Softmax state and weighted values of NT x 16 rows: lane (n, g) has row n of each 16, and the dimensions
// (4 g + r) * DIM / 16 + i in acc[.][i][r].
template <int DIM, int NT>
struct RowState {
  float top[NT], sum[NT];  // the reference of the weights, in powers of two; their sum over this lane's tokens only
  f32x4 acc[NT][DIM / 16];
};

// Queries of an item, as the right operand of K Q^T: fragment i of 16 rows holds, for lane (n, g), eight dimensions of
// row n from g * DIM / 4 + 8 i on. They stay in registers where they are few, else in LDS, where the four waves share them.
template <int DIM, int NT, int PARTS>
struct Queries {
  static constexpr int kFrags = PARTS * NT * (DIM / 32);
  static constexpr bool kShared = kFrags > 8;
  u32x4 own[kShared ? 1 : kFrags];
  const u32x4 *shared;
  __device__ __forceinline__ u32x4 at(int part, int n, int i, int lane) const {
    const int f = (part * NT + n) * (DIM / 32) + i;
    if constexpr (kShared) return shared[f * kWave + lane];
    else return own[f];
  }
};

// Which tokens of a tile the rows of a lane see.
template <int NT>
struct Sight {
  int last[NT];   // tokens up to here ...
  int after[NT];  // ... from behind here, or
  int sinks;      // before here
  int begin, end, sink_end;  // no row of the item sees any outside of [begin, end) and [0, sink_end)
};

// Scale bytes from here on make values that are infinite in bfloat16, or not a number.
constexpr uint32_t kWild = 253;

// One wave's step over 32 tokens.
//   S^T = K Q^T, 16 tokens x 16 rows at a time: lane (n, g) gets the scores of row n with tokens 4g .. 4g + 3, which is
//   the place that the weights need to have as the right operand of O^T += V^T P^T (contraction over tokens, which may be
//   numbered in any order as long as both operands agree): nothing crosses lanes but the maximum.
// Keys and values become bfloat16 exactly. The weights of float16 queries are held as the sum of two bfloat16 (16 bits), as
// are the queries themselves; with bfloat16 queries the weights are rounded to bfloat16, an error of the size of the
// result's own rounding.
// `whole`: all rows see all tokens. Otherwise scores are masked; and values that are not finite in bfloat16 must not meet the
// weight 0 of a row that does not see them: they are left out (`wild` says so) and added at the end of the item.
// Returns whether the item has to be begun again (see below).
template <int DIM, int NT, int PARTS>
__device__ __forceinline__ bool attend_tile(KvTile<DIM> &t, const Queries<DIM, NT, PARTS> &q, RowState<DIM, NT> &st,
                                            float scale2, int lane, bool whole, int token0, bool there0, bool there1,
                                            const Sight<NT> &sight, bool &wild) {
  const int g = lane >> 4;
  f32x4 s[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < DIM / 32; ++i) {
    u32x4 k[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float f = scale_operand(t.key_scale[half][i / 4]);
      const uint32_t c = t.key[half][i];
      k[half] = u32x4{decode2_bf16<0>(c, f), decode2_bf16<1>(c, f), decode2_bf16<2>(c, f), decode2_bf16<3>(c, f)};
    }
    if constexpr (NT * DIM >= 512) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const u32x4 x = q.at(p, n, i, lane);
        s[n][0] = mfma(k[0], x, s[n][0]);
        s[n][1] = mfma(k[1], x, s[n][1]);
      }
  }
  if constexpr (NT * DIM >= 512) __builtin_amdgcn_sched_barrier(0);
  if (!whole) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int token = token0 + 16 * (j / 4) + 4 * g + j % 4;
        const bool sees = (j < 4 ? there0 : there1) && token <= sight.last[n] &&
                          (token > sight.after[n] || token < sight.sinks);
        s[n][j / 4][j % 4] = sees ? s[n][j / 4][j % 4] : kNothing;
      }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((t.value_scale[j / 4] >> (8 * (j % 4)) & 255u) >= kWild) {
        const int token = token0 + 16 * (j / 4) + 4 * g + j % 4;
        t.value_scale[j / 4] &= ~(255u << (8 * (j % 4)));
        wild |= (j < 4 ? there0 : there1) && token < sight.end && (token >= sight.begin || token < sight.sink_end);
      }
  }
  // Weights are taken relative to the maximum of the first tile in which a row saw anything. With floats' exponents any
  // reference near the true maximum does as well, so nothing is rescaled; where a score passes it by 2^40, which ordinary
  // scores do not, the wave begins its tokens again with the greater one.
  bool passed = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float x = s[n][0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) x = fmaxf(x, s[n][j / 4][j % 4]);
    const float most = across_max(x) * scale2;
    st.top[n] = st.top[n] == kNothing ? most : st.top[n];
    if (most > st.top[n] + 40.0f) passed = true, st.top[n] = most;
  }
  u32x4 w[PARTS][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float base = fmaxf(st.top[n], kLowest);
    float e[8], sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j / 4][j % 4], scale2, -base));
      sum += e[j];
    }
    st.sum[n] += sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t hi = pack_bf16(e[2 * j], e[2 * j + 1]);
      w[0][n][j] = hi;
      if constexpr (PARTS == 2)
        w[1][n][j] = pack_bf16(e[2 * j] - __uint_as_float(hi << 16), e[2 * j + 1] - __uint_as_float(hi & 0xffff0000u));
    }
  }
  // The conversion reads nothing of a scale but its exponent field, so the byte need not be cut out.
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    f[j] = __uint_as_float(j % 4 == 3 ? t.value_scale[j / 4] >> 1 : t.value_scale[j / 4] << (23 - 8 * (j % 4)));
#pragma unroll
  for (int word = 0; word < KvTile<DIM>::kValueWords; ++word) {
    auto two = [&](auto byte) {  // dimensions 2 B and 2 B + 1 of this lane's
      if constexpr (NT * DIM >= 512) __builtin_amdgcn_sched_barrier(0);
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
  return __ballot(passed) != 0;
}

// q . K[j] of one row and token, element by element.
template <typename T, int DIM>
__device__ float score_of(const T *q, const uint8_t *codes, const uint8_t *scales, int page) {
  float s = 0;
#pragma unroll 1
  for (int p = 0; p < DIM / 8; ++p) {
    const uint32_t c = reinterpret_cast<const uint32_t *>(codes)[p];
    const float f = scale_operand(scales[p / 4 * page]);
    const f32x2 x[4] = {decode2_f32<0>(c, f), decode2_f32<1>(c, f), decode2_f32<2>(c, f), decode2_f32<3>(c, f)};
#pragma unroll
    for (int i = 0; i < 8; ++i) s += static_cast<float>(q[8 * p + i]) * x[i / 2][i % 2];
  }
  return s;
}

// ---- the kernel ------------------------------------------------------------------------

// What the waves of a workgroup exchange at the end of an item.
template <int DIM>
struct JoinShared {
  static constexpr int kStride = DIM + 4;  // rows shifted against each other over the banks
  alignas(16) float acc[4][16 * kStride];
  float top[4][16], sum[4][16];
};

// Waves per SIMD that the registers are meant for.
constexpr int attn_waves(int dim, int tiles) { return tiles * dim <= 64 ? 4 : tiles * dim <= 128 ? 3 : 2; }

template <typename T, int DIM, int NT>
__global__ __launch_bounds__(256, attn_waves(DIM, NT)) void page_attention_kernel(
    AttnArgs a, const AttnItem *items, const int32_t *item_count, float *parts, float *part_stats, JoinRecord *records) {
  constexpr int kRows = 16 * NT;
  constexpr int kParts = std::is_same<T, _Float16>::value ? 2 : 1;
  using Q = Queries<DIM, NT, kParts>;
  union Shared {
    JoinShared<DIM> join;
    u32x4 queries[Q::kShared ? Q::kFrags * kWave : 1];
    uint64_t scan[4];
  };
  __shared__ Shared shared;
  __shared__ int64_t found[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n_lane = lane & 15, g = lane >> 4;
  const int kv_heads = a.v.kv_heads;

  // rows of no request
  {
    int64_t row_lo = a.tokens, row_hi = a.tokens;
    if (a.requests > 0) {
      row_lo = min(max(load_int(a.starts, 0, a.len_bytes), int64_t{0}), a.tokens);
      row_hi = min(max(load_int(a.starts, a.requests, a.len_bytes), row_lo), a.tokens);
    }
    const int64_t none = row_lo + a.tokens - row_hi;
    if (none > 0) {
      const int64_t row16 = static_cast<int64_t>(a.heads) * DIM / 8;  // pieces of 16 bytes
      for (int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x; i < none * row16; i += int64_t{gridDim.x} * 256) {
        const int64_t row = i / row16;
        reinterpret_cast<uint4 *>(a.out)[(row < row_lo ? row : row - row_lo + row_hi) * row16 + i % row16] =
            uint4{0, 0, 0, 0};
      }
      if (a.lse)
        for (int64_t i = int64_t{blockIdx.x} * 256 + threadIdx.x; i < none * a.heads; i += int64_t{gridDim.x} * 256) {
          const int64_t row = i / a.heads;
          a.lse[(row < row_lo ? row : row - row_lo + row_hi) * a.heads + i % a.heads] = kNothing;
        }
    }
  }

  // Where this workgroup's units begin: in the list of items, or, without one, by counting: each thread a run of requests.
  int64_t per_head, mine = 0, at = 0, each = 0, b_lo = 0;
  if (items) {
    per_head = same(items[same(*item_count)].unit);
  } else {
    each = (a.requests + 255) / 256;
    b_lo = min(threadIdx.x * each, a.requests);
    const int64_t b_hi = min(b_lo + each, a.requests);
    for (int64_t b = b_lo; b < b_hi; ++b) mine += attn_units<kRows>(a, attn_request(a, b));
    uint64_t total;
    at = static_cast<int64_t>(block_exclusive_scan<uint64_t, 256>(static_cast<uint64_t>(mine), shared.scan, &total));
    per_head = same(static_cast<int64_t>(total));
  }
  const int64_t U = per_head * kv_heads;
  // With a unit for everyone, neighbours in the numbering of units are on one XCD: they read the same pages. With fewer
  // units than workgroups each has one, on all XCDs.
  const int64_t G = min(int64_t{gridDim.x}, U);
  const int64_t wg = G == gridDim.x && G % 8 == 0 ? (blockIdx.x & 7) * (G / 8) + (blockIdx.x >> 3) : blockIdx.x;
  if (threadIdx.x == 0) records[wg].first = -1;
  if (wg >= G) return;
  const int64_t u_begin = same(wg * U / G), u_end = same((wg + 1) * U / G);
  int head = same(static_cast<int>(u_begin / per_head));
  const int64_t x = u_begin - head * per_head;  // within one head's units
  int64_t b, item = 0;
  int row0 = 0;
  Request req;
  Span span;
  int64_t u_item;  // the item's first unit
  if (items) {
    const int64_t count = same(*item_count);
    int64_t lo = 0, width = count;  // the item is among [lo, lo + width)
    while (width > 1) {
      const int64_t step = (width + 255) / 256;
      const int64_t i = lo + threadIdx.x * step, end = min(i + step, lo + width);
      if (i < lo + width && items[i].unit <= x && x < items[end].unit) found[0] = i, found[1] = end - i;
      __syncthreads();
      lo = found[0], width = found[1];
      __syncthreads();
    }
    item = same(lo);
    const AttnItem it = items[item];
    b = same(it.request), row0 = same(it.row0);
    req = same(attn_request(a, b));
    span = same(attn_span<kRows>(a, req, row0));
    u_item = head * per_head + same(it.unit);
  } else {
    if (at <= x && x < at + mine) {
      int64_t i = b_lo, before = at;
      for (;; ++i) {
        const int64_t n = attn_units<kRows>(a, attn_request(a, i));
        if (x < before + n) break;
        before += n;
      }
      found[0] = i, found[1] = before;
    }
    __syncthreads();
    b = same(found[0]), u_item = head * per_head + same(found[1]);
    req = same(attn_request(a, b));
    span = same(attn_span<kRows>(a, req, 0));
    while (u_item + span.units <= u_begin) {
      u_item += span.units;
      row0 += kRows;
      span = same(attn_span<kRows>(a, req, row0));
    }
  }

  // scores in powers of two; a negative scale goes to the queries' signs
  // (a scale of 0 becomes the smallest number, with which a masked score stays where it is)
  const float scale2 = fmaxf(fabsf(a.scale) * 1.44269504088896340736f, __uint_as_float(1u));
  const uint32_t flip = a.scale < 0 ? 0x80008000u : 0u;
  const LaneOffsets offsets = lane_offsets<DIM>(lane, 1 << a.v.log2_page);
  for (int64_t u = u_begin; u < u_end;) {
    const int rows = min(kRows, req.queries * a.group - row0);
    Q q;
    q.shared = shared.queries;
    Sight<NT> sight;
    sight.sinks = a.window > 0 ? a.sinks : 0;
    sight.begin = span.begin, sight.end = span.end, sight.sink_end = span.sink_end;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 16 * n + n_lane;
      const uint32_t row = row0 + min(r, rows - 1);
      const uint32_t token = row / static_cast<uint32_t>(a.group);
      const int h = head * a.group + static_cast<int>(row - token * a.group);
      const int pos = r < rows ? req.before + static_cast<int>(token) : -1;
      sight.last[n] = min(pos, a.limit - 1);
      sight.after[n] = a.window > 0 && pos >= 0 ? pos - a.window : -1;
      const T *src = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head +
                     g * (DIM / 4);
      constexpr int kSteps = DIM / 32;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (Q::kShared && ((n * kSteps + i) & 3) != wave) continue;  // the waves fill LDS together
        u32x4 y = reinterpret_cast<const u32x4 *>(src)[i] ^ flip, z;
        if constexpr (kParts == 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const uint32_t both = y[j];
            const f16x2 v = __builtin_bit_cast(f16x2, both);
            const float v0 = static_cast<float>(v[0]), v1 = static_cast<float>(v[1]);
            const uint32_t hi = pack_bf16(v0, v1);
            y[j] = hi;
            z[j] = pack_bf16(v0 - __uint_as_float(hi << 16), v1 - __uint_as_float(hi & 0xffff0000u));
          }
        }
        if constexpr (Q::kShared) {
          shared.queries[(n * kSteps + i) * kWave + lane] = y;
          if constexpr (kParts == 2) shared.queries[((NT + n) * kSteps + i) * kWave + lane] = z;
        } else {
          q.own[n * kSteps + i] = y;
          if constexpr (kParts == 2) q.own[(NT + n) * kSteps + i] = z;
        }
      }
    }
    if constexpr (Q::kShared) __syncthreads();
    // All rows see a whole tile that ends at or before the first row's place and begins in the last row's window.
    const int pos_first = same(min(
        req.before + static_cast<int>(static_cast<uint32_t>(row0) / static_cast<uint32_t>(a.group)), a.limit - 1));
    const int after_last = same(
        a.window > 0
            ? max(req.before + static_cast<int>(static_cast<uint32_t>(row0 + rows - 1) / static_cast<uint32_t>(a.group)), -1) -
                  a.window
            : -1);
    const int32_t *table = a.table + b * a.table_stride;
    const int first = same(static_cast<int>(u - u_item));
    const int last = same(static_cast<int>(min(u_item + span.units, u_end) - u_item));
    auto token_of = [&](int k) {  // unit k's first token of this wave
      return (k < span.sink_tiles ? k : span.tile0 + k - span.sink_tiles) * kUnit + wave * kWaveTokens;
    };
    // The page of the 16 tokens from j on; -1 where no row sees any of them.
    auto page_at = [&](const int32_t *entries, const Span &sp, int j) {
      int p = -1;
      if (j < sp.end && (j + 15 >= sp.begin || j < sp.sink_end)) p = entries[j >> a.v.log2_page];
      return p >= 0 && p < a.v.pages ? p : -1;
    };
    // Whether all rows see all of a wave's 32 tokens from token0 on, on pages p0 and p1.
    auto tile_whole = [&](int token0, int p0, int p1) {
      return p0 >= 0 && p1 >= 0 && token0 + kWaveTokens - 1 <= pos_first &&
             (token0 > after_last || token0 + kWaveTokens <= sight.sinks);
    };
    // The pages of the next 32 units' tokens, one 16 of them a lane: -1 where no row sees any.
    int page_of = -1, page_base = 0;
    auto look_up = [&](int k0) {
      page_base = k0;
      const int k = k0 + (lane >> 1);
      page_of = k < last ? page_at(table, span, token_of(k) + 16 * (lane & 1)) : -1;
    };
    struct Step {
      int token0, page0, page1;
    };
    // The next unit from k on that has anything for this wave; `last` if there is none.
    auto find = [&](int k) {
      for (; k < last; ++k) {
        if (k - page_base >= 32) look_up(k);
        const int at = 2 * (k - page_base);
        if (__builtin_amdgcn_readlane(page_of, at) >= 0 || __builtin_amdgcn_readlane(page_of, at + 1) >= 0) break;
      }
      return k;
    };
    KvTile<DIM> ahead;
    auto fetch = [&](int k) {
      Step s;
      s.token0 = token_of(k);
      s.page0 = __builtin_amdgcn_readlane(page_of, 2 * (k - page_base));
      s.page1 = __builtin_amdgcn_readlane(page_of, 2 * (k - page_base) + 1);
      const int mask = (1 << a.v.log2_page) - 1;  // a half that is not there is loaded as page 0 and not looked at
      load_half<DIM>(a.v, head, max(s.page0, 0), s.token0 & mask, offsets, 0, ahead);
      load_half<DIM>(a.v, head, max(s.page1, 0), (s.token0 + 16) & mask, offsets, 1, ahead);
      return s;
    };
    bool wild = false, again;
    RowState<DIM, NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n) st.top[n] = kNothing;
    // Nothing in this loop changes the accumulators but the products, on every way through it: only so do they stay in one
    // place.
    do {
      again = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        st.sum[n] = 0;
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i) st.acc[n][i] = f32x4{0, 0, 0, 0};
      }
      look_up(first);
      int k = find(first);
      if (k >= last) break;
      Step next = fetch(k);
      bool more;
      do {
        const Step now = next;
        KvTile<DIM> t = ahead;
        k = find(k + 1);
        more = k < last;
        if (more) next = fetch(k);
        const bool whole = tile_whole(now.token0, now.page0, now.page1);
        again = attend_tile<DIM, NT, kParts>(t, q, st, scale2, lane, whole, now.token0, now.page0 >= 0, now.page1 >= 0, sight,
                                             wild);
      } while (more && !again);
    } while (again);
    u = u_item + last;

    // The four waves' states, 16 rows at a time, into the result or into a part.
    const bool begins = u_item >= u_begin, ends = last == span.units;
    const int64_t slot = 2 * wg + (begins ? 1 : 0);
    const bool any_wild = __syncthreads_or(wild);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (16 * n < rows) {
        const float sum = across_sum(st.sum[n]);
        if (g == 0) {
          shared.join.top[wave][n_lane] = st.top[n];
          shared.join.sum[wave][n_lane] = sum;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < DIM / 16; i += 4)
            *reinterpret_cast<f32x4 *>(
                &shared.join.acc[wave][n_lane * JoinShared<DIM>::kStride + (4 * g + r) * (DIM / 16) + i]) =
                f32x4{st.acc[n][i][r], st.acc[n][i + 1][r], st.acc[n][i + 2][r], st.acc[n][i + 3][r]};
        __syncthreads();
        const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (DIM / 16);
        if (16 * n + r < rows) {
          float top = kNothing;
#pragma unroll
          for (int v = 0; v < 4; ++v) top = fmaxf(top, shared.join.top[v][r]);
          const float base = fmaxf(top, kLowest);
          float f[4], total = 0;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            f[v] = __builtin_amdgcn_exp2f(shared.join.top[v][r] - base);
            total += f[v] * shared.join.sum[v][r];
          }
          const uint32_t row = row0 + 16 * n + r;
          const uint32_t token = row / static_cast<uint32_t>(a.group);
          const int h = head * a.group + static_cast<int>(row - token * a.group);
          const int64_t line = (req.first_row + token) * a.heads + h;
          f32x4 o[DIM / 64];
#pragma unroll
          for (int i = 0; i < DIM / 64; ++i) {
            o[i] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int v = 0; v < 4; ++v)
              o[i] += f[v] * *reinterpret_cast<const f32x4 *>(&shared.join.acc[v][r * JoinShared<DIM>::kStride + d0 + 4 * i]);
          }
          if (any_wild) {
            const int pos = req.before + static_cast<int>(token);
            const int see_last = min(pos, a.limit - 1), see_after = a.window > 0 && pos >= 0 ? pos - a.window : -1;
            const T *q_row = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head;
            const int page = 1 << a.v.log2_page;
#pragma unroll 1
            for (int j16 = 0; j16 < (last - first) * (kUnit / 16); ++j16) {
              const int k = first + j16 / (kUnit / 16);
              const int j0 = (k < span.sink_tiles ? k : span.tile0 + k - span.sink_tiles) * kUnit + j16 % (kUnit / 16) * 16;
              const int t0 = j0 & ~(kWaveTokens - 1);
              const int p0 = page_at(table, span, t0), p1 = page_at(table, span, t0 + 16), at = j0 == t0 ? p0 : p1;
              if (at < 0 || tile_whole(t0, p0, p1)) continue;
              const int64_t tile = int64_t{2} * head << a.v.log2_page;
              const int off = j0 & (page - 1);
              const uint8_t *codes = a.v.cache + at * a.v.cache_stride + (tile + off) * (DIM / 2);
              const uint8_t *sc = a.v.scales + at * a.v.scales_stride + tile * (DIM / 32) + off;
#pragma unroll 1
              for (int i = 0; i < 16; ++i) {
                const int j = j0 + i;
                const uint32_t byte = sc[(DIM / 32 + d0 / 32) * page + i];
                if (byte < kWild || j > see_last || (j <= see_after && j >= sight.sinks)) continue;
                const float x = score_of<T, DIM>(q_row, codes + i * (DIM / 2), sc + i, page);
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(a.scale < 0 ? -x : x, scale2, -base));
                const uint8_t *v = codes + (page + i) * (DIM / 2) + d0 / 2;
#pragma unroll
                for (int d = 0; d < DIM / 16; d += 2) {
                  const f32x2 y = decode2_f32<0>(v[d / 2], scale_operand(byte));
                  o[d / 4][d % 4] += e * y[0];
                  o[d / 4][d % 4 + 1] += e * y[1];
                }
              }
            }
          }
          const float inv = total == 0 ? 0 : 1 / total;
#pragma unroll
          for (int i = 0; i < DIM / 64; ++i) {
            if (begins && ends) {
              typedef T out_vec __attribute__((ext_vector_type(4)));
              *reinterpret_cast<out_vec *>(static_cast<T *>(a.out) + line * DIM + d0 + 4 * i) =
                  out_vec{static_cast<T>(o[i][0] * inv), static_cast<T>(o[i][1] * inv), static_cast<T>(o[i][2] * inv),
                          static_cast<T>(o[i][3] * inv)};
            } else {
              *reinterpret_cast<f32x4 *>(parts + (slot * kRows + 16 * n + r) * DIM + d0 + 4 * i) = o[i];
            }
          }
          if ((threadIdx.x & 15) == 0) {
            if (begins && ends) {
              if (a.lse) a.lse[line] = total == 0 ? kNothing : (top + __builtin_log2f(total)) * 0.69314718055994530942f;
            } else {
              part_stats[(slot * kRows + 16 * n + r) * 2] = top;
              part_stats[(slot * kRows + 16 * n + r) * 2 + 1] = total;
            }
          }
        }
        __syncthreads();
      }
    }
    if (!begins && ends && threadIdx.x == 0) {
      // begun by the last workgroup whose units begin at the item's first unit or before it
      records[wg] = JoinRecord{static_cast<int32_t>(((u_item + 1) * G - 1) / U), head, rows, row0, req.first_row};
    }
    if (u >= u_end) break;
    // the next item
    u_item = u;
    if (items) {
      if (++item == same(*item_count)) item = 0, ++head;
      const AttnItem it = items[item];
      if (same(it.request) != b) req = same(attn_request(a, same(it.request)));
      b = same(it.request), row0 = same(it.row0);
    } else {
      row0 += kRows;
      if (row0 >= req.queries * a.group) {
        row0 = 0;
        do {
          if (++b == a.requests) b = 0, ++head;
          req = same(attn_request(a, b));
        } while (req.queries == 0);
      }
    }
    span = same(attn_span<kRows>(a, req, row0));
  }
}

// Puts the parts of the items together that more than one workgroup had a share in. Every workgroup makes itself a list of the
// rows to join (a grid that has a workgroup for each row that there could be takes longer to start than to run). Where they
// are few, a workgroup takes one at a time, its teams of DIM / 4 threads a part each; else every team takes a row.
constexpr int kMostGroups = 256 * 4;

template <typename T, int DIM, int ROWS>
__global__ __launch_bounds__(256) void page_attention_join_kernel(AttnArgs a, const float *parts, const float *part_stats,
                                                                  const JoinRecord *records, int groups) {
  constexpr int kLanes = DIM / 4, kTeams = 256 / kLanes, kEach = kMostGroups / 256;
  __shared__ uint32_t before[kMostGroups + 1];  // rows to join in front of each workgroup's record
  __shared__ uint32_t scan[4];
  __shared__ f32x4 acc_shared[kTeams][kLanes];
  __shared__ float top_shared[kTeams], sum_shared[kTeams];
  uint32_t rows[kEach], mine = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int w = threadIdx.x * kEach + i;
    rows[i] = w < groups && records[w].first >= 0 ? records[w].rows : 0;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += rows[i];
  uint32_t total;
  uint32_t at = block_exclusive_scan<uint32_t, 256>(mine, scan, &total);
#pragma unroll
  for (int i = 0; i < kEach; ++i) before[threadIdx.x * kEach + i] = at, at += rows[i];
  if (threadIdx.x == 0) before[kMostGroups] = total;
  __syncthreads();
  const int team = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  const bool few = total <= 2 * gridDim.x;
  const uint32_t step = few ? 1 : kTeams;
  for (uint32_t base_row = blockIdx.x * step; base_row < total; base_row += gridDim.x * step) {
    const uint32_t row_at = few ? base_row : base_row + team;
    float top = kNothing, sum = 0;
    f32x4 acc = {0, 0, 0, 0};
    int64_t line_out = 0;
    if (row_at < total) {
      int w_end = 0, last = groups - 1;  // the last record with no more rows in front of it
      while (w_end < last) {
        const int mid = (w_end + last + 1) >> 1;
        if (before[mid] <= row_at) w_end = mid; else last = mid - 1;
      }
      const JoinRecord rec = records[w_end];
      const int r = row_at - before[w_end];
      const uint32_t row = rec.row0 + r, token = row / static_cast<uint32_t>(a.group);
      line_out = (rec.first_row + token) * a.heads + rec.head * a.group + (row - token * a.group);
      constexpr int kBatch = 4;  // parts in flight
      const int stride = few ? kTeams : 1;
      for (int w0 = rec.first + (few ? team : 0); w0 <= w_end; w0 += stride * kBatch) {
        f32x2 stats[kBatch];
        f32x4 o[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int64_t w = min(w0 + i * stride, w_end);
          const int64_t line = (2 * w + (w == rec.first ? 1 : 0)) * ROWS + r;
          stats[i] = *reinterpret_cast<const f32x2 *>(part_stats + line * 2);
          o[i] = *reinterpret_cast<const f32x4 *>(parts + line * DIM + lane * 4);
        }
        float next = top;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) next = fmaxf(next, stats[i][0]);
        const float base = fmaxf(next, kLowest), f = __builtin_amdgcn_exp2f(top - base);
        sum *= f, acc *= f;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (w0 + i * stride > w_end) continue;
          const float e = __builtin_amdgcn_exp2f(stats[i][0] - base);
          sum += stats[i][1] * e;
          acc += o[i] * e;
        }
        top = next;
      }
    }
    if (few) {
      acc_shared[team][lane] = acc;
      if (lane == 0) top_shared[team] = top, sum_shared[team] = sum;
      __syncthreads();
      for (int i = 0; i < kTeams; ++i) top = fmaxf(top, top_shared[i]);
      const float base = fmaxf(top, kLowest);
      sum = 0, acc = f32x4{0, 0, 0, 0};
      for (int i = 0; i < kTeams; ++i) {
        const float f = __builtin_amdgcn_exp2f(top_shared[i] - base);
        sum += f * sum_shared[i];
        acc += f * acc_shared[i][lane];
      }
      __syncthreads();
    }
    if (row_at < total && (!few || team == 0)) {
      const float inv = sum == 0 ? 0 : 1 / sum;
      typedef T out_vec __attribute__((ext_vector_type(4)));
      *reinterpret_cast<out_vec *>(static_cast<T *>(a.out) + line_out * DIM + lane * 4) = out_vec{
          static_cast<T>(acc[0] * inv), static_cast<T>(acc[1] * inv), static_cast<T>(acc[2] * inv), static_cast<T>(acc[3] * inv)};
      if (a.lse && lane == 0) a.lse[line_out] = sum == 0 ? kNothing : (top + __builtin_log2f(sum)) * 0.69314718055994530942f;
    }
  }
}

// ---- launch ------------------------------------------------------------------------

struct AttnShape {
  int tiles;       // of 16 rows an item
  int64_t groups;  // workgroups
  int64_t items;   // room in the list of items; 0: none, every request is one item of a head
  int64_t parts_bytes, stats_bytes, record_bytes, item_bytes, first_bytes;
  int64_t bytes() const { return parts_bytes + stats_bytes + record_bytes + item_bytes + first_bytes; }
};

// How many rows an item has, and how many workgroups share the units: as many as the card holds at once.
inline AttnShape attn_shape(int64_t tokens, int heads, int kv_heads, int dim, int64_t requests, int64_t max_query_len) {
  const int64_t longest = max_query_len > 0 ? std::min(max_query_len, tokens) : std::max<int64_t>(tokens - requests + 1, 1);
  const int64_t group = heads / kv_heads, rows = longest * group;
  AttnShape s;
  s.tiles = rows <= 16 ? 1 : rows <= 32 || dim == 256 ? 2 : 4;
  s.groups = 256 * attn_waves(dim, s.tiles);
  s.items = rows > 16 * s.tiles ? tokens * group / (16 * s.tiles) + requests : 0;
  const int64_t lines = 2 * s.groups * 16 * s.tiles;
  s.parts_bytes = lines * dim * 4;
  s.stats_bytes = lines * 8;
  s.record_bytes = s.groups * static_cast<int64_t>(sizeof(JoinRecord));
  s.item_bytes = s.items ? (s.items + 2) * static_cast<int64_t>(sizeof(AttnItem)) : 0;  // the count behind the last one
  s.first_bytes = s.items ? (requests + 4) / 4 * 16 : 0;
  return s;
}

template <typename T, int DIM, int NT>
void launch_tiles(const AttnArgs &a, const AttnShape &s, void *scratch, hipStream_t stream) {
  char *at = static_cast<char *>(scratch);
  float *parts = reinterpret_cast<float *>(at);
  float *stats = reinterpret_cast<float *>(at += s.parts_bytes);
  JoinRecord *records = reinterpret_cast<JoinRecord *>(at += s.stats_bytes);
  AttnItem *items = nullptr;
  int32_t *count = nullptr;
  if (s.items) {
    items = reinterpret_cast<AttnItem *>(at += s.record_bytes);
    count = reinterpret_cast<int32_t *>(items + s.items + 1);
    int32_t *first_item = reinterpret_cast<int32_t *>(at += s.item_bytes);
    hipLaunchKernelGGL((page_attention_items_kernel<16 * NT>), dim3(1), dim3(1024), 0, stream, a, first_item, items,
                       s.items, count);
  }
  // no more workgroups than there can be units
  const int64_t units = (a.tokens * a.group / (16 * NT) + a.requests) * a.v.kv_heads * (a.limit / kUnit + 1);
  const unsigned groups = static_cast<unsigned>(std::min(s.groups, std::max<int64_t>(units, 1)));
  hipLaunchKernelGGL((page_attention_kernel<T, DIM, NT>), dim3(groups), dim3(256), 0, stream, a, items, count, parts, stats,
                     records);
  hipLaunchKernelGGL((page_attention_join_kernel<T, DIM, 16 * NT>), dim3(std::min(groups, 512u)), dim3(256), 0, stream, a,
                     parts, stats, records, static_cast<int>(groups));
}

template <typename T, int DIM>
void launch_dim(const AttnArgs &a, const AttnShape &s, void *scratch, hipStream_t stream) {
  if (s.tiles == 1) return launch_tiles<T, DIM, 1>(a, s, scratch, stream);
  if (s.tiles == 2) return launch_tiles<T, DIM, 2>(a, s, scratch, stream);
  if constexpr (DIM < 256) launch_tiles<T, DIM, 4>(a, s, scratch, stream);
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
  return attn_shape(tokens, heads, kv_heads, dim, requests, max_query_len).bytes();
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
  SHMT_REQUIRE(tokens * heads < (int64_t{1} << 30), "query rows x heads must be below 2^30");
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
  const AttnShape shape = attn_shape(tokens, heads, cache->kv_heads, cache->dim, requests, max_query_len);
  if (scratch_bytes < shape.bytes() || !scratch) {
    set_error("scratch too small: %lld bytes, needed %lld", static_cast<long long>(scratch_bytes),
              static_cast<long long>(shape.bytes()));
    return SHMT_ENOMEM;
  }
  SHMT_REQUIRE((reinterpret_cast<int64_t>(scratch) & 15) == 0, "scratch has to begin on 16 bytes");
  constexpr int64_t kMost = 0x7fffffff;  // a longer window, or more sinks, than any request has tokens
  const AttnArgs a{v, query, query_token_stride, query_head_stride, tokens, heads, heads / cache->kv_heads, block_table,
                   table_stride, query_starts, kv_lens, len_bytes, requests, softmax_scale,
                   static_cast<int32_t>(std::min(window, kMost)), static_cast<int32_t>(std::min(sinks, kMost)),
                   v.pages > 0 ? static_cast<int32_t>(width * cache->page) : 0, out, lse};
  if (elem_type == SHMT_F16) launch_attention<_Float16>(a, cache->dim, shape, scratch, as_stream(stream));
  else launch_attention<__bf16>(a, cache->dim, shape, scratch, as_stream(stream));
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
