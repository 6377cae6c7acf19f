// What the two attention kernels over the paged 4-bit cache share: how the work is cut and numbered, how tokens are read and
// decoded, the join of parts.
#pragma once
#include "common.h"
#include "paged_dev.h"
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
// place. Units are numbered (few rows: request by request, head by head, row tile by row tile; many: head by head, request by
// request, row tile by row tile), and workgroups take equal runs of them, so all end at about the same time whatever the
// lengths are. An item may be shared by several workgroups; each leaves a part (reference, sum, weighted values), which
// page_attention_join_kernel puts together.
constexpr int kUnit = 128;  // tokens: four waves of 32
constexpr int kWaveTokens = 32;
constexpr float kNothing = -__builtin_inff();
constexpr float kLowest = -3.40282347e38f;  // the lowest float, subtracted instead of kNothing, so that nothing stays nothing

// Beginning and ending an item costs about as much as this many units: so many are added to each, without tokens in them, for
// the sake of even shares.
constexpr int item_cost(int rows) { return rows > 32 ? 2 : 1; }

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
  s.units = max(s.sink_tiles + (s.end + kUnit - 1) / kUnit - s.tile0, 1) + item_cost(ROWS);
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

// Division of numbers that mostly fit 32 bits.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
  if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
}

// U units for G workgroups: workgroup w takes units floor(w U / G) up to floor((w + 1) U / G), so that longer shares are spread
// evenly over the workgroups, and with them over the XCDs.
struct Shares {
  int64_t U, G, each, more;
  __device__ __forceinline__ Shares(int64_t units, int64_t groups) : U(units), G(groups), each(divide(units, groups)) {
    more = U - each * G;
  }
  __device__ __forceinline__ int64_t begin(int64_t w) const { return w * each + divide(w * more, G); }
  __device__ __forceinline__ int64_t owner(int64_t u) const { return divide((u + 1) * G - 1, U); }  // of unit u
};

// Where a workgroup begins, as the thread that found it tells the others.
struct Found {
  Request req;
  int64_t request, before, units;  // units in front of the request (many: of the item), of the request for one head
};

// Rows in front of row_lo and from row_hi on, which belong to no request, are 0.
template <typename T, int DIM>
__device__ __forceinline__ void attn_clear_rows(const AttnArgs &a, int64_t row_lo, int64_t row_hi) {
  const int64_t none = row_lo + a.tokens - row_hi;
  if (none <= 0) return;
  const int64_t row16 = static_cast<int64_t>(a.heads) * DIM / 8;  // pieces of 16 bytes
  for (int64_t i = int64_t{blockIdx.x} * blockDim.x + threadIdx.x; i < none * row16; i += int64_t{gridDim.x} * blockDim.x) {
    const int64_t row = i / row16;
    reinterpret_cast<uint4 *>(a.out)[(row < row_lo ? row : row - row_lo + row_hi) * row16 + i % row16] = uint4{0, 0, 0, 0};
  }
  if (!a.lse) return;
  for (int64_t i = int64_t{blockIdx.x} * blockDim.x + threadIdx.x; i < none * a.heads; i += int64_t{gridDim.x} * blockDim.x) {
    const int64_t row = i / a.heads;
    a.lse[(row < row_lo ? row : row - row_lo + row_hi) * a.heads + i % a.heads] = kNothing;
  }
}

__device__ __forceinline__ int row_token(const AttnArgs &a, int row) {
  return static_cast<int>(static_cast<uint32_t>(row) / static_cast<uint32_t>(a.group));
}

// First token of an item's unit.
__device__ __forceinline__ int unit_token(const Span &s, int k) {
  return (k < s.sink_tiles ? k : s.tile0 + k - s.sink_tiles) * kUnit;
}

// The page of the 16 tokens from j on; -1 where no row of the item sees any of them.
__device__ __forceinline__ int page_at(const AttnArgs &a, const int32_t *table, const Span &s, int j) {
  int p = -1;
  if (j < s.end && (j + 15 >= s.begin || j < s.sink_end)) p = table[j >> a.v.log2_page];
  return p >= 0 && p < a.v.pages ? p : -1;
}

// What a row at place `pos` sees: tokens up to `last` that are behind `after`, or first ones.
struct Sees {
  int last, after;
};
__device__ __forceinline__ Sees row_sees(const AttnArgs &a, int pos) {
  return {min(max(pos, -1), a.limit - 1), a.window > 0 && pos >= 0 ? pos - a.window : -1};
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

// Where 16 tokens of one head lie: the first one's key and its scale. Lanes hold those of the tokens to come; a wave takes one
// lane's for a load, so that nothing of it is computed per lane or per step.
struct Place16 {
  uint32_t row_lo, row_hi, scale_lo, scale_hi;
  __device__ __forceinline__ Place16 of_lane(int l) const {
    return {static_cast<uint32_t>(__builtin_amdgcn_readlane(row_lo, l)), static_cast<uint32_t>(__builtin_amdgcn_readlane(row_hi, l)),
            static_cast<uint32_t>(__builtin_amdgcn_readlane(scale_lo, l)),
            static_cast<uint32_t>(__builtin_amdgcn_readlane(scale_hi, l))};
  }
  __device__ __forceinline__ const uint8_t *row() const {
    return reinterpret_cast<const uint8_t *>(static_cast<uint64_t>(row_hi) << 32 | row_lo);
  }
  __device__ __forceinline__ const uint8_t *scale() const {
    return reinterpret_cast<const uint8_t *>(static_cast<uint64_t>(scale_hi) << 32 | scale_lo);
  }
};
// Those of page `at` from the place of token j on.
template <int DIM>
__device__ __forceinline__ Place16 place16(const PagedView &v, int head, int at, int j) {
  const int off = j & ((1 << v.log2_page) - 1);
  const int64_t tile = int64_t{2} * head << v.log2_page;
  const uint64_t row = reinterpret_cast<uint64_t>(v.cache + at * v.cache_stride + (tile + off) * (DIM / 2));
  const uint64_t scale = reinterpret_cast<uint64_t>(v.scales + at * v.scales_stride + tile * (DIM / 32) + off);
  return {static_cast<uint32_t>(row), static_cast<uint32_t>(row >> 32), static_cast<uint32_t>(scale),
          static_cast<uint32_t>(scale >> 32)};
}

// Loads 16 tokens.
template <int DIM>
__device__ __forceinline__ void load_half(const Place16 &at, int page, const LaneOffsets &o, int half, KvTile<DIM> &t) {
  const uint8_t *rows = at.row(), *sc = at.scale();
  if constexpr (DIM == 64) {
    const uint2 x = *reinterpret_cast<const uint2 *>(rows + o.key);
    t.key[half][0] = x.x, t.key[half][1] = x.y;
    t.key_scale[half][0] = sc[o.key_scale];
  } else {
#pragma unroll
    for (int i = 0; i < DIM / 128; ++i) {
      const uint4 x = *reinterpret_cast<const uint4 *>(rows + o.key + 16 * i);
      t.key[half][4 * i] = x.x, t.key[half][4 * i + 1] = x.y, t.key[half][4 * i + 2] = x.z, t.key[half][4 * i + 3] = x.w;
      t.key_scale[half][i] = sc[o.key_scale + i * page];
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

// The weights of eight scores of a row, in units of `unit` powers of two, relative to its reference, as the right operand of
// V^T P^T.
template <int PARTS, int NT>
__device__ __forceinline__ void weights(const f32x4 (&s)[2], float unit, float top, float &sum, u32x4 (&w)[PARTS][NT], int n) {
  const float base = fmaxf(top, kLowest);
  float e[8], add = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 4][j % 4], unit, -base));
    add += e[j];
  }
  sum += add;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t hi = pack_bf16(e[2 * j], e[2 * j + 1]);
    w[0][n][j] = hi;
    if constexpr (PARTS == 2)
      w[1][n][j] = pack_bf16(e[2 * j] - __uint_as_float(hi << 16), e[2 * j + 1] - __uint_as_float(hi & 0xffff0000u));
  }
}

// References. Weights are taken relative to the maximum of the first tile in which a row sees anything: with floats' exponents
// any reference near the true maximum does as well as that, so there is no maximum to follow from tile to tile and nothing to
// rescale (kFirst). Two things make that too little. A row's later scores may be so much greater that its weights sum up to more
// than 2^40: then the tokens are begun again, with a reference that is greater by as much (kRaised). And a weight comes
// from the product score * scale as it is, the reference is that product rounded: from 2^30 on, half a unit in its last place
// is more than an exponent of 2 may move by, and weights would be anything. Where a reference is far from 0 (2^12), or
// raising it once was not enough, the tokens are gone through twice, with scores in powers of two that are rounded: once for
// each row's maximum (kMaximum), once with that as the reference (kRounded), to which no weight is above 1. So there are four
// passes at most, whatever the scores are. Waves that share a row may have weighted it either way: below 2^12 that makes a
// difference of 2^-13 of a weight, and scores that are tied stay tied above.
enum : int { kFirst, kRaised, kMaximum, kRounded };
constexpr float kPassed = 1099511627776.0f;  // 2^40
constexpr float kFar = 4096.0f;

template <int NT>
__device__ __forceinline__ float most_of(const f32x4 (&s)[NT][2], int n) {
  float x = s[n][0][0];
#pragma unroll
  for (int j = 1; j < 8; ++j) x = fmaxf(x, s[n][j / 4][j % 4]);
  return across_max(x);
}

// What softmax_scale makes of scores, in powers of two. A negative scale goes to the queries' signs; a scale of 0 becomes the
// smallest number, with which a masked score stays where it is.
__device__ __forceinline__ float powers_of_two(const AttnArgs &a) {
  return fmaxf(fabsf(a.scale) * 1.44269504088896340736f, __uint_as_float(1u));
}

// Rows without a reference take this tile's maximum. Returns whether any is still without; `again` and `far` are set for one
// that is far from 0.
template <int NT, typename State, typename Flag>
__device__ __forceinline__ bool first_reference(const f32x4 (&s)[NT][2], float scale2, State &st, Flag &again, Flag &far) {
  bool none = false, is_far = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float most = most_of<NT>(s, n) * scale2;
    st.top[n] = st.top[n] == kNothing ? most : st.top[n];
    none |= st.top[n] == kNothing;
    is_far |= st.top[n] != kNothing && fabsf(st.top[n]) >= kFar;
  }
  if (__ballot(is_far)) again = far = 1;
  return __ballot(none) != 0;
}

// Scores in powers of two, rounded; and, on the way to the maximum, that as far as it is known.
template <int NT, typename State>
__device__ __forceinline__ void round_scores(f32x4 (&s)[NT][2], float scale2, State &st, int pass) {
#pragma clang fp contract(off)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) s[n][j / 4][j % 4] = s[n][j / 4][j % 4] * scale2;
  if (pass != kMaximum) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) st.top[n] = fmaxf(st.top[n], most_of<NT>(s, n));
}

// Where a row's sum has passed 2^40: a reference that is greater by the sum's logarithm, so that no weight so far is above 1 to
// it, and a new sum, which is for the rest of the pass to see whether that is enough. `again` is set if there is such a row,
// `far` if its reference is far from 0 (an infinite sum has an infinite logarithm).
template <int NT, typename State, typename Flag>
__device__ __forceinline__ void raise_reference(State &st, Flag &again, Flag &far) {
  bool passed = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) passed |= st.sum[n] > kPassed;
  if (__builtin_expect(__ballot(passed) == 0, 1)) return;
  bool is_far = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float sum = across_max(st.sum[n]);
    if (sum > kPassed) {
      st.top[n] += __builtin_log2f(sum), st.sum[n] = 0;
      is_far |= fabsf(st.top[n]) >= kFar;
    }
  }
  again = 1;
  if (__ballot(is_far)) far = 1;
}

// Scale bytes from here on make values that are infinite in bfloat16, or not a number.
constexpr uint32_t kWild = 253;

// One wave's step over 32 tokens.
//   S^T = K Q^T, 16 tokens x 16 rows at a time: lane (n, g) gets the scores of row n with tokens 4g .. 4g + 3, which is
//   the place that the weights need to have as the right operand of O^T += V^T P^T (contraction over tokens, which may be
//   numbered in any order as long as both operands agree): nothing crosses lanes but the maximum.
// Keys and values become bfloat16 exactly. Weights are held as the sum of two bfloat16 (16 bits), as are float16 queries.
// Rounded to one, the weights of bfloat16 queries would save half of the second product and move results by as much as their
// own rounding does (64 ragged decodes: 2.3e-3 off instead of 1.66e-3, which is the result's rounding alone). That buys
// nothing where HBM is the bound (these 84.5 us either way, 32 decodes of 8,000 tokens with 128 / 256 dimensions 57 / 113 us
// against 57 / 113, with 64 41 against 38; 7 tokens each of 16 requests 45 against 40).
// `whole`: all rows see all tokens. Otherwise scores are masked; and values that are not finite in bfloat16 must not meet the
// weight 0 of a row that does not see them: they are left out (`wild` says so) and added at the end of the item.
// FIRST: `pass` is kFirst or kRaised; rows may be `waiting` for a reference. `again` is set if the wave has to begin its tokens
// again, `far` if with rounded scores.
template <bool FIRST, int DIM, int NT, int PARTS>
__device__ __forceinline__ void attend_tile(KvTile<DIM> &t, const Queries<DIM, NT, PARTS> &q, RowState<DIM, NT> &st,
                                            float scale2, int pass, int lane, bool whole, int token0, bool there0,
                                            bool there1, const Sight<NT> &sight, bool &wild, bool &waiting, bool &again,
                                            bool &far) {
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
  if constexpr (!FIRST) round_scores<NT>(s, scale2, st, pass);
  else if (waiting) waiting = first_reference<NT>(s, scale2, st, again, far);
  u32x4 w[2][NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) weights<2>(s[n], FIRST ? scale2 : 1.0f, st.top[n], st.sum[n], w, n);
  if constexpr (FIRST) raise_reference<NT>(st, again, far);
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
        for (int p = 0; p < 2; ++p) {
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

// Eight values of a query row as a fragment: bfloat16 as they are, float16 as the sum of two. What is not a row is 0: its
// scores are its reference then, whatever the rows beside it score.
template <typename T>
__device__ __forceinline__ void query_fragment(const T *src, bool there, uint32_t flip, u32x4 &y, u32x4 &z) {
  y = (*reinterpret_cast<const u32x4 *>(src) ^ flip) & (there ? 0xffffffffu : 0u);
  if constexpr (std::is_same<T, _Float16>::value) {
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

// Adds, for one row and DIM / 16 of its dimensions from d0 on, the values of the 16 tokens from j0 on (page `at`) that the
// products left out: those that are not finite in bfloat16 and that the row sees.
template <typename T, int DIM>
__device__ __forceinline__ void add_left_out(const AttnArgs &a, int head, int at, int j0, const T *q_row, const Sees &sees,
                                             float scale2, float base, int d0, f32x4 (&o)[DIM / 64]) {
#pragma clang fp contract(off)
  if (at < 0) return;
  const int page = 1 << a.v.log2_page, off = j0 & (page - 1);
  const int64_t tile = int64_t{2} * head << a.v.log2_page;
  const uint8_t *codes = a.v.cache + at * a.v.cache_stride + (tile + off) * (DIM / 2);
  const uint8_t *sc = a.v.scales + at * a.v.scales_stride + tile * (DIM / 32) + off;
  const int sinks = a.window > 0 ? a.sinks : 0;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const int j = j0 + i;
    const uint32_t byte = sc[(DIM / 32 + d0 / 32) * page + i];
    if (byte < kWild || j > sees.last || (j <= sees.after && j >= sinks)) continue;
    const float x = score_of<T, DIM>(q_row, codes + i * (DIM / 2), sc + i, page);
    const float e = __builtin_amdgcn_exp2f((a.scale < 0 ? -x : x) * scale2 - base);  // scores rounded, as in kRounded
    const uint8_t *v = codes + (page + i) * (DIM / 2) + d0 / 2;
#pragma unroll
    for (int d = 0; d < DIM / 16; d += 2) {
      const f32x2 y = decode2_f32<0>(v[d / 2], scale_operand(byte));
      o[d / 4][d % 4] += e * y[0];
      o[d / 4][d % 4 + 1] += e * y[1];
    }
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
  const bool few = total <= 1024;
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

// What a launch works with besides its arguments.
struct AttnScratch {
  float *parts, *stats;  // two parts a workgroup; {maximum, sum} of each row
  JoinRecord *records;
  AttnItem *items;       // many rows: the list of items, the count behind it
  int32_t *count, *first_item;
  int64_t room;          // items
};

// How many rows an item has, and how many workgroups share the units: as many as the card holds at once.
struct AttnShape {
  bool many;       // rows: 32 a wave instead of 16 or 32 a workgroup
  int rows;        // of an item
  int64_t groups;  // workgroups
  int64_t items;   // many: room in the list
  int64_t parts_bytes, stats_bytes, record_bytes, item_bytes, first_bytes;
  int64_t bytes() const { return parts_bytes + stats_bytes + record_bytes + item_bytes + first_bytes; }
};

constexpr int many_rows(int dim) { return dim == 256 ? 128 : 256; }

// paged_attention_many.hip
void launch_attention_many(const AttnArgs &a, int dim, int elem_type, unsigned groups, const AttnScratch &s, hipStream_t stream);
int attn_many_groups();

}  // namespace shmt
