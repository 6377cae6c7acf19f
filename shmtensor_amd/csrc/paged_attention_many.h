// Attention over the paged key/value cache: the kernel for many rows a request (prompts, chunks of prompts, large trees, whole
// answers over an encoder's states), in which the waves of a workgroup share the rows.
#pragma once
#include "paged_attention.h"

namespace shmt {

// Items of all requests with the units in front of each, for calls in which a request has many row tiles: one workgroup.
// items[0 .. n) and, behind the last, the number of units; *count = n. (Only starts that descend could make more items than
// there is room for.)
template <int SEEN, int ROWS, bool FINE>
__global__ __launch_bounds__(1024) void page_attention_items_kernel(AttnArgs a, int32_t *first_item, AttnItem *items,
                                                                    int64_t room, int32_t *count) {
  __shared__ uint64_t lds[16];
  int64_t n = 0;
  for (int64_t base = 0; base < a.requests; base += 1024) {
    const int64_t b = base + threadIdx.x;
    int64_t mine = 0;
    if (b < a.requests) mine = (attn_request<SEEN>(a, b).queries * a.group + ROWS - 1) / ROWS;
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
      mine = attn_span<SEEN, ROWS, FINE>(a, attn_request<SEEN>(a, lo), row0).units;
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

// A workgroup's item is 256 rows, 32 (two 16s) to each of eight waves. They decode a tile of 128 tokens together, an eighth
// each, into LDS as bfloat16 fragments of the two products (a kilobyte each, lane by lane, so that reading and writing them is
// free of bank conflicts), and each multiplies its own rows with all of it. While a tile is multiplied the next one is
// decoded into the other half of the LDS and the one behind it is on its way from memory; a tile costs one barrier.
// The products are those of the kernel for few rows: S^T = K Q^T leaves the weights where O^T += V^T P^T wants them. For chains in
// 4 bits the weights of bfloat16 queries are rounded to one bfloat16, an error of the size of the result's own rounding (2.3e-3 in
// all instead of 1.66e-3): in two parts the prompts below take 1.36 ms instead of 1.06, with 64 dimensions 1.00 instead of 0.79.
// For all else they have two parts as in the kernel for few rows, and both kernels are as near to the definition (1.66e-3): the
// trees below take 275 us so and 226 in one part, the answers 91 and 76, two prompts of 8,192 in 8 bits 1.48 ms and 1.17.
// Bound by what the vector units and the matrix cores have to issue: for 64 tokens a wave has 64 products, of which each keeps
// the vector units from about 9 of its 16 cycles (measured with one wave of each kind on a SIMD), and some 200 vector
// instructions, two thirds of them the softmax. Two prompts of 8,192 tokens, 32 query and 8 key heads of 128, bfloat16: 1.06
// ms, 1,004 TFLOP/s; a library's product of 8,192^3 reaches 1,206 here. Measured on the way, same case: 64 rows and every wave
// its own tokens 2.24 ms; 128 rows and four waves, tiles of 64 decoded once, 1.63; reading ahead in LDS, 1.56; addresses held
// by lanes and items weighted, 1.37; no maximum from tile to tile, 1.23; 256 rows and tiles of 128, 1.08 (64 dimensions 0.94
// to 0.82); what follows for large scores in the same loop but out of the way, 1.06 (0.78). Products and softmaxes ordered by hand to
// run beside each other lost (1.71 against 1.56), priorities for the products brought nothing; products on the 4-bit keys
// themselves would need the queries in 8 bits, and lose bits of sums whose terms differ by much (2^-14 of the terms' sizes,
// measured).
// At 256 dimensions 32 rows leave room for one wave on a SIMD only: eight waves of 16 rows and tiles of 64 tokens, as the LDS
// has room for. They read it twice as often but wait less: two prompts of 4,096 tokens, other sizes as above, 0.80 ms (0.76
// now, 710 TFLOP/s) against 1.02 with four waves of 32 rows and tiles of 32 tokens and 0.95 with eight and 32; chunks of 17 to
// 2,000 tokens behind a window 87 us against 95 and 92.
// Trees of 24 to 64 nodes, four heads to one of the cache's, behind 1,000 to 12,000 tokens, 40 requests: 275 us; what is lost there
// are waves without rows and the ends of items, 8 us each. 6 answers of 100 to 1,200 tokens over an encoder's 700 to 5,000
// states in 8 bits: 91 us, 58 of them in the tiles. At 128 dimensions bfloat16 spills 22 vector registers for trees and 4 to 6 for
// states and 8 bits (chains in 4 bits none), float16 28 to 67 (24); at 256 dimensions 11 to 27 (12), float16 34 to 70 (36); at 64 none.
template <int BITS, int DIM>
struct ManyShape {
  static constexpr int kTile = DIM == 256 ? 64 : 128;  // tokens
  static constexpr int kHalves = kTile / 16, kGroups = kTile / 32;
  static constexpr int kKeyFrags = DIM / 32, kValueFrags = DIM / 16;  // of 16 tokens; of 32 tokens
  static constexpr int kRows = many_rows(DIM), kWaves = 8, kThreads = kWave * kWaves;
  static constexpr int NT = kRows / 16 / kWaves;                         // 16 rows each of a wave
  static constexpr int kKeyShare = kHalves * kKeyFrags / kWaves;         // fragments: a wave's share of the keys
  static constexpr int kWords = BITS / 4;                                // of a fragment, a lane
};

// A wave's share of a tile, as it comes from memory: keys of 16 tokens (at 256 dimensions half of each lane's quarter), values
// of 32 tokens.
template <int BITS, int DIM>
struct RawTile {
  uint32_t key[ManyShape<BITS, DIM>::kKeyShare * ManyShape<BITS, DIM>::kWords];
  uint32_t key_scale;
  uint32_t value[8];
  uint32_t value_scale[2];
};

template <int BITS, int DIM>
struct ManyStage {
  u32x4 key[ManyShape<BITS, DIM>::kHalves][ManyShape<BITS, DIM>::kKeyFrags][kWave];
  u32x4 value[ManyShape<BITS, DIM>::kGroups][ManyShape<BITS, DIM>::kValueFrags][kWave];
};

template <typename T, int BITS, int SEEN, int DIM>
__global__ __launch_bounds__((ManyShape<BITS, DIM>::kThreads), 2) void page_attention_many_kernel(
    AttnArgs a, const AttnItem *items, const int32_t *item_count, float *parts, float *part_stats, JoinRecord *records) {
  using Shape = ManyShape<BITS, DIM>;
  constexpr int kThreads = Shape::kThreads;
  constexpr int kRows = Shape::kRows, NT = Shape::NT, kSteps = DIM / 32, kTile = Shape::kTile, kHalves = Shape::kHalves;
  constexpr int kParts = std::is_same<T, _Float16>::value ? 2 : 1;
  constexpr int kSub = kUnit / kTile;  // tiles of a unit
  constexpr bool kOther = BITS == 8 || SEEN != SHMT_SEEN_CAUSAL;  // than chains in 4 bits
  constexpr int kWeightParts = kOther ? 2 : kParts;
  __shared__ ManyStage<BITS, DIM> stage[2];
  __shared__ Found found;
  __shared__ uint64_t scan[Shape::kWaves];
  __shared__ int64_t row_range[2];  // rows of any request
  __shared__ int32_t first_item[kThreads];
  __shared__ int again_at[2], far_any, wild_any;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n_lane = lane & 15, g = lane >> 4;
  // The units of one head, and, later, the item that holds a given one of them: from the list of items, or, without one (not
  // more than 256 requests, few items), by counting.
  int64_t per_head, count;
  if (items) {
    count = same(*item_count), per_head = same(items[count].unit);
    const Request r0 = attn_request<SEEN>(a, 0), r1 = attn_request<SEEN>(a, a.requests - 1);
    attn_clear_rows<T, DIM>(a, r0.first_row, r1.first_row + r1.queries);
  } else {
    if (threadIdx.x == 0) row_range[0] = row_range[1] = a.tokens;
    __syncthreads();
    Request r{};
    if (threadIdx.x < a.requests) {
      r = attn_request<SEEN>(a, threadIdx.x);
      if (threadIdx.x == 0) row_range[0] = r.first_row;
      if (threadIdx.x == a.requests - 1) row_range[1] = r.first_row + r.queries;
    }
    const uint64_t mine = (r.queries * a.group + kRows - 1) / kRows;
    uint64_t all;
    const uint64_t at = block_exclusive_scan<uint64_t, kThreads>(mine, scan, &all);
    first_item[threadIdx.x] = static_cast<int32_t>(at);
    count = same(static_cast<int64_t>(all));
    __syncthreads();
    attn_clear_rows<T, DIM>(a, row_range[0], row_range[1]);
    per_head = 0;
  }
  // Item i of a head, without the list.
  auto item_of = [&](int64_t i, Request *r, int *row0) {
    int lo = 0, hi = static_cast<int>(a.requests) - 1;  // the last request whose first item is i or before it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_item[mid] <= i) lo = mid; else hi = mid - 1;
    }
    *r = attn_request<SEEN>(a, lo);
    *row0 = static_cast<int>(i - first_item[lo]) * kRows;
    return lo;
  };
  // Of the last kThreads items, or fewer, which mostly are all: the thread's own, and the units in front of it.
  Found own{};
  uint64_t own_units = 0;
  if (!items)
    for (int64_t base = 0; base < count; base += kThreads) {
      uint64_t all;
      own_units = 0;
      if (base + threadIdx.x < count) {
        int r0;
        own.request = item_of(base + threadIdx.x, &own.req, &r0);
        own.units = r0;
        own_units = attn_span<SEEN, kRows, kOther>(a, own.req, r0).units;
      }
      own.before = per_head + static_cast<int64_t>(block_exclusive_scan<uint64_t, kThreads>(own_units, scan, &all));
      per_head += same(static_cast<int64_t>(all));
    }
  const int64_t U = per_head * a.v.kv_heads;
  // With a unit for everyone, neighbours in the numbering of units are on one XCD: they read the same pages.
  const int64_t G = min(int64_t{gridDim.x}, kOther && !a.alone ? U / kFineUnits : U);
  const int64_t wg = G == gridDim.x && G % 8 == 0 ? (blockIdx.x & 7) * (G / 8) + (blockIdx.x >> 3) : blockIdx.x;
  if (threadIdx.x == 0) records[wg].first = -1;
  if (wg >= G) return;
  const Shares shares(U, G);
  const int64_t u_begin = shares.begin(wg), u_end = shares.begin(wg + 1);
  int head = same(static_cast<int>(divide(u_begin, per_head)));
  const int64_t x = u_begin - head * per_head;  // within one head's units
  int64_t b, u_item;                            // the item's request and first unit
  int row0;
  Request req;
  if (items) {
    int64_t item = 0, width = count;  // the item is among [item, item + width)
    while (width > 1) {
      const int64_t step = (width + kThreads - 1) / kThreads;
      const int64_t i = item + threadIdx.x * step, end = min(i + step, item + width);
      if (i < item + width && items[i].unit <= x && x < items[end].unit) found.before = i, found.units = end - i;
      __syncthreads();
      item = same(found.before), width = same(found.units);
      __syncthreads();
    }
    const AttnItem it = items[item];
    b = same(it.request), row0 = same(it.row0), u_item = head * per_head + same(it.unit);
    req = same(attn_request<SEEN>(a, b));
  } else {
    if (own.before <= x && x < own.before + static_cast<int64_t>(own_units)) found = own;
    int64_t before = 0;
    for (int64_t base = 0; base + kThreads < count; base += kThreads) {
      uint64_t mine = 0, all;
      Request r{};
      int r0 = 0, lo = 0;
      lo = item_of(base + threadIdx.x, &r, &r0);
      mine = attn_span<SEEN, kRows, kOther>(a, r, r0).units;
      const int64_t at = before + static_cast<int64_t>(block_exclusive_scan<uint64_t, kThreads>(mine, scan, &all));
      if (at <= x && x < at + static_cast<int64_t>(mine)) found = Found{r, lo, at, r0};
      before += same(static_cast<int64_t>(all));
      if (x < before) break;
    }
    __syncthreads();
    b = same(found.request), row0 = same(static_cast<int>(found.units)), u_item = head * per_head + same(found.before);
    req = same(found.req);
  }

  const uint32_t flip = a.scale < 0 ? 0x80008000u : 0u;
  const int page = 1 << a.v.log2_page;
  // a wave's share of the decoding
  const int key_half = DIM == 256 ? wave >> 1 : wave, key_frag0 = DIM == 256 ? 4 * (wave & 1) : 0;
  const int value_group = DIM == 256 ? wave >> 2 : wave >> 1, value_word = DIM == 256 ? wave >> 1 & 1 : 0;
  const uint32_t key_at = n_lane * (DIM * BITS / 8) + g * (DIM * BITS / 32) + key_frag0 * BITS;
  const uint32_t key_scale_at = (DIM == 64 ? g >> 1 : g * (DIM / 128) + key_frag0 / 4) * page + n_lane;
  // Of the sixteenth of a value that a lane has, waves take different dimensions: in 4 bits the even and odd waves halves of one
  // word, in 8 bits words of their own (64 dimensions: halves).
  const int value_dim0 = DIM == 64 ? 2 * (wave & 1) : 8 * value_word + 4 * (wave & 1);
  const uint32_t value_at =
      (page + 4 * g) * (DIM * BITS / 8) + n_lane * (DIM * BITS / 128) + (BITS == 8 ? value_dim0 : value_word * 4);
  const uint32_t value_scale_at = (DIM / 32 + n_lane * (DIM / 16) / 32) * page + 4 * g;

  auto next_item = [&] {
    row0 += kRows;
    if (row0 >= req.queries * a.group) {
      row0 = 0;
      do {
        if (++b == a.requests) b = 0, ++head;
        req = same(attn_request<SEEN>(a, b));
      } while (req.queries == 0);
    }
  };
  int64_t u = u_begin;
  if constexpr (kOther) {  // of what others have begun, units without tokens may be left, and are nobody's part
    const Span span = same(attn_span<SEEN, kRows, kOther>(a, req, row0));
    if (u - u_item > (span.tiles - 1) * int64_t{span.weight}) {
      u = u_item += span.units;
      if (u >= u_end) return;
      next_item();
    }
  }
  while (u < u_end) {
    const Span span = same(attn_span<SEEN, kRows, kOther>(a, req, row0));
    const int rows = min(kRows, req.queries * a.group - row0);
    u32x4 q[kParts][NT][kSteps];
    int see_last[NT], see_after[NT], see_number[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 16 * (wave * NT + n) + n_lane;
      const int row = row0 + min(r, rows - 1), token = row_token(a, row);
      const int h = head * a.group + row - token * a.group;
      const Sees sees = row_sees<SEEN>(a, req, token, r < rows);
      see_last[n] = sees.last, see_after[n] = sees.after, see_number[n] = sees.number;
      const T *src = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head +
                     g * (DIM / 4);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) query_fragment<T>(src + 8 * i, r < rows, flip, q[0][n][i], q[kParts - 1][n][i]);
    }
    const int sinks = a.window > 0 ? a.sinks : 0;
    // Waves without a row only decode: of up to 128 rows the first four multiply, one on each SIMD. (16 rows to a wave in turn, so
    // that the SIMDs share what there is, brought 8 % for 160 and 192 rows of bfloat16 and lost 5 to 9 % for 128 and 256,
    // with weights in one part; chains in 4 bits lose 2 % by the question itself, two prompts 1,071 us instead of 1,050.)
    const bool has_rows = !kOther || 16 * wave * NT < rows;
    // the first and the last place of the wave's rows, and of the item's
    const int r_first = min(16 * wave * NT, rows - 1), r_last = min(16 * (wave + 1) * NT - 1, rows - 1);
    auto place = [&](int r) { return place_of<SEEN>(req, row_token(a, row0 + r)); };
    auto after = [&](int r) { return a.window > 0 ? max(place(r), -1) - a.window : -1; };
    const int wave_first = same(seen_by_all<SEEN>(a, req, row_token(a, row0 + r_first))), wave_after = same(after(r_last));
    const int item_first = same(seen_by_all<SEEN>(a, req, row_token(a, row0))), item_after = same(after(rows - 1));
    const int32_t *table = a.table + b * a.table_stride;
    const bool alone = kOther && a.alone;
    // A tile is the workgroup's that its first unit belongs to.
    auto tiles_before = [&](int64_t units) {
      const int n = same(static_cast<int>(units));
      return kOther ? min((n + span.weight - 1) / span.weight, span.tiles) : n;
    };
    const int first = alone ? 0 : tiles_before(u - u_item) * kSub;
    const int last = (alone ? span.tiles : tiles_before(min(u_item + span.units, u_end) - u_item)) * kSub;

    auto token_of = [&](int t) { return unit_token(span, t / kSub) + t % kSub * kTile; };  // of the item's tile t
    // Where the next tiles' tokens lie, 16 tokens a lane, and of which of them any row sees any.
    constexpr int kAhead = kWave / kHalves;
    Place16 places;
    uint64_t present = 0;
    int page_base = 0;
    auto look_up = [&](int t0) {
      page_base = t0;
      const int t = t0 + lane / kHalves, j = token_of(t) + lane % kHalves * 16;
      const int p = t < last ? page_at(a, table, span, j) : -1;
      places = place16<BITS, DIM>(a.v, head, max(p, 0), j);  // what is not there is loaded from page 0 and not looked at
      present = __ballot(p >= 0);
    };
    auto present_of = [&](int t) {
      return static_cast<uint32_t>(present >> ((t - page_base) * kHalves)) & ((1u << kHalves) - 1);
    };
    // The next tile from t on of which any row sees something; `last` if there is none.
    auto find = [&](int t) {
      for (; t < last; ++t) {
        if (t - page_base >= kAhead) look_up(t);
        if (present_of(t)) break;
      }
      return t;
    };
    struct Step {
      int token0;
      uint32_t there;  // a bit for each 16 tokens
      bool whole;      // all rows of the item see all of it
    };
    RawTile<BITS, DIM> raw;
    auto sees_all = [&](int token0, uint32_t there, int pos_first, int after_last) {
      return there == (1u << kHalves) - 1 && token0 + kTile - 1 <= pos_first &&
             (token0 > after_last || token0 + kTile <= sinks);
    };
    auto fetch = [&](int t) {
      Step s;
      s.token0 = token_of(t);
      s.there = present_of(t);
      s.whole = sees_all(s.token0, s.there, item_first, item_after);
      const int at = (t - page_base) * kHalves;
      {
        const Place16 x = places.of_lane(at + key_half);
        load_words<Shape::kKeyShare * Shape::kWords>(x.row() + key_at, raw.key);
        raw.key_scale = x.scale()[key_scale_at];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Place16 x = places.of_lane(at + 2 * value_group + half);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint8_t *y = x.row() + value_at + r * (DIM * BITS / 8);
          load_words<DIM == 64 ? 0 : 1>(y, &raw.value[4 * half + r]);
        }
        raw.value_scale[half] = *reinterpret_cast<const uint32_t *>(x.scale() + value_scale_at);
      }
      return s;
    };
    // A wave's share of the fragments of the tile in `raw`.
    auto decode = [&](const Step &s, ManyStage<BITS, DIM> &to) {
      const float fk = scale_operand(raw.key_scale);
#pragma unroll
      for (int i = 0; i < Shape::kKeyShare; ++i)
        to.key[key_half][key_frag0 + i][lane] = decode_fragment<BITS>(&raw.key[i * Shape::kWords], fk);
      if (!s.whole) {
        // Values that are not finite in bfloat16 must not meet the weight 0 of a row that does not see them: they are left
        // out here and added at the end of the item.
        bool wild = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((raw.value_scale[j / 4] >> (8 * (j % 4)) & 255u) >= kWild<BITS>) {
            const int half = 2 * value_group + j / 4, token = s.token0 + 16 * half + 4 * g + j % 4;
            raw.value_scale[j / 4] &= ~(255u << (8 * (j % 4)));
            wild |= (s.there >> half & 1) && token < span.end && (token >= span.begin || token < span.sink_end);
          }
        if (wild) wild_any = 1;
        if constexpr (BITS == 8) {  // two codes of 8 bits are not numbers: where nobody looks they may stand, and must not meet a 0
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int half = 2 * value_group + j / 4, token = s.token0 + 16 * half + 4 * g + j % 4;
            const bool seen = (s.there >> half & 1) && token < span.end && (token >= span.begin || token < span.sink_end);
            raw.value[j] = seen ? raw.value[j] : 0;
          }
        }
      }
      // The conversion reads nothing of a scale but its exponent field, so the byte need not be cut out.
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = __uint_as_float(j % 4 == 3 ? raw.value_scale[j / 4] >> 1 : raw.value_scale[j / 4] << (23 - 8 * (j % 4)));
      auto two = [&](auto pair, int frag) {  // dimensions 2 I and 2 I + 1 of a lane's word
        constexpr int I = decltype(pair)::value;
        uint32_t x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = decode_two<BITS, I>(raw.value[j], f[j]);
        u32x4 lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
          hi[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
        }
        to.value[value_group][frag][lane] = lo;
        to.value[value_group][frag + 1][lane] = hi;
      };
      if constexpr (BITS == 4) {  // bytes 0, 1 or 2, 3 of the words (at 64 dimensions byte 0 or 1)
#pragma unroll
        for (int j = 0; j < 8; ++j) raw.value[j] >>= (DIM == 64 ? 8 : 16) * (wave & 1);
      }
      two(std::integral_constant<int, 0>{}, value_dim0);
      if constexpr (DIM > 64) two(std::integral_constant<int, 1>{}, value_dim0 + 2);
    };

    RowState<DIM, NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n)  // no row waits for nothing
      st.top[n] = 16 * (wave * NT + n) + n_lane < rows ? kNothing : 0;
    bool waiting = true;
    // A wave's rows and the tile in `from`, in pass `pass` (see kFirst), which takes scores in units of `unit` powers of two.
    // `again` is set if the item has to be begun again, far_any if with rounded scores.
    auto multiply = [&](const Step &s, const ManyStage<BITS, DIM> &from, int pass, float unit, int &again) {
      const bool whole = sees_all(s.token0, s.there, wave_first, wave_after);
      // All fragments of a product are on their way from LDS before it begins: those of the values under the softmax, those
      // of the next keys under the values' product. Reads of LDS keep their place at the fences, all else may move.
      auto fence = [] { __builtin_amdgcn_sched_barrier(0x67f); };
      u32x4 keys[kSteps][2], values[Shape::kValueFrags];
      auto read_keys = [&](int group) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) keys[i][half] = from.key[2 * group + half][i][lane];
        fence();
      };
      read_keys(0);
#pragma unroll
      for (int group = 0; group < Shape::kGroups; ++group) {
        f32x4 x[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int p = 0; p < kParts; ++p) x[n][half] = mfma(keys[i][half], q[p][n][i], x[n][half]);
#pragma unroll
        for (int i = 0; i < Shape::kValueFrags; ++i) values[i] = from.value[group][i][lane];
        fence();
        if (!whole) {
          const int token_0 = s.token0 + 32 * group;
          if (SEEN == SHMT_SEEN_TREE && token_0 + 32 > req.before) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int half = 2 * group + j / 4, token = token_0 + 16 * (j / 4) + 4 * g + j % 4;
              int4 node = make_int4(0, 0, 0, 0);  // nobody is below it
              if (token >= req.before && token < span.end) node = a.nodes[req.first_row + (token - req.before)];
              const int at = req.before + node.z;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const bool old = token <= see_last[n] && (token > see_after[n] || token < sinks);
                const bool own = is_above(node, see_number[n]) && (at > see_after[n] || at < sinks);
                x[n][j / 4][j % 4] = (s.there >> half & 1) && (old || own) ? x[n][j / 4][j % 4] : kNothing;
              }
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int half = 2 * group + j / 4, token = token_0 + 16 * (j / 4) + 4 * g + j % 4;
                const bool sees = (s.there >> half & 1) && token <= see_last[n] && (token > see_after[n] || token < sinks);
                x[n][j / 4][j % 4] = sees ? x[n][j / 4][j % 4] : kNothing;
              }
          }
        }
        if (__builtin_expect(waiting, 0)) {  // in the last passes always
          if (pass < kMaximum) waiting = first_reference<NT>(x, unit, st, again, far_any);
          else round_scores<NT>(x, powers_of_two(a), st, pass);
        }
        u32x4 w[kWeightParts][NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) weights<kWeightParts>(x[n], unit, st.top[n], st.sum[n], w, n);
        raise_reference<NT>(st, again, far_any);
        if (group + 1 < Shape::kGroups) read_keys(group + 1);
#pragma unroll
        for (int i = 0; i < Shape::kValueFrags; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int p = 0; p < kWeightParts; ++p) st.acc[n][i] = mfma(values[i], w[p][n], st.acc[n][i]);
      }
    };

    if (threadIdx.x == 0) again_at[0] = again_at[1] = far_any = wild_any = 0;
    // The passes share one loop: with a second one for the last two, registers of the first were spilled (1.17 ms instead of
    // 1.08 for the two prompts).
    for (int pass = kFirst;;) {
      const float unit = pass < kMaximum ? powers_of_two(a) : 1.0f;
      bool again = false;
      waiting |= pass >= kMaximum;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (pass == kMaximum) st.top[n] = kNothing;
        st.sum[n] = 0;
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i) st.acc[n][i] = f32x4{0, 0, 0, 0};
      }
      __syncthreads();  // flags cleared; nobody reads the stages
      look_up(first);
      int t = find(first);
      if (t >= last) break;
      Step now = fetch(t);
      decode(now, stage[0]);
      t = find(t + 1);
      bool more = t < last;
      Step next = fetch(more ? t : page_base);
      __syncthreads();
      for (int k = 0;; ++k) {
        // Behind the last tile some tile is decoded once more, where nobody reads it.
        decode(next, stage[~k & 1]);
        const int t_then = more ? find(t + 1) : last;
        const Step then = fetch(t_then < last ? t_then : page_base);
        if (has_rows) multiply(now, stage[k & 1], pass, unit, again_at[k & 1]);
        __syncthreads();
        // This word is written again two tiles on only, behind the next barrier: all waves read the same.
        again = pass < kMaximum && again_at[k & 1] != 0;
        if (!more || again) break;
        now = next, next = then, t = t_then;
        more = t < last;
      }
      if (pass < kMaximum ? !again : pass == kRounded) break;
      __syncthreads();  // all have read again_at
      if (threadIdx.x == 0) again_at[0] = again_at[1] = 0;
      pass = pass == kFirst && same(far_any) == 0 ? kRaised : std::max<int>(pass + 1, kMaximum);
    }
    u = kOther ? min(u_item + span.units, u_end) : u_item + last / kSub;

    // Each wave's rows into the result or into a part.
    const bool begins = u_item >= u_begin, ends = alone || last >= (kOther ? span.tiles : span.units) * kSub;
    const int64_t slot = 2 * wg + (begins ? 1 : 0);
    const bool add_wild = same(wild_any) != 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 16 * (wave * NT + n) + n_lane;
      const float total = across_sum(st.sum[n]);
      if (r >= rows) continue;
      const int row = row0 + r, token = row_token(a, row), h = head * a.group + row - token * a.group;
      const int64_t line = (req.first_row + token) * a.heads + h;
      const float base = fmaxf(st.top[n], kLowest), inv = total == 0 ? 0 : 1 / total;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int d0 = (4 * g + r4) * (DIM / 16);
        f32x4 o[DIM / 64];
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i) o[i / 4][i % 4] = st.acc[n][i][r4];
        if (add_wild) {
          const Sees sees = row_sees<SEEN>(a, req, token, true);
          const T *q_row = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head;
#pragma unroll 1
          for (int t = first; t < last; ++t) {
            uint32_t there = 0;
            for (int half = 0; half < kHalves; ++half)
              there |= (page_at(a, table, span, token_of(t) + 16 * half) >= 0 ? 1u : 0u) << half;
            if (sees_all(token_of(t), there, item_first, item_after)) continue;
#pragma unroll 1
            for (int half = 0; half < kHalves; ++half) {
              const int j0 = token_of(t) + 16 * half;
              add_left_out<T, BITS, SEEN, DIM>(a, head, page_at(a, table, span, j0), j0, q_row, req, sees, powers_of_two(a), base,
                                               d0, o);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < DIM / 64; ++i) {
          if (begins && ends) {
            typedef T out_vec __attribute__((ext_vector_type(4)));
            *reinterpret_cast<out_vec *>(static_cast<T *>(a.out) + line * DIM + d0 + 4 * i) =
                out_vec{static_cast<T>(o[i][0] * inv), static_cast<T>(o[i][1] * inv), static_cast<T>(o[i][2] * inv),
                        static_cast<T>(o[i][3] * inv)};
          } else {
            *reinterpret_cast<f32x4 *>(parts + part_at<DIM, kRows>(slot * kRows + r, (4 * g + r4) * (DIM / 64) + i)) = o[i];
          }
        }
      }
      if (g == 0) {
        if (begins && ends) {
          if (a.lse) a.lse[line] = total == 0 ? kNothing : (st.top[n] + __builtin_log2f(total)) * 0.69314718055994530942f;
        } else {
          part_stats[(slot * kRows + r) * 2] = st.top[n];
          part_stats[(slot * kRows + r) * 2 + 1] = total;
        }
      }
    }
    __syncthreads();  // wild_any has been read
    if (!begins && ends && threadIdx.x == 0) {
      records[wg] = JoinRecord{static_cast<int32_t>(shares.owner(u_item)), head, rows, row0, req.first_row};
    }
    if (u >= u_end) break;
    // the next item
    u_item = u;
    next_item();
  }
}

template <typename T, int BITS, int SEEN, int DIM>
void launch_many(const AttnArgs &a, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  // A list of items costs a launch; every workgroup counts for itself where that takes no longer, or there is nothing to count.
  const AttnItem *items = nullptr;
  if (a.requests > 256 || (a.requests > 0 && s.room > 1024)) {
    hipLaunchKernelGGL((page_attention_items_kernel<SEEN, many_rows(DIM), BITS == 8 || SEEN != SHMT_SEEN_CAUSAL>), dim3(1),
                       dim3(1024), 0, stream, a, s.first_item, s.items, s.room, s.count);
    items = s.items;
  }
  hipLaunchKernelGGL((page_attention_many_kernel<T, BITS, SEEN, DIM>), dim3(groups), dim3(ManyShape<BITS, DIM>::kThreads), 0,
                     stream, a, items, s.count, s.parts, s.stats, s.records);
  if (a.alone) return;
  hipLaunchKernelGGL((page_attention_join_kernel<T, DIM, many_rows(DIM)>), dim3(2048), dim3(256), 0, stream, a,
                     s.parts, s.stats, s.records, static_cast<int>(groups));
}

template <typename T, int BITS, int SEEN>
void launch_many(const AttnArgs &a, int dim, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  if (dim == 64) launch_many<T, BITS, SEEN, 64>(a, groups, s, stream);
  else if (dim == 128) launch_many<T, BITS, SEEN, 128>(a, groups, s, stream);
  else launch_many<T, BITS, SEEN, 256>(a, groups, s, stream);
}

template <int BITS, int SEEN>
void launch_attention_many(const AttnArgs &a, int dim, int elem_type, unsigned groups, const AttnScratch &s,
                           hipStream_t stream) {
  if (elem_type == SHMT_F16) launch_many<_Float16, BITS, SEEN>(a, dim, groups, s, stream);
  else launch_many<__bf16, BITS, SEEN>(a, dim, groups, s, stream);
}

}  // namespace shmt
