// Attention over the paged key/value cache: the kernel for few rows a request (decode, a few speculated tokens, small trees), in
// which the waves of a workgroup share the tokens. Of a cache in 4 bits, where nothing else is said:
//
// The work: every token that a request holds is read once for each of its heads, dim bytes and dim / 16 scale bytes, and a
// decode step is bound by that. A wave takes 32 tokens a step, 2,176 or 4,352 bytes at 64 or 128 dimensions, while the next 32
// are on their way; three waves a SIMD keep 52 KB of a compute unit's share of HBM in flight. Units of 128 tokens are dealt out
// evenly (paged_attention.h), so a batch of ragged requests, one long request and anything between are one case. Measured, 32
// requests of 8,000 tokens, 8 heads of 128, bfloat16: 57 us, 4.9 TB/s, what a copy reaches; 64 ragged requests of 1,000 to
// 16,000 tokens 85 us, 4.4 TB/s; one request of 130,000 tokens with float16 queries 46 us, 3.1 TB/s, of which the join 7 us.
// At 64 dimensions half the bytes come with the same softmax, and the vector units are what it waits for: 96 requests with a
// window of 4,000 tokens, float16, 66 us, 3.1 TB/s (some 230 vector instructions for 32 tokens of a wave).
// In 8 bits twice the bytes come with the same softmax: 64 ragged requests as above 143 us, 5.2 TB/s. More
// than 32 rows read the cache once for each 32: a tree of 65 rows behind 100,000 tokens in 8 bits, float16, 120 us, in which 651 MB
// come from HBM (counted; the cache has 211), 6.0 TB/s, with vector units at 46 % and matrix cores at 30 % of the time. Over an encoder's states, 80 requests of 300 to 1,500, 5 rows each, 16 heads of 64, 37 us, of which the join 5.
#pragma once
#include "paged_attention.h"

namespace shmt {

// What the waves of a workgroup exchange at the end of an item.
template <int DIM>
struct JoinShared {
  static constexpr int kStride = DIM + 4;  // rows shifted against each other over the banks
  alignas(16) float acc[4][16 * kStride];
  float top[4][16], sum[4][16];
};

template <typename T, int BITS, int SEEN, int DIM, int NT>
__global__ __launch_bounds__(256, (attn_waves(BITS, SEEN, std::is_same<T, _Float16>::value, DIM, NT))) void page_attention_kernel(
    AttnArgs a, float *parts, float *part_stats, JoinRecord *records) {
  constexpr int kRows = 16 * NT;
  constexpr int kParts = std::is_same<T, _Float16>::value ? 2 : 1;
  constexpr bool kOther = BITS == 8 || SEEN != SHMT_SEEN_CAUSAL;  // than chains in 4 bits
  using Q = Queries<DIM, NT, kParts>;
  union Shared {
    JoinShared<DIM> join;
    u32x4 queries[Q::kShared ? Q::kFrags * kWave : 1];
    uint64_t scan[4];
  };
  __shared__ Shared shared;
  __shared__ Found found;
  __shared__ int64_t row_range[2];  // rows of any request
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n_lane = lane & 15, g = lane >> 4;
  const int kv_heads = a.v.kv_heads;

  // Where this workgroup's units begin: each thread counts a run of requests.
  const int64_t each = (a.requests + 255) / 256, b_lo = min(threadIdx.x * each, a.requests), b_hi = min(b_lo + each, a.requests);
  int64_t mine = 0;
  if (threadIdx.x == 0) row_range[0] = row_range[1] = a.requests > 0 ? 0 : a.tokens;
  __syncthreads();
  for (int64_t i = b_lo; i < b_hi; ++i) {
    const Request r = attn_request<SEEN>(a, i);
    mine += attn_units<SEEN, kRows>(a, r) * kv_heads;
    if (i == 0) row_range[0] = r.first_row;
    if (i == a.requests - 1) row_range[1] = r.first_row + r.queries;
  }
  uint64_t total;
  const int64_t at =
      static_cast<int64_t>(block_exclusive_scan<uint64_t, 256>(static_cast<uint64_t>(mine), shared.scan, &total));
  const int64_t U = same(static_cast<int64_t>(total));
  attn_clear_rows<T, DIM>(a, row_range[0], row_range[1]);
  // With a unit for everyone, neighbours in the numbering of units are on one XCD: they read the same lines of scales and
  // of the table. With fewer units than workgroups each has one, on all XCDs.
  const int64_t G = min(int64_t{gridDim.x}, U);
  const int64_t wg = G == gridDim.x && G % 8 == 0 ? (blockIdx.x & 7) * (G / 8) + (blockIdx.x >> 3) : blockIdx.x;
  if (threadIdx.x == 0) records[wg].first = -1;
  if (wg >= G) return;
  const Shares shares(U, G);
  const int64_t u_begin = shares.begin(wg), u_end = shares.begin(wg + 1);
  if (at <= u_begin && u_begin < at + mine) {
    int64_t before = at;
    for (int64_t i = b_lo;; ++i) {
      const Request r = attn_request<SEEN>(a, i);
      const int64_t n = attn_units<SEEN, kRows>(a, r);
      if (u_begin < before + n * kv_heads) {
        found = Found{r, i, before, n};
        break;
      }
      before += n * kv_heads;
    }
  }
  __syncthreads();
  int64_t b = same(found.request), u_item = same(found.before);  // the item's first unit
  int row0 = 0;
  Request req = same(found.req);
  const int64_t per_head = same(found.units);
  int head = same(static_cast<int>(divide(u_begin - u_item, per_head)));
  u_item += head * per_head;
  Span span = same(attn_span<SEEN, kRows>(a, req, 0));
  while (u_item + span.units <= u_begin) {
    u_item += span.units;
    row0 += kRows;
    span = same(attn_span<SEEN, kRows>(a, req, row0));
  }

  const float scale2 = powers_of_two(a);
  const uint32_t flip = a.scale < 0 ? 0x80008000u : 0u;
  const LaneOffsets offsets = lane_offsets<BITS, DIM>(lane, 1 << a.v.log2_page);
  auto next_item = [&] {
    row0 += kRows;
    if (row0 >= req.queries * a.group) {
      row0 = 0;
      if (++head == kv_heads) {
        head = 0;
        do req = same(attn_request<SEEN>(a, ++b)); while (req.queries == 0);
      }
    }
    span = same(attn_span<SEEN, kRows>(a, req, row0));
  };
  int64_t u = u_begin;
  // Of what others have begun, units without tokens may be left, and are nobody's part. (Chains in 4 bits make it one.)
  if (kOther && u - u_item >= span.tiles) {
    u = u_item += span.units;
    if (u >= u_end) return;
    next_item();
  }
  while (u < u_end) {
    const int rows = min(kRows, req.queries * a.group - row0);
    Sight<NT> sight;
    sight.sinks = a.window > 0 ? a.sinks : 0;
    sight.begin = span.begin, sight.end = span.end, sight.sink_end = span.sink_end;
    sight.fresh = req.before;
    if constexpr (SEEN == SHMT_SEEN_TREE) sight.node = a.nodes + (req.first_row - req.before);
    // All rows see a whole tile that ends at or before the first row's place and begins in the last row's window.
    const int pos_first = same(seen_by_all<SEEN>(a, req, row_token(a, row0)));
    const int after_last = same(a.window > 0 ? max(place_of<SEEN>(req, row_token(a, row0 + rows - 1)), -1) - a.window : -1);
    const int32_t *table = a.table + b * a.table_stride;
    const bool alone = kOther && a.alone;
    const int first = alone ? 0 : same(static_cast<int>(u - u_item));
    const int last = alone ? span.tiles : same(static_cast<int>(min(u_item + span.units, u_end) - u_item));
    auto token_of = [&](int k) { return unit_token(span, k) + wave * kWaveTokens; };  // unit k's first token of this wave
    // Whether all rows see all of a wave's 32 tokens from token0 on, of which `there` are present.
    auto tile_whole = [&](int token0, uint32_t there) {
      return there == 3 && token0 + kWaveTokens - 1 <= pos_first &&
             (token0 > after_last || token0 + kWaveTokens <= sight.sinks);
    };
    // Where the next 32 units' tokens lie, 16 a lane, and of which of them any row sees any.
    Place16 places;
    uint64_t present = 0;
    int page_base = 0;
    auto look_up = [&](int k0) {
      page_base = k0;
      const int k = k0 + (lane >> 1), j = token_of(k) + 16 * (lane & 1);
      const int p = k < last ? page_at(a, table, span, j) : -1;
      places = place16<BITS, DIM>(a.v, head, max(p, 0), j);  // what is not there is loaded from page 0 and not looked at
      present = __ballot(p >= 0);
    };
    struct Step {
      int token0;
      uint32_t there;  // a bit for each 16 tokens
    };
    auto present_of = [&](int k) { return static_cast<uint32_t>(present >> (2 * (k - page_base))) & 3u; };
    // The next unit from k on that has anything for this wave; `last` if there is none.
    auto find = [&](int k) {
      for (; k < last; ++k) {
        if (k - page_base >= 32) look_up(k);
        if (present_of(k)) break;
      }
      return k;
    };
    // In 4 bits the next tile waits in registers of its own. In 8 those would be too many: the next keys are loaded into the place of
    // the present ones when these have been multiplied, the next values likewise, and two or three waves a SIMD have enough in flight.
    constexpr bool kInPlace = BITS == 8;
    KvTile<BITS, DIM> ahead;
    auto fetch_keys = [&](int k) {
      const int at = 2 * (k - page_base);
#pragma unroll
      for (int half = 0; half < 2; ++half) load_keys<BITS, DIM>(places.of_lane(at + half), 1 << a.v.log2_page, offsets, half, ahead);
    };
    auto fetch_values = [&](int k) {
      const int at = 2 * (k - page_base);
#pragma unroll
      for (int half = 0; half < 2; ++half) load_values<BITS, DIM>(places.of_lane(at + half), offsets, half, ahead);
    };
    auto fetch = [&](int k) {
      if constexpr (kInPlace) {
        fetch_keys(k);
        fetch_values(k);
      } else {
        const int at = 2 * (k - page_base);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const Place16 x = places.of_lane(at + half);
          load_keys<BITS, DIM>(x, 1 << a.v.log2_page, offsets, half, ahead);
          load_values<BITS, DIM>(x, offsets, half, ahead);
        }
      }
      return Step{token_of(k), present_of(k)};
    };
    // The first tile, which is on its way before the queries are. (Chains in 4 bits ask for their queries first: that is how they
    // were measured, and turned round they gain nothing.)
    int k_first = 0;
    Step step_first{};
    auto begin_tokens = [&] {
      look_up(first);
      k_first = find(first);
      if (k_first < last) step_first = fetch(k_first);
    };
    if constexpr (kOther) begin_tokens();
    Q q;
    q.shared = shared.queries;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 16 * n + n_lane;
      const uint32_t row = row0 + min(r, rows - 1);
      const uint32_t token = row / static_cast<uint32_t>(a.group);
      const int h = head * a.group + static_cast<int>(row - token * a.group);
      const Sees sees = row_sees<SEEN>(a, req, static_cast<int>(token), r < rows);
      sight.last[n] = sees.last, sight.after[n] = sees.after, sight.number[n] = sees.number;
      const T *src = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head +
                     g * (DIM / 4);
      constexpr int kSteps = DIM / 32;
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if (Q::kShared && ((n * kSteps + i) & 3) != wave) continue;  // the waves fill LDS together
        u32x4 y, z;
        query_fragment<T>(src + 8 * i, r < rows, flip, y, z);
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
    bool wild = false, waiting = true, far = false;
    RowState<DIM, NT> st;
#pragma unroll
    for (int n = 0; n < NT; ++n) st.top[n] = 16 * n + n_lane < rows ? kNothing : 0;  // what is not a row waits for nothing
    // A pass over the tokens (see kFirst); returns whether another has to follow. The last two are a loop of their own, which
    // costs the first ones no registers. Nothing in the loop changes the accumulators but the products, on every way through it:
    // only so do they stay in one place.
    auto go = [&](auto is_first, int pass) {
      constexpr bool kIsFirst = decltype(is_first)::value;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (!kIsFirst && pass == kMaximum) st.top[n] = kNothing;
        st.sum[n] = 0;
#pragma unroll
        for (int i = 0; i < DIM / 16; ++i) st.acc[n][i] = f32x4{0, 0, 0, 0};
      }
      if (!kOther || pass != kFirst) begin_tokens();
      int k = k_first;
      if (k >= last) return false;
      Step next = step_first;
      bool more, again = false;
      do {
        const Step now = next;
        const bool whole = tile_whole(now.token0, now.there);
        auto attend = [&](KvTile<BITS, DIM> &t, auto keys_done, auto values_done) {
          attend_tile<kIsFirst, BITS, SEEN, DIM, NT, kParts>(t, q, st, scale2, pass, lane, whole, now.token0, now.there & 1,
                                                             now.there & 2, sight, wild, waiting, again, far, keys_done,
                                                             values_done);
        };
        if constexpr (kInPlace) {
          k = find(k + 1);
          more = k < last;
          const int then = more ? k : page_base;  // behind the last tile some tile is loaded once more
          next = Step{token_of(then), present_of(then)};
          attend(ahead, [&] { fetch_keys(then); }, [&] { fetch_values(then); });
        } else {
          KvTile<BITS, DIM> t = ahead;
          k = find(k + 1);
          more = k < last;
          if (more) next = fetch(k);
          attend(t, [] {}, [] {});
        }
      } while (more && !again);
      return again;
    };
    bool again = true;
    for (int pass = kFirst; pass <= kRaised && again && !far; ++pass) again = go(std::true_type{}, pass);
    if (again)
      for (int pass = kMaximum; pass <= kRounded; ++pass) go(std::false_type{}, pass);
    u = u_item + (alone ? 1 : last);

    // The four waves' states, 16 rows at a time, into the result or into a part.
    const bool begins = u_item >= u_begin, ends = alone || last >= (kOther ? span.tiles : span.units);
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
            const Sees sees = row_sees<SEEN>(a, req, static_cast<int>(token), true);
            const T *q_row = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head;
            for (int k = first; k < last; ++k)
#pragma unroll 1
              for (int w = 0; w < kUnit / kWaveTokens; ++w) {
                const int t0 = unit_token(span, k) + w * kWaveTokens;
                const int p0 = page_at(a, table, span, t0), p1 = page_at(a, table, span, t0 + 16);
                if (tile_whole(t0, (p0 >= 0 ? 1u : 0u) | (p1 >= 0 ? 2u : 0u))) continue;
                add_left_out<T, BITS, SEEN, DIM>(a, head, p0, t0, q_row, req, sees, scale2, base, d0, o);
                add_left_out<T, BITS, SEEN, DIM>(a, head, p1, t0 + 16, q_row, req, sees, scale2, base, d0, o);
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
      records[wg] = JoinRecord{static_cast<int32_t>(shares.owner(u_item)), head, rows, row0, req.first_row};
    }
    if (u >= u_end) break;
    // the next item
    u_item = u;
    next_item();
  }
}

template <typename T, int BITS, int SEEN, int DIM, int NT>
void launch_few(const AttnArgs &a, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  hipLaunchKernelGGL((page_attention_kernel<T, BITS, SEEN, DIM, NT>), dim3(groups), dim3(256), 0, stream, a, s.parts, s.stats,
                     s.records);
  if (a.alone) return;
  // a workgroup of the join for each row, as far as 512 go
  const unsigned rows = static_cast<unsigned>(std::min<int64_t>(a.tokens * a.heads, 512));
  hipLaunchKernelGGL((page_attention_join_kernel<T, DIM, 16 * NT>), dim3(rows), dim3(256), 0, stream, a, s.parts, s.stats,
                     s.records, static_cast<int>(groups));
}

template <typename T, int BITS, int SEEN, int DIM>
void launch_few(const AttnArgs &a, int rows, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  if (rows == 16) launch_few<T, BITS, SEEN, DIM, 1>(a, groups, s, stream);
  else launch_few<T, BITS, SEEN, DIM, 2>(a, groups, s, stream);
}

template <typename T, int BITS, int SEEN>
void launch_few(const AttnArgs &a, int dim, int rows, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  if (dim == 64) launch_few<T, BITS, SEEN, 64>(a, rows, groups, s, stream);
  else if (dim == 128) launch_few<T, BITS, SEEN, 128>(a, rows, groups, s, stream);
  else launch_few<T, BITS, SEEN, 256>(a, rows, groups, s, stream);
}

template <int BITS, int SEEN>
void launch_attention_few(const AttnArgs &a, int dim, int elem_type, int rows, unsigned groups, const AttnScratch &s,
                          hipStream_t stream) {
  if (elem_type == SHMT_F16) launch_few<_Float16, BITS, SEEN>(a, dim, rows, groups, s, stream);
  else launch_few<__bf16, BITS, SEEN>(a, dim, rows, groups, s, stream);
}

}  // namespace shmt
