// Attention over the paged key/value cache held in 4 bits (shmt_page_attention): the kernel for few rows a request (decode,
// a few speculated tokens), in which the waves of a workgroup share the tokens, and the entry point.
//
// The work: every token that a request holds is read once for each of its heads, dim bytes and dim / 16 scale bytes, and a
// decode step is bound by that. A wave takes 32 tokens a step, 2,176 or 4,352 bytes at 64 or 128 dimensions, while the next 32
// are on their way; three waves a SIMD keep 52 KB of a compute unit's share of HBM in flight. Units of 128 tokens are dealt out
// evenly (paged_attention.h), so a batch of ragged requests, one long request and anything between are one case. Measured, 32
// requests of 8,000 tokens, 8 heads of 128, bfloat16: 57 us, 4.9 TB/s, what a copy reaches; 64 ragged requests of 1,000 to
// 16,000 tokens 85 us, 4.4 TB/s; one request of 130,000 tokens with float16 queries 46 us, 3.1 TB/s, of which the join 7 us.
// At 64 dimensions half the bytes come with the same softmax, and the vector units are what it waits for: 96 requests with a
// window of 4,000 tokens, float16, 66 us, 3.1 TB/s (some 230 vector instructions for 32 tokens of a wave).
#include "paged_attention.h"
#include "paged_host.h"

namespace shmt {

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
    AttnArgs a, float *parts, float *part_stats, JoinRecord *records) {
  constexpr int kRows = 16 * NT;
  constexpr int kParts = std::is_same<T, _Float16>::value ? 2 : 1;
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
    const Request r = attn_request(a, i);
    mine += attn_units<kRows>(a, r) * kv_heads;
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
      const Request r = attn_request(a, i);
      const int64_t n = attn_units<kRows>(a, r);
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
  Span span = same(attn_span<kRows>(a, req, 0));
  while (u_item + span.units <= u_begin) {
    u_item += span.units;
    row0 += kRows;
    span = same(attn_span<kRows>(a, req, row0));
  }

  const float scale2 = powers_of_two(a);
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
      const Sees sees = row_sees(a, pos);
      sight.last[n] = sees.last, sight.after[n] = sees.after;
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
    // All rows see a whole tile that ends at or before the first row's place and begins in the last row's window.
    const int pos_first = same(min(req.before + row_token(a, row0), a.limit - 1));
    const int after_last = same(a.window > 0 ? max(req.before + row_token(a, row0 + rows - 1), -1) - a.window : -1);
    const int32_t *table = a.table + b * a.table_stride;
    const int first = same(static_cast<int>(u - u_item));
    const int last = same(static_cast<int>(min(u_item + span.units, u_end) - u_item));
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
      places = place16<DIM>(a.v, head, max(p, 0), j);  // what is not there is loaded from page 0 and not looked at
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
    KvTile<DIM> ahead;
    auto fetch = [&](int k) {
      const int at = 2 * (k - page_base);
      load_half<DIM>(places.of_lane(at), 1 << a.v.log2_page, offsets, 0, ahead);
      load_half<DIM>(places.of_lane(at + 1), 1 << a.v.log2_page, offsets, 1, ahead);
      return Step{token_of(k), present_of(k)};
    };
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
      look_up(first);
      int k = find(first);
      if (k >= last) return false;
      Step next = fetch(k);
      bool more, again = false;
      do {
        const Step now = next;
        KvTile<DIM> t = ahead;
        k = find(k + 1);
        more = k < last;
        if (more) next = fetch(k);
        const bool whole = tile_whole(now.token0, now.there);
        attend_tile<kIsFirst, DIM, NT, kParts>(t, q, st, scale2, pass, lane, whole, now.token0, now.there & 1, now.there & 2,
                                               sight, wild, waiting, again, far);
      } while (more && !again);
      return again;
    };
    bool again = true;
    for (int pass = kFirst; pass <= kRaised && again && !far; ++pass) again = go(std::true_type{}, pass);
    if (again)
      for (int pass = kMaximum; pass <= kRounded; ++pass) go(std::false_type{}, pass);
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
            const Sees sees = row_sees(a, req.before + static_cast<int>(token));
            const T *q_row = static_cast<const T *>(a.query) + (req.first_row + token) * a.query_token + h * a.query_head;
            for (int k = first; k < last; ++k)
#pragma unroll 1
              for (int w = 0; w < kUnit / kWaveTokens; ++w) {
                const int t0 = unit_token(span, k) + w * kWaveTokens;
                const int p0 = page_at(a, table, span, t0), p1 = page_at(a, table, span, t0 + 16);
                if (tile_whole(t0, (p0 >= 0 ? 1u : 0u) | (p1 >= 0 ? 2u : 0u))) continue;
                add_left_out<T, DIM>(a, head, p0, t0, q_row, sees, scale2, base, d0, o);
                add_left_out<T, DIM>(a, head, p1, t0 + 16, q_row, sees, scale2, base, d0, o);
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
    row0 += kRows;
    if (row0 >= req.queries * a.group) {
      row0 = 0;
      if (++head == kv_heads) {
        head = 0;
        do req = same(attn_request(a, ++b)); while (req.queries == 0);
      }
    }
    span = same(attn_span<kRows>(a, req, row0));
  }
}

// ---- launch ------------------------------------------------------------------------

inline AttnShape attn_shape(int64_t tokens, int heads, int kv_heads, int dim, int elem_type, int64_t requests,
                            int64_t max_query_len) {
  const int64_t longest = max_query_len > 0 ? std::min(max_query_len, tokens) : std::max<int64_t>(tokens - requests + 1, 1);
  const int64_t group = heads / kv_heads, rows = longest * group;
  AttnShape s;
  // Which kernel. 32 rows at a time, read anew for each 32, against 256 (128) rows that share what is decoded, of which a last
  // item that is not full costs as much as a full one. 16 requests of 8,000 tokens, 8 heads, us by the kernels for few and for many:
  //   128 dimensions, bfloat16: 128 rows a request 130 and 135, 160 rows 167 and 136, 256 rows 236 and 144, 288 rows 277 and 243;
  //   float16: 192 rows 208 and 212, 224 rows 245 and 214, 352 rows 376 and 386, 384 rows 405 and 388;
  //   64 dimensions: bfloat16 128 rows 102 and 105, 160 rows 123 and 106; float16 192 rows 141 and 152, 224 rows 176 and 153;
  //   256 dimensions: 64 rows 179 and 185, 96 rows 293 and 191; float16 64 rows 193 and 277, 96 rows 312 and 282.
  // So an item costs as much as 4 (float16 6, 256 dimensions 2) of 32 rows. Where there are few items most of the card idles
  // behind the first of them: one request of 8,000 tokens, 384 / 512 / 768 rows: 49 / 58 / 75 us and 49 / 58 / 56 us.
  const int64_t few_items = (rows + 31) / 32, many_items = (rows + many_rows(dim) - 1) / many_rows(dim);
  const int64_t worth = dim == 256 ? 2 : elem_type == SHMT_F16 ? 6 : 4;
  s.many = rows > 2 * many_rows(dim) || (few_items > worth * many_items && tokens * group * kv_heads >= 16384);
  s.rows = s.many ? many_rows(dim) : rows <= 16 ? 16 : 32;
  s.groups = s.many ? attn_many_groups() : 256 * attn_waves(dim, s.rows / 16);
  s.items = s.many ? tokens * group / s.rows + requests : 0;
  const int64_t lines = 2 * s.groups * s.rows;
  s.parts_bytes = lines * dim * 4;
  s.stats_bytes = lines * 8;
  s.record_bytes = s.groups * static_cast<int64_t>(sizeof(JoinRecord));
  s.item_bytes = s.items ? (s.items + 2) * static_cast<int64_t>(sizeof(AttnItem)) : 0;  // the count behind the last one
  s.first_bytes = s.items ? (requests + 4) / 4 * 16 : 0;
  return s;
}

template <typename T, int DIM, int NT>
void launch_few(const AttnArgs &a, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  hipLaunchKernelGGL((page_attention_kernel<T, DIM, NT>), dim3(groups), dim3(256), 0, stream, a, s.parts, s.stats, s.records);
  hipLaunchKernelGGL((page_attention_join_kernel<T, DIM, 16 * NT>), dim3(std::min(groups, 512u)), dim3(256), 0, stream, a,
                     s.parts, s.stats, s.records, static_cast<int>(groups));
}

template <typename T, int DIM>
void launch_few(const AttnArgs &a, int rows, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  if (rows == 16) launch_few<T, DIM, 1>(a, groups, s, stream);
  else launch_few<T, DIM, 2>(a, groups, s, stream);
}

template <typename T>
void launch_few(const AttnArgs &a, int dim, int rows, unsigned groups, const AttnScratch &s, hipStream_t stream) {
  if (dim == 64) launch_few<T, 64>(a, rows, groups, s, stream);
  else if (dim == 128) launch_few<T, 128>(a, rows, groups, s, stream);
  else launch_few<T, 256>(a, rows, groups, s, stream);
}

void launch_attention(const AttnArgs &a, int dim, int elem_type, const AttnShape &shape, void *scratch, hipStream_t stream) {
  char *at = static_cast<char *>(scratch);
  AttnScratch s{};
  s.parts = reinterpret_cast<float *>(at);
  s.stats = reinterpret_cast<float *>(at += shape.parts_bytes);
  s.records = reinterpret_cast<JoinRecord *>(at += shape.stats_bytes);
  s.items = reinterpret_cast<AttnItem *>(at += shape.record_bytes);
  s.count = reinterpret_cast<int32_t *>(s.items + shape.items + 1);
  s.first_item = reinterpret_cast<int32_t *>(at += shape.item_bytes);
  s.room = shape.items;
  // no more workgroups than there can be units
  const int64_t units = (a.tokens * a.group / shape.rows + a.requests) * a.v.kv_heads *
                        (a.limit / kUnit + 1 + item_cost(shape.rows));
  const unsigned groups = static_cast<unsigned>(std::min(shape.groups, std::max<int64_t>(units, 1)));
  if (shape.many) launch_attention_many(a, dim, elem_type, groups, s, stream);
  else if (elem_type == SHMT_F16) launch_few<_Float16>(a, dim, shape.rows, groups, s, stream);
  else launch_few<__bf16>(a, dim, shape.rows, groups, s, stream);
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
  SHMT_REQUIRE(tokens * heads < (int64_t{1} << 30), "query rows x heads must be below 2^30");
  SHMT_REQUIRE(requests >= 0 && requests < (int64_t{1} << 31), "the number of requests must be in [0, 2^31)");
  SHMT_REQUIRE(width >= 0 && width <= (int64_t{1} << 30) / cache->page,
               "the block table holds too many tokens: more than 2^30 a request");
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
  constexpr int64_t kMost = 0x7fffffff;  // a longer window, or more sinks, than any request has tokens
  const AttnArgs a{v, query, query_token_stride, query_head_stride, tokens, heads, heads / cache->kv_heads, block_table,
                   table_stride, query_starts, kv_lens, len_bytes, requests, softmax_scale,
                   static_cast<int32_t>(std::min(window, kMost)), static_cast<int32_t>(std::min(sinks, kMost)),
                   v.pages > 0 ? static_cast<int32_t>(width * cache->page) : 0, out, lse};
  launch_attention(a, cache->dim, elem_type, shape, scratch, as_stream(stream));
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
