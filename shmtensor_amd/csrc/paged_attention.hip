// Attention over the paged key/value cache: which kernel a call takes, and the entry points (shmt_page_attention,
// shmt_page_attention_as). The kernels are in paged_attention_few.h and paged_attention_many.h, compiled in a file each for 4
// and 8 bits and each rule of what a row sees.
#include "paged_attention.h"
#include "paged_host.h"

namespace shmt {

// ---- launch ------------------------------------------------------------------------

// Up to how many tokens, as far as the table has room for them, an item is one workgroup's own. Nothing is joined then, which
// spares a launch and the parts, but an item's tiles come one after the other. us, dealt out and alone, 8 heads of 4 query heads:
// few rows, 128 dimensions, one request of 256 / 512 / 1,024 tokens, 4 rows: 13.5 and 10.0 / 13.5 and 11.7 / 13.7 and 15.0; 64
// requests, 32 rows: 19.7 and 16.9 / 24.3 and 21.7; 256 dimensions in 8 bits, one request, 32 rows: 22.6 and 20.9 / 22.7 and 25.8.
// Many rows, trees, one request, 256 rows of 256 / 512 tokens: 22.1 and 15.6 / 22.6 and 17.3; 8 requests: 37.4 and 32.2 / 40.5 and
// 42.2.
// Chains in 4 bits are always dealt out, and keep their results.
constexpr int alone_tokens(bool many, int dim) { return many || dim == 256 ? 256 : 512; }

// `limit`: the tokens that a row of the table has room for; -1: not known, room for all that may be chosen.
inline AttnShape attn_shape(int64_t tokens, int heads, int kv_heads, int bits, int seen, int dim, int elem_type, int64_t requests,
                            int64_t max_query_len, int64_t limit) {
  const int64_t longest = max_query_len > 0 ? std::min(max_query_len, tokens) : std::max<int64_t>(tokens - requests + 1, 1);
  const int64_t group = heads / kv_heads, rows = longest * group;
  AttnShape s;
  // Which kernel. 32 rows at a time, read anew for each 32, against 256 (128) rows that share what is decoded, of which a last
  // item that is not full costs as much as a full one. 16 requests of 8,000 tokens, 8 heads, us by the kernels for few and for many:
  //   128 dimensions, bfloat16: 128 rows a request 130 and 135, 160 rows 167 and 136, 256 rows 236 and 144, 288 rows 277 and 243;
  //   float16: 192 rows 208 and 212, 224 rows 245 and 214, 352 rows 376 and 386, 384 rows 405 and 388;
  //   64 dimensions: bfloat16 128 rows 102 and 105, 160 rows 123 and 106; float16 192 rows 141 and 152, 224 rows 176 and 153;
  //   256 dimensions: 64 rows 179 and 185, 96 rows 293 and 191; float16 64 rows 193 and 277, 96 rows 312 and 282.
  // So an item of chains in 4 bits costs as much as 4 (float16 6, 256 dimensions 2) of 32 rows. Where there are few items most of the
  // card idles behind the first of them: one request of 8,000 tokens, 384 / 512 / 768 rows: 49 / 58 / 75 us and 49 / 58 / 56 us.
  // Trees, an encoder's states and 8 bits, where the weights of bfloat16 queries have two parts too: a last item of half the rows or
  // fewer is told apart, as the waves that have none of them only decode. As above, bfloat16, us, few and many:
  //   128 dimensions: trees in 4 bits 128 rows 128 and 143, 160 rows 167 and 191, 192 rows 191 and 194, 224 rows 227 and 196, 320 rows
  //   313 and 320, 384 rows 368 and 319; in 8 bits 96 rows 142 and 151, 128 rows 145 and 152, 160 rows 211 and 203, 320 rows 362 and 341;
  //   states in 4 bits 160 rows 166 and 185, 192 rows 189 and 188; chains in 8 bits 128 rows 133 and 144, 160 rows 206 and 198;
  //   64 dimensions: trees in 4 bits 128 rows 103 and 106, 160 rows 130 and 144, 192 rows 151 and 147, 320 rows 245 and 240; in 8 bits
  //   160 rows 137 and 152, 192 rows 155 and 153; states in 4 bits 160 rows 128 and 138, 192 rows 147 and 140;
  //   256 dimensions: trees in 4 bits 64 rows 162 and 177, 96 rows 243 and 235, 160 rows 389 and 395; in 8 bits 32 rows 124 and 178, 64
  //   rows 197 and 188, 96 rows 330 and 249.
  // float16, trees: 128 dimensions in 4 bits, 128 rows 141 and 164, 192 rows 216 and 224, 224 rows 251 and 228, 320 rows 344 and 409;
  //   256 dimensions: 64 rows 187 and 232, 96 rows 289 and 280, in 8 bits 96 rows 357 and 363, 128 rows 402 and 374.
  const bool f16 = elem_type == SHMT_F16;
  const bool other = bits == 8 || seen != SHMT_SEEN_CAUSAL;  // than chains in 4 bits
  const int64_t few_items = (rows + 31) / 32, whole = rows / many_rows(dim), rest = rows % many_rows(dim);
  const int64_t worth = dim == 256 ? 2 + (f16 && bits == 8) : f16 ? 6 : !other ? 4 : dim == 64 ? 5 : bits == 8 ? 4 : 6;
  int64_t last = rest > 0 ? worth : 0;  // what the last item is worth
  if (other && rest > 0 && rest <= many_rows(dim) / 2) last = dim == 256 ? 2 - (!f16 && bits == 8) : 4;
  s.many = rows > 2 * many_rows(dim) || (few_items > worth * whole + last && tokens * group * kv_heads >= 16384);
  auto few_groups = [&](int rows_of_item) { return int64_t{256} * attn_waves(bits, seen, f16, dim, rows_of_item / 16); };
  s.alone = other && limit >= 0 && limit <= alone_tokens(s.many, dim);
  s.rows = s.many ? many_rows(dim) : rows <= 16 ? 16 : 32;
  s.groups = s.many ? attn_many_groups() : few_groups(s.rows);
  s.room_rows = s.groups * s.rows;
  s.room_groups = s.groups;
  // 16 rows at a time where that leaves no workgroup more than one unit: one request of 912 tokens, 36 rows, 15.0 us instead of
  // 17.4; alone, 256 tokens, 32 rows: 10.9 us instead of 13.7.
  if (other && !s.many && s.rows == 32) {
    const int64_t groups = few_groups(16), items = requests * kv_heads * ((rows + 15) / 16);
    s.room_rows = std::max(s.room_rows, groups * 16), s.room_groups = std::max(s.room_groups, groups);
    if (limit >= 0 && items <= groups / (s.alone ? 1 : limit / kUnit + 1 + item_cost(16))) s.rows = 16, s.groups = groups;
  }
  s.items = s.many ? tokens * group / s.rows + requests : 0;
  const int64_t lines = 2 * s.room_rows;
  s.parts_bytes = lines * dim * 4;
  s.stats_bytes = lines * 8;
  s.record_bytes = s.room_groups * static_cast<int64_t>(sizeof(JoinRecord));
  s.item_bytes = s.items ? (s.items + 2) * static_cast<int64_t>(sizeof(AttnItem)) : 0;  // the count behind the last one
  s.first_bytes = s.items ? (requests + 4) / 4 * 16 : 0;
  return s;
}

void launch_attention(AttnArgs a, int bits, int seen, int dim, int elem_type, const AttnShape &shape, void *scratch,
                      hipStream_t stream) {
  char *at = static_cast<char *>(scratch);
  AttnScratch s{};
  s.parts = reinterpret_cast<float *>(at);
  s.stats = reinterpret_cast<float *>(at += shape.parts_bytes);
  s.records = reinterpret_cast<JoinRecord *>(at += shape.stats_bytes);
  s.items = reinterpret_cast<AttnItem *>(at += shape.record_bytes);
  s.count = reinterpret_cast<int32_t *>(s.items + shape.items + 1);
  s.first_item = reinterpret_cast<int32_t *>(at += shape.item_bytes);
  s.room = shape.items;
  a.alone = shape.alone;
  // no more workgroups than there can be units
  const int64_t units = (a.tokens * a.group / shape.rows + a.requests) * a.v.kv_heads *
                        (a.alone ? 1 : a.limit / kUnit + 1 + item_cost(shape.rows));
  const unsigned groups = static_cast<unsigned>(std::min(shape.groups, std::max<int64_t>(units, 1)));
  auto launch = [&](auto bits, auto seen) {
    constexpr int kBits = decltype(bits)::value, kSeen = decltype(seen)::value;
    if (shape.many) launch_attention_many<kBits, kSeen>(a, dim, elem_type, groups, s, stream);
    else launch_attention_few<kBits, kSeen>(a, dim, elem_type, shape.rows, groups, s, stream);
  };
  auto with_seen = [&](auto bits) {
    if (seen == SHMT_SEEN_TREE) launch(bits, std::integral_constant<int, SHMT_SEEN_TREE>{});
    else if (seen == SHMT_SEEN_ALL) launch(bits, std::integral_constant<int, SHMT_SEEN_ALL>{});
    else launch(bits, std::integral_constant<int, SHMT_SEEN_CAUSAL>{});
  };
  if (bits == 8) with_seen(std::integral_constant<int, 8>{});
  else with_seen(std::integral_constant<int, 4>{});
}

}  // namespace shmt

using namespace shmt;

extern "C" {

int64_t shmt_page_attention_as_scratch_bytes(int64_t tokens, int heads, int kv_heads, int bits, int seen, int dim, int elem_type,
                                             int64_t requests, int64_t max_query_len) {
  if (tokens < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || (bits != 4 && bits != 8) ||
      seen < SHMT_SEEN_CAUSAL || seen > SHMT_SEEN_ALL || (dim != 64 && dim != 128 && dim != 256) ||
      (elem_type != SHMT_F16 && elem_type != SHMT_BF16) || requests < 0 || max_query_len < 0) {
    set_error("bad arguments for the attention's scratch size");
    return -1;
  }
  return attn_shape(tokens, heads, kv_heads, bits, seen, dim, elem_type, requests, max_query_len, -1).bytes();
}

int64_t shmt_page_attention_scratch_bytes(int64_t tokens, int heads, int kv_heads, int dim, int elem_type,
                                          int64_t requests, int64_t max_query_len) {
  return shmt_page_attention_as_scratch_bytes(tokens, heads, kv_heads, 4, SHMT_SEEN_CAUSAL, dim, elem_type, requests,
                                              max_query_len);
}

int shmt_page_attention(const shmt_paged_cache *cache, const void *query, int64_t query_token_stride,
                        int64_t query_head_stride, int elem_type, int64_t tokens, int heads,
                        const int32_t *block_table, int64_t width, int64_t table_stride, const void *query_starts,
                        const void *kv_lens, int len_bytes, int64_t requests, float softmax_scale, int64_t window,
                        int64_t sinks, int64_t max_query_len, void *out, float *lse, void *scratch,
                        int64_t scratch_bytes, void *stream) {
  return shmt_page_attention_as(cache, 4, SHMT_SEEN_CAUSAL, nullptr, query, query_token_stride, query_head_stride, elem_type,
                                tokens, heads, block_table, width, table_stride, query_starts, kv_lens, len_bytes, requests,
                                softmax_scale, window, sinks, max_query_len, out, lse, scratch, scratch_bytes, stream);
}

int shmt_page_attention_as(const shmt_paged_cache *cache, int bits, int seen, const int32_t *nodes, const void *query,
                           int64_t query_token_stride, int64_t query_head_stride, int elem_type, int64_t tokens, int heads,
                           const int32_t *block_table, int64_t width, int64_t table_stride, const void *query_starts,
                           const void *kv_lens, int len_bytes, int64_t requests, float softmax_scale, int64_t window,
                           int64_t sinks, int64_t max_query_len, void *out, float *lse, void *scratch,
                           int64_t scratch_bytes, void *stream) {
  PagedView v;
  const int rc = paged_view(cache, bits, &v);
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
  SHMT_REQUIRE(seen == SHMT_SEEN_CAUSAL || seen == SHMT_SEEN_TREE || seen == SHMT_SEEN_ALL, "unknown rule of what is seen: %d",
               seen);
  SHMT_REQUIRE(seen != SHMT_SEEN_ALL || window == 0, "rows that see all have no window");
  SHMT_REQUIRE(softmax_scale == softmax_scale && softmax_scale - softmax_scale == 0, "softmax_scale must be finite");
  if (tokens == 0) return SHMT_OK;
  SHMT_REQUIRE(query && out, "query or out is null");
  SHMT_REQUIRE(requests == 0 || (query_starts && kv_lens), "query_starts or kv_lens is null");
  SHMT_REQUIRE(requests == 0 || width == 0 || (block_table && table_stride >= width), "block_table is null or narrow");
  SHMT_REQUIRE(((reinterpret_cast<int64_t>(query) | query_token_stride * 2 | query_head_stride * 2) & 15) == 0,
               "every row of query has to begin on 16 bytes");
  SHMT_REQUIRE((reinterpret_cast<int64_t>(out) & 15) == 0, "out has to begin on 16 bytes");
  SHMT_REQUIRE(seen != SHMT_SEEN_TREE || (nodes && (reinterpret_cast<int64_t>(nodes) & 15) == 0),
               "nodes is null or does not begin on 16 bytes");
  const AttnShape shape = attn_shape(tokens, heads, cache->kv_heads, bits, seen, cache->dim, elem_type, requests, max_query_len,
                                     v.pages > 0 ? width * cache->page : 0);
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
                   v.pages > 0 ? static_cast<int32_t>(width * cache->page) : 0, out, lse, 0,
                   seen == SHMT_SEEN_TREE ? reinterpret_cast<const int4 *>(nodes) : nullptr};
  launch_attention(a, bits, seen, cache->dim, elem_type, shape, scratch, as_stream(stream));
  SHMT_LAUNCH_CHECK();
  return SHMT_OK;
}

}  // extern "C"
