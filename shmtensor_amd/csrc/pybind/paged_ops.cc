// The paged key/value cache held in 4 bits, as operators of ShmTensorLib:
// page_plan, page_set, page_fetch, page_attention (no counterpart in the
// reference; what they compute is in include/shmt.h). Host C++ only: tensors
// are checked here, outputs and scratch come from torch's caching allocator,
// the work goes to torch's current stream and nothing waits for it.
#include <ATen/hip/EmptyTensor.h>

#include <cmath>

#include "shim.h"

namespace shim {

namespace {

// A new contiguous tensor on the device of `like`, without the dispatcher's round (a small call makes five of them).
torch::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const torch::Tensor &like) {
  return torch::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

int elem_type(at::ScalarType t, const char *name) {
  if (t == torch::kFloat32) return SHMT_F32;
  if (t == torch::kFloat16) return SHMT_F16;
  if (t == torch::kBFloat16) return SHMT_BF16;
  TORCH_CHECK(false, name, " can only be float32, float16 or bfloat16, got ", t);
}

void check_device(const torch::Tensor &t, const torch::Tensor &like, const char *name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", the cache on ", like.device());
}

// Nothing is learned through the rounded rows of a cache: a gradient that somebody waits for is refused, not lost.
void check_no_grad(const torch::Tensor &t, const char *name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
              " requires a gradient, which the paged cache does not give: call it under torch.no_grad() or detach() first");
}

bool page_contiguous(const torch::Tensor &t) {
  int64_t want = 1;
  for (int64_t d = 4; d >= 1; --d) {
    if (t.size(d) > 1 && t.stride(d) != want) return false;
    want *= t.size(d);
  }
  return true;
}

shmt_paged_cache describe(const torch::Tensor &cache, const torch::Tensor &scales) {
  TORCH_CHECK(cache.is_cuda(), "cache must be a CUDA tensor");
  TORCH_CHECK(cache.device().index() == c10::hip::current_device(), "cache is on ", cache.device(),
              ", which is not the current device");
  check_device(scales, cache, "scales");
  TORCH_CHECK(cache.scalar_type() == torch::kUInt8 && scales.scalar_type() == torch::kUInt8,
              "cache and scales must be uint8 tensors");
  TORCH_CHECK(cache.dim() == 5 && cache.size(2) == 2, "cache must be [pages, kv_heads, 2, page, dim / 2], got ",
              cache.sizes());
  const int64_t pages = cache.size(0), heads = cache.size(1), page = cache.size(3), half = cache.size(4);
  TORCH_CHECK(half == 32 || half == 64 || half == 128, "a row must have 64, 128 or 256 values, not ", half * 2);
  TORCH_CHECK(scales.dim() == 5 && scales.size(0) == pages && scales.size(1) == heads && scales.size(2) == 2 &&
                  scales.size(3) == half / 16 && scales.size(4) == page,
              "scales must be [pages, kv_heads, 2, dim / 32, page] of the same cache, got ", scales.sizes(), " beside ",
              cache.sizes());
  TORCH_CHECK(page <= 256 && heads >= 1 && heads <= 65535, "a page must hold 16, 32, 64, 128 or 256 tokens of 1 to 65535 heads");
  // within a page everything is contiguous; pages may lie apart
  TORCH_CHECK(pages == 0 || (page_contiguous(cache) && page_contiguous(scales)),
              "the pages of cache and scales must be contiguous");
  shmt_paged_cache c;
  c.cache = cache.data_ptr();
  c.scales = scales.data_ptr();
  c.pages = pages;
  c.cache_page_stride = pages > 1 ? cache.stride(0) : 0;
  c.scales_page_stride = pages > 1 ? scales.stride(0) : 0;
  c.kv_heads = static_cast<int>(heads);
  c.dim = static_cast<int>(half * 2);
  c.page = static_cast<int>(page);
  return c;
}

// Rows [tokens, heads, dim] as the kernels read them: any strides between tokens and heads as long as every row
// begins on 16 bytes; others are copied.
torch::Tensor rows_on_16(const torch::Tensor &t) {
  const int64_t e = static_cast<int64_t>(t.element_size());
  const bool fine = t.numel() == 0 ||
                    (t.stride(2) == 1 && (reinterpret_cast<intptr_t>(t.data_ptr()) & 15) == 0 &&
                     (t.size(0) == 1 || t.stride(0) * e % 16 == 0) && (t.size(1) == 1 || t.stride(1) * e % 16 == 0));
  return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t stride_of(const torch::Tensor &t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// A block table, row by row.
int64_t table_stride(const torch::Tensor &t) {
  TORCH_CHECK(t.is_cuda(), "block_table must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == torch::kInt32, "block_table must be an int32 tensor, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 2, "block_table must be [requests, pages of a request], got ", t.sizes());
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, "the rows of block_table must be contiguous");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), "the rows of block_table overlap");
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

}  // namespace

// Block tables and slot maps of a step from its requests' lengths (shmt_page_plan).
std::vector<torch::Tensor> page_plan(torch::Tensor cached_lens, torch::Tensor new_lens, torch::Tensor block_table,
                                     torch::Tensor free_pages, int64_t page, int64_t max_tokens) {
  const int64_t stride = table_stride(block_table);
  TORCH_CHECK(block_table.device().index() == c10::hip::current_device(), "block_table is on ", block_table.device(),
              ", which is not the current device");
  cached_lens = cuda_ids(cached_lens, "cached_lens");
  new_lens = cuda_ids(new_lens, "new_lens");
  TORCH_CHECK(cached_lens.scalar_type() == new_lens.scalar_type(), "cached_lens and new_lens must have one type");
  const int64_t n = block_table.size(0);
  TORCH_CHECK(cached_lens.dim() == 1 && new_lens.dim() == 1 && cached_lens.numel() == n && new_lens.numel() == n,
              "cached_lens and new_lens must hold a length for each row of block_table (", n, ")");
  TORCH_CHECK(free_pages.is_cuda() && free_pages.scalar_type() == torch::kInt32 && free_pages.dim() == 1,
              "free_pages must be a one-dimensional int32 CUDA tensor");
  for (const auto &t : {cached_lens, new_lens, free_pages})
    TORCH_CHECK(t.device() == block_table.device(), "all tensors must be on one device");
  TORCH_CHECK(max_tokens >= 0 && max_tokens < (int64_t{1} << 31), "max_tokens must be in [0, 2^31)");
  TORCH_CHECK(page > 0 && page <= 256, "a page must hold 16, 32, 64, 128 or 256 tokens, not ", page);
  free_pages = free_pages.contiguous();
  auto empty = [&](int64_t size, at::ScalarType type) { return new_tensor({size}, type, block_table); };
  torch::Tensor starts = empty(n + 1, torch::kInt32), kv_lens = empty(n, torch::kInt32);
  torch::Tensor positions = empty(max_tokens, torch::kInt32), slots = empty(max_tokens, torch::kInt64);
  torch::Tensor counts = empty(2, torch::kInt64);
  const int64_t scratch_bytes = shmt_page_plan_scratch_bytes(n);
  torch::Tensor scratch = scratch_bytes > 0 ? device_bytes(scratch_bytes) : torch::Tensor();
  check(shmt_page_plan(cached_lens.data_ptr(), new_lens.data_ptr(), static_cast<int>(cached_lens.element_size()), n,
                       block_table.data_ptr<int32_t>(), block_table.size(1), stride, free_pages.data_ptr<int32_t>(),
                       free_pages.numel(), static_cast<int>(page), max_tokens, starts.data_ptr<int32_t>(),
                       kv_lens.data_ptr<int32_t>(), positions.data_ptr<int32_t>(), slots.data_ptr<int64_t>(),
                       counts.data_ptr<int64_t>(), scratch_bytes > 0 ? scratch.data_ptr() : nullptr, scratch_bytes,
                       current_stream()));
  return {starts, kv_lens, positions, slots, counts};
}

// Rows of keys and values rounded into their slots (shmt_page_set).
void page_set(const torch::Tensor &cache, const torch::Tensor &scales, torch::Tensor slots, torch::Tensor keys,
              torch::Tensor values) {
  const shmt_paged_cache c = describe(cache, scales);
  slots = cuda_ids(slots, "slots");
  check_device(slots, cache, "slots");
  check_device(keys, cache, "keys");
  check_device(values, cache, "values");
  check_no_grad(keys, "keys");
  check_no_grad(values, "values");
  const int64_t n = slots.numel();
  const int64_t sizes[3] = {n, c.kv_heads, c.dim};
  const at::IntArrayRef shape(sizes);
  TORCH_CHECK(keys.sizes() == shape && values.sizes() == shape, "keys and values must be [slots, kv_heads, dim] = ",
              shape, ", got ", keys.sizes(), " and ", values.sizes());
  TORCH_CHECK(keys.scalar_type() == values.scalar_type(), "keys and values must have one type");
  const int type = elem_type(keys.scalar_type(), "keys and values");
  if (n == 0) return;
  keys = rows_on_16(keys);
  values = rows_on_16(values);
  check(shmt_page_set(&c, slots.data_ptr(), static_cast<int>(slots.element_size()), n, keys.data_ptr(),
                      stride_of(keys, 0), stride_of(keys, 1), values.data_ptr(), stride_of(values, 0),
                      stride_of(values, 1), type, current_stream()));
}

// The values that the rows at `slots` stand for (shmt_page_fetch).
std::vector<torch::Tensor> page_fetch(const torch::Tensor &cache, const torch::Tensor &scales, torch::Tensor slots,
                                      at::ScalarType dtype) {
  const shmt_paged_cache c = describe(cache, scales);
  slots = cuda_ids(slots, "slots");
  check_device(slots, cache, "slots");
  const int type = elem_type(dtype, "dtype");
  torch::Tensor keys = new_tensor({slots.numel(), c.kv_heads, c.dim}, dtype, cache);
  torch::Tensor values = new_tensor({slots.numel(), c.kv_heads, c.dim}, dtype, cache);
  check(shmt_page_fetch(&c, slots.data_ptr(), static_cast<int>(slots.element_size()), slots.numel(), keys.data_ptr(),
                        values.data_ptr(), type, current_stream()));
  return {keys, values};
}

// Attention of the requests' new tokens over the cache (shmt_page_attention).
py::object page_attention(torch::Tensor query, const torch::Tensor &cache, const torch::Tensor &scales,
                          const torch::Tensor &block_table, torch::Tensor query_starts, torch::Tensor kv_lens,
                          std::optional<double> softmax_scale, int64_t window, int64_t sinks, int64_t max_query_len,
                          bool return_lse) {
  const shmt_paged_cache c = describe(cache, scales);
  check_device(query, cache, "query");
  check_no_grad(query, "query");
  check_device(block_table, cache, "block_table");
  const int64_t stride = table_stride(block_table);
  query_starts = cuda_ids(query_starts, "query_starts");
  kv_lens = cuda_ids(kv_lens, "kv_lens");
  check_device(query_starts, cache, "query_starts");
  check_device(kv_lens, cache, "kv_lens");
  TORCH_CHECK(query_starts.scalar_type() == kv_lens.scalar_type(), "query_starts and kv_lens must have one type");
  TORCH_CHECK(query.scalar_type() == torch::kFloat16 || query.scalar_type() == torch::kBFloat16,
              "query can only be float16 or bfloat16, got ", query.scalar_type());
  TORCH_CHECK(query.dim() == 3 && query.size(2) == c.dim, "query must be [tokens, heads, ", c.dim, "], got ",
              query.sizes());
  TORCH_CHECK(query.size(1) >= 1 && query.size(1) <= 65535 && query.size(1) % c.kv_heads == 0, query.size(1),
              " query heads do not share ", c.kv_heads, " heads of the cache evenly");
  const int64_t n = block_table.size(0), tokens = query.size(0), heads = query.size(1);
  TORCH_CHECK(query_starts.dim() == 1 && query_starts.numel() == n + 1 && kv_lens.dim() == 1 && kv_lens.numel() == n,
              "block_table has ", n, " requests: query_starts must hold one entry more, kv_lens as many");
  TORCH_CHECK(window >= 0 && sinks >= 0 && max_query_len >= 0, "window, sinks and max_query_len must be >= 0");
  torch::Tensor out = new_tensor({tokens, heads, c.dim}, query.scalar_type(), query);
  torch::Tensor lse;
  if (return_lse) lse = new_tensor({tokens, heads}, torch::kFloat32, query);
  if (tokens > 0) {
    query = rows_on_16(query);
    const int64_t scratch_bytes = shmt_page_attention_scratch_bytes(tokens, static_cast<int>(heads), c.kv_heads, c.dim,
                                                                    elem_type(query.scalar_type(), "query"), n,
                                                                    max_query_len);
    TORCH_CHECK(scratch_bytes >= 0, shmt_last_error());
    torch::Tensor scratch = new_tensor({scratch_bytes}, torch::kUInt8, cache);
    const float scale = softmax_scale ? static_cast<float>(*softmax_scale)
                                      : 1.0f / std::sqrt(static_cast<float>(c.dim));
    check(shmt_page_attention(&c, query.data_ptr(), stride_of(query, 0), stride_of(query, 1),
                              elem_type(query.scalar_type(), "query"), tokens, static_cast<int>(heads),
                              block_table.data_ptr<int32_t>(), block_table.size(1), stride, query_starts.data_ptr(),
                              kv_lens.data_ptr(), static_cast<int>(kv_lens.element_size()), n, scale, window, sinks,
                              max_query_len, out.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
                              scratch.data_ptr(), scratch_bytes, current_stream()));
  }
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

void register_paged_ops(py::module &m) {
  m.def("page_plan", &page_plan, py::arg("cached_lens"), py::arg("new_lens"), py::arg("block_table"),
        py::arg("free_pages"), py::arg("page"), py::arg("max_tokens"),
        "Pages and slots for the new tokens of a step: extends block_table in place with pages from free_pages and "
        "returns [query_starts, kv_lens, positions, slots, counts]; counts = [new tokens, pages taken]. Tokens "
        "without a page have slot -1.");
  m.def("page_set", &page_set, py::arg("cache"), py::arg("scales"), py::arg("slots"), py::arg("keys"),
        py::arg("values"),
        "Rounds rows of keys and values [n, kv_heads, dim] to 4 bits and writes them to their slots (-1: nowhere).");
  m.def("page_fetch", &page_fetch, py::arg("cache"), py::arg("scales"), py::arg("slots"), py::arg("dtype"),
        "[keys, values]: what the rows at `slots` stand for, in `dtype`; 0 for slots outside the cache.");
  m.def("page_attention", &page_attention, py::arg("query"), py::arg("cache"), py::arg("scales"),
        py::arg("block_table"), py::arg("query_starts"), py::arg("kv_lens"), py::arg("softmax_scale") = py::none(),
        py::arg("window") = 0, py::arg("sinks") = 0, py::arg("max_query_len") = 0, py::arg("return_lse") = false,
        "Attention of each request's new tokens (the last of its kv_lens tokens) over what the cache holds for it, or "
        "over a window of it and the first `sinks` tokens. out [tokens, heads, dim], with return_lse (out, lse).");
}

}  // namespace shim
