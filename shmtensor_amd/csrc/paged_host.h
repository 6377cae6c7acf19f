// Checks of a paged cache's description, shared by its entry points.
#pragma once
#include "common.h"
#include "paged_dev.h"

namespace shmt {

// log2 of a page size that the kernels handle, or -1.
inline int paged_log2(int page) {
  for (int l = 4; l <= 8; ++l)
    if (page == 1 << l) return l;
  return -1;
}

inline int paged_view(const shmt_paged_cache *c, PagedView *v) {
  SHMT_REQUIRE(c != nullptr, "the cache is null");
  SHMT_REQUIRE(c->dim == 64 || c->dim == 128 || c->dim == 256, "a row must have 64, 128 or 256 values, not %d", c->dim);
  const int log2_page = paged_log2(c->page);
  SHMT_REQUIRE(log2_page >= 0, "a page must hold 16, 32, 64, 128 or 256 tokens, not %d", c->page);
  SHMT_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 65535, "the number of heads must be in [1, 65535]");
  SHMT_REQUIRE(c->pages >= 0 && c->pages < (int64_t{1} << 31), "the number of pages must be in [0, 2^31)");
  const int64_t values = int64_t{c->kv_heads} * 2 * c->page * c->dim;
  SHMT_REQUIRE(c->pages <= 1 || (c->cache_page_stride >= values / 2 && c->scales_page_stride >= values / 32),
               "pages overlap");
  SHMT_REQUIRE(c->pages == 0 || (c->cache && c->scales), "the cache's memory is null");
  SHMT_REQUIRE(((reinterpret_cast<int64_t>(c->cache) | reinterpret_cast<int64_t>(c->scales) | c->cache_page_stride |
                 c->scales_page_stride) & 15) == 0,
               "every page of the cache and of its scales has to begin on 16 bytes");
  *v = PagedView{static_cast<uint8_t *>(c->cache), static_cast<uint8_t *>(c->scales), c->cache_page_stride,
                 c->scales_page_stride, c->pages, c->kv_heads, log2_page};
  return SHMT_OK;
}

}  // namespace shmt
