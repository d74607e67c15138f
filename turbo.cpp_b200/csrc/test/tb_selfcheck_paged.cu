// Host-side check of the paged cache's address arithmetic (no device needed).
#include "tb_paged.cuh"

using namespace tb;

// row_offset for a cache of this shape, page id, position and head.
extern "C" __attribute__((visibility("default"))) int64_t tb_selfcheck_paged_row(const tb_paged_cache *c, int32_t id,
                                                                                 int t, int64_t head) {
  const int size = dtype_size(c->dtype);
  PagedPools p = {};
  p.page_stride = c->page_stride * size;
  p.token_stride = c->token_stride * size;
  p.head_stride = c->head_stride * size;
  p.n_pages = (uint32_t)c->n_pages;
  p.mask = c->page_size - 1;
  return row_offset(p, id, t, head);
}
