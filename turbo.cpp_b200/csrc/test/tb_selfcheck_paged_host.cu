// Host-side checks of the paged attention's launch arithmetic (no device needed).
#include "tb_paged.cuh"

using namespace tb;

extern "C" __attribute__((visibility("default"))) int64_t tb_selfcheck_prefix_splits(int64_t items, int64_t tiles,
                                                                                     int64_t ctas, int64_t most) {
  return prefix_splits(items, tiles, ctas, most);
}

// Candidates that the choice looks at.
extern "C" __attribute__((visibility("default"))) int64_t tb_selfcheck_prefix_splits_looks(int64_t items, int64_t tiles,
                                                                                           int64_t ctas, int64_t most) {
  int64_t looks = 0;
  prefix_splits(items, tiles, ctas, most, &looks);
  return looks;
}

// row_offset in the pools that the kernels are given for this cache.
extern "C" __attribute__((visibility("default"))) int64_t tb_selfcheck_paged_row_of(const tb_paged_cache *c, int64_t id,
                                                                                    int64_t t, int64_t head) {
  const PagedPools p = paged_pools(c);
  return (1 << p.shift) != c->page_size ? -2 : row_offset(p, (int32_t)id, (int)t, head);
}
