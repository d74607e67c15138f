// tb_paged.cuh -- what the kernels over the paged key/value cache share.
#pragma once

#include <cuda.h>

#include "tb_internal.cuh"

namespace tb {

// Activation rows (queries, new keys and values, outputs) of a run-time type.
struct ActRows {
  const void *p;
  int64_t ld;  // elements between rows
  int dtype;
};

// The device side of tb_paged_cache / tb_paged_batch.
struct PagedPools {
  const char *k, *v;
  int64_t page_stride, token_stride, head_stride;  // bytes
  uint32_t n_pages;
  int shift, mask;  // position t: slot t & mask of its page t >> shift
};
struct PagedSeqs {
  const int32_t *lens, *table;
  int64_t table_stride;
  int batch;
  int max_len;  // max_pages * page_size
};

// The pools of a cache whose descriptor has been checked.
inline PagedPools paged_pools(const tb_paged_cache *c) {
  const int size = dtype_size(c->dtype);
  PagedPools p = {};
  p.k = static_cast<const char *>(c->k);
  p.v = static_cast<const char *>(c->v);
  // the stride of a single element is never used, and may be anything
  p.page_stride = c->n_pages > 1 ? c->page_stride * size : 0;
  p.token_stride = c->page_size > 1 ? c->token_stride * size : 0;
  p.head_stride = c->kv_heads > 1 ? c->head_stride * size : 0;
  p.n_pages = (uint32_t)c->n_pages;
  p.mask = c->page_size - 1;
  while ((1 << p.shift) < c->page_size) ++p.shift;
  return p;
}

// Byte offset of a key/value head's row at slot t & mask of page `id`, or -1
// where the page id lies outside the pool: the only way from a page table to
// an address in this code (TMA checks its coordinates itself).
__host__ __device__ inline int64_t row_offset(const PagedPools &p, int32_t id, int t, int64_t head) {
  if ((uint32_t)id >= p.n_pages) return -1;
  return id * p.page_stride + (t & p.mask) * p.token_stride + head * p.head_stride;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Checks and converts the two descriptors; `who` names the entry point.
tb_status paged_args(const tb_paged_cache *c, const tb_paged_batch *b, int act_dtype, const char *who,
                     PagedPools *pools, PagedSeqs *seqs);

// Behind a prefix each query row has several partial results: one per split of
// the prefix and a last one of the sequence's own keys.  Unnormalised outputs
// acc[D] with their running maximum m (of scale * log2(e) * q.k) and sum l; row
// r of key/value head h, part p: acc at ((h * rows + r) * parts + p) * D.
struct PrefixParts {
  float *acc;
  float2 *ml;
  int rows;    // batch * group
  int splits;  // 0: no prefix
  int parts;   // splits + 1
  int few;        // few items and short sequences behind it
  int join_here;  // the kernel of the sequences' own keys joins the parts
  // else per item of that kernel: its first CTA's slot and how many CTAs share it (0: one, its part is the row's last)
  int2 *own;
  int slot_rows;  // rows of a slot
  int *begun;     // 1 once the prefix's kernel has seen every earlier one's end; zero between calls
};

// The prefix's kernel, one thread of each CTA, behind its griddepcontrol.wait:
// the next kernel may begin.  That one reads what earlier kernels wrote
// (lengths, tables, pages, queries) but none of this one's results, and waits
// for this one only at its end; what makes the earlier writes visible to it is
// this release, which it acquires (earlier_kernels_seen).
__device__ __forceinline__ void let_next_begin(const PrefixParts &p) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
    asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(p.begun), "r"(1) : "memory");
  pdl_launch_dependents();
}
// All threads of a CTA of the next kernel: false where it has to wait for the prefix's end instead.
__device__ __forceinline__ bool earlier_kernels_seen(const PrefixParts &p) {
  int v = 0;
  if (threadIdx.x == 0) asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.begun) : "memory");
  return __syncthreads_or(v == 1) != 0;
}

// The pools as 4-d tensors [page][token][head][head_dim] for TMA: a box is up
// to `box_rows` tokens of one page and head, 128 bytes of each row, swizzled.
struct PagedMaps {
  CUtensorMap k, v;
};
// `rows` tokens per box at most; *box_rows gets the smaller of that and page_size.
tb_status paged_maps(const tb_paged_cache *c, int rows, const char *who, PagedMaps *maps, int *box_rows);

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int head, int token, int page,
                                        uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(head), "r"(token), "r"(page), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Waits for a barrier's phase; once a wait has run out (bit 0 of the error
// word is set then), later ones return at once, so that the kernel ends.  So
// nothing that decides how often a loop runs or which barriers a thread comes to
// is read from what such a wait orders: a call whose waits ran out multiplies
// what is there and ends.  A reader that gave up on a stage does not hand it
// back: a copy into it may still be under way, and its barrier must not be told
// to expect another one on top.
__device__ __forceinline__ void wait_phase(uint64_t *bar, uint32_t phase, uint32_t *err, bool &dead,
                                           uint64_t limit_ns) {
  if (!dead && !mbar_wait_bounded(bar, phase, err, limit_ns)) dead = true;
}
// What `dead` begins as in a warp: with a limit of 0 no wait may wait at all.  (Asked at each wait, the limit cost the
// tensor cores' loop 3 to 5 %.)
__device__ __forceinline__ bool begin_dead(uint64_t limit_ns, uint32_t *err) {
  if (limit_ns == 0 && (threadIdx.x & 31) == 0) atomicOr(err, ERR_TIMEOUT);
  return limit_ns == 0;
}

// The end of a loading warp that has issued `issued` tiles into STAGES stages:
// its last copies have landed, even where no other warp waits for them any more.
template <int STAGES>
__device__ __forceinline__ void wait_copies(uint64_t *full, int issued, uint32_t *err) {
  for (int k = max(issued - STAGES, 0); k < issued; ++k)
    if (!mbar_wait_bounded(full + k % STAGES, (k / STAGES) & 1, err)) return;
}

// A tile of T keys or values of a sequence of len tokens, in boxes of one page.
struct TileBoxes {
  int n, first;  // boxes that begin before len; page id of this lane's first one
};
template <int T>
__device__ __forceinline__ TileBoxes tile_boxes(const PagedPools &p, int box_shift, const int32_t *table, int len,
                                                int tile) {
  const int lane = threadIdx.x & 31;
  TileBoxes b;
  b.n = (min(max(len - tile * T, 0), T) + (1 << box_shift) - 1) >> box_shift;
  b.first = lane < b.n ? table[(tile * T + (lane << box_shift)) >> p.shift] : 0;
  return b;
}

// One warp: the tile's rows (RB bytes each) into shared memory, 128-byte
// columns T * 128 bytes apart.  A page id outside the pool is given to TMA as
// page -1, whose rows are zeros.  With two maps both tiles are fetched, the
// second T * RB bytes behind the first.
template <int T, int RB, int SIZE>
__device__ __forceinline__ void load_rows(uint32_t dst0, uint64_t *full, const CUtensorMap *m0, const CUtensorMap *m1,
                                          const PagedPools &p, int box_shift, const int32_t *table, TileBoxes b,
                                          int tile, int kvh, uint32_t *err) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)((b.n << box_shift) * (m1 ? 2 : 1) * RB));
  __syncwarp();
  for (int i = lane; i < b.n; i += 32) {
    const int t = tile * T + (i << box_shift);
    int page = i == lane ? b.first : table[t >> p.shift];
    if ((uint32_t)page >= p.n_pages) {
      atomicOr(err, ERR_INDEX);
      page = -1;
    }
    const uint32_t dst = dst0 + (i << (box_shift + 7));
#pragma unroll
    for (int c = 0; c < RB / 128; ++c) {
      tma_box(dst + c * T * 128, m0, c * (128 / SIZE), kvh, t & p.mask, page, full);
      if (m1) tma_box(dst + T * RB + c * T * 128, m1, c * (128 / SIZE), kvh, t & p.mask, page, full);
    }
  }
}

// Two floats as one register of type CT, to nearest, and what is left of them.
template <int CT>
__device__ __forceinline__ uint32_t pack_rest(float &x, float &y) {
  uint32_t u;
  if constexpr (CT == TB_F16) {
    const __half2 h = __floats2half2_rn(x, y);
    u = *reinterpret_cast<const uint32_t *>(&h);
    const float2 f = __half22float2(h);
    x -= f.x, y -= f.y;
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    u = *reinterpret_cast<const uint32_t *>(&h);
    x -= __uint_as_float(u << 16), y -= __uint_as_float(u & 0xFFFF0000u);
  }
  return u;
}

// The exponent e of the power of two that brings a maximum into [2^14, 2^15)
// (0 for 0, inf and NaN), so that fp32 queries fit fp16 parts.
__device__ __forceinline__ int fp16_exp(float mx) {
  const int E = (int)(__float_as_uint(mx) >> 23);
  return mx == 0.f || E == 255 ? 0 : min(max(141 - E, -126), 126);
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

__device__ __forceinline__ void sts128_zero(uint32_t addr) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-byte words of a row as floats (F32: 4, F16 and BF16: 8); exact.
template <int DT>
struct Word;
template <>
struct Word<TB_F32> {
  static constexpr int n = 4, size = 4;
  static __device__ __forceinline__ void get(const uint4 &w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 put(const float *f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Word<TB_F16> {
  static constexpr int n = 8, size = 2;
  static __device__ __forceinline__ void get(const uint4 &w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 put(const float *f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct Word<TB_BF16> {
  static constexpr int n = 8, size = 2;
  static __device__ __forceinline__ void get(const uint4 &w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16), f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float *f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

// N consecutive activations (N = 4 or 8) starting at element i, as floats.
template <int N>
__device__ __forceinline__ void load_act(const void *p, int64_t i, int dtype, float (&f)[N]) {
  if (dtype == TB_F32) {
    const uint4 *s = reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + i);
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      float g[4];
      Word<TB_F32>::get(s[k], g);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * k + e] = g[e];
    }
  } else {  // 16-bit activations meet 16-bit caches only, whose words hold 8 elements
    static_assert(N == 4 || N == 8, "");
    if constexpr (N == 8) {
      const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
      if (dtype == TB_F16) Word<TB_F16>::get(w, f);
      else Word<TB_BF16>::get(w, f);
    }
  }
}

__device__ __forceinline__ void store_act1(void *p, int64_t i, int dtype, float x) {
  if (dtype == TB_F32) static_cast<float *>(p)[i] = x;
  else if (dtype == TB_F16) static_cast<__half *>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

// What an attention launch is given (tb_paged_attention.cu).
struct AttnArgs {
  PagedPools pools;
  PagedSeqs seqs;
  ActRows q;
  void *out;
  int64_t ldo;
  int kv_heads, group, head_groups;  // head_groups: items per (sequence, key/value head)
  float scale2;                      // scale * log2(e)
  int max_ctas;
  int *counters;    // [kMaxCtas], zero between launches
  float *slot_acc;  // [2 kMaxCtas][8 HW][D]
  float2 *slot_ml;  // [2 kMaxCtas][8 HW]
  PrefixParts prefix;
  const int32_t *prefix_table;
  int prefix_len;
  int lead;  // tiles of a short prefix that the decode kernel takes before each sequence's own, instead of a kernel
  int box_shift;  // a TMA box holds 1 << box_shift tokens
  uint64_t wait_ns;  // limit of the kernels' waits
};

// The fewest splits that finish first: `items` row tiles of `tiles` key tiles each on `ctas` CTAs at a time, `most`
// splits at most.  Only the most splits of a number of waves can be that, and waves beyond the first sixteen numbers that
// add a split gain next to nothing (each number tried costs a call two divisions).  Measured against one wave of CTAs
// wherever that many items are (with 16-bit probabilities in one part): 300 x 128 heads behind 8192 keys of 64 (152 row
// tiles) 191 us, with one split 239; 2 x 32 heads (8 row tiles) 12.5 and 15.0.
inline int64_t prefix_splits(int64_t items, int64_t tiles, int64_t ctas, int64_t most, int64_t *looks = nullptr) {
  constexpr int64_t kStart = 6;  // a CTA's start and end, in tiles
  if (most > tiles) most = tiles;
  int64_t best = 1, least = INT64_MAX, waves = (items + ctas - 1) / ctas;
  for (int look = 0; look < 16; ++look) {
    const int64_t n = waves * ctas / items < most ? waves * ctas / items : most;
    const int64_t share = (tiles + n - 1) / n, fewest = (tiles + share - 1) / share;  // the fewest of the same share
    const int64_t time = (items * fewest + ctas - 1) / ctas * (share + kStart);
    if (time < least) best = fewest, least = time;
    if (looks) ++*looks;
    if (n == most) break;
    const int64_t next = (items * (n + 1) + ctas - 1) / ctas;
    waves = next > waves ? next : waves + 1;
  }
  return best;
}

// Sets the prefix's splits, as far as the workspace holds their results.
void set_prefix_splits(AttnArgs &a, int64_t items, int64_t tiles, int64_t ctas);

// A launch that may begin while the kernel before it ends; the kernel waits
// (griddepcontrol.wait) before it reads what that one wrote.
template <typename F, typename... A>
tb_status launch_pdl(F *kern, dim3 grid, int threads, size_t smem, cudaStream_t s, const char *who, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) return fail(TB_ECUDA, "%s: %s", who, cudaGetErrorString(e));
  return check_launch(who);
}

// The prefix on tcgen05 (tb_paged_prefix.cu), 16-bit caches; sets a.prefix.splits.  The maps' boxes are those of 64 keys.
tb_status launch_prefix_tc(AttnArgs &a, const PagedMaps &maps, int cache_dtype, int head_dim, const DeviceState *st,
                           cudaStream_t s, const char *who);

}  // namespace tb
