// tb_paged_append.cu -- tb_rope_paged_append: RoPE of a call's queries and keys
// and the append of its keys and values to a paged cache, one launch for any
// mix of prompts and single tokens.
//
//   q_out = R(p) q,  K[p] = R(p) k,  V[p] = v,
//   R(p): y0 = x0 c - x1 s, y1 = x0 s + x1 c for the pairs (i, i + head_dim/2),
// with tb_rope's fused multiply-adds in fp32, so an fp32 cache holds what
// tb_rope and tb_copy would have put there bit for bit.
//
// It moves every element once and computes next to nothing, so bytes bound it:
// 33k tokens of 32 + 8 + 8 heads of 128 in fp16 take 124 us (6.5 TB/s of the
// measured 6.55), 8k tokens of fp32 heads of 64 into bf16 pages 34.9 us (6.1
// TB/s), one token 2.1 us.
// A thread takes 16 bytes of a head's first half and the 16 they are paired
// with, for one to four heads of one token, so that its cosines and sines are
// read once, and the token's sequence, position and page are found once per
// warp: a 32-way search of `starts` by ballot, then one table entry.  The data
// loads do not depend on that chain and are issued before it.
#include <algorithm>
#include <atomic>

#include "tb_paged.cuh"

namespace tb {

tb_status paged_args(const tb_paged_cache *c, const tb_paged_batch *b, int act_dtype, const char *who,
                     PagedPools *pools, PagedSeqs *seqs) {
  if (!c || !b) return fail(TB_EINVAL, "%s: null descriptor", who);
  if (c->dtype != TB_F32 && c->dtype != TB_F16 && c->dtype != TB_BF16)
    return fail(TB_EINVAL, "%s: cache dtype %d (fp32, fp16 or bf16)", who, c->dtype);
  if (act_dtype != TB_F32 && act_dtype != c->dtype)
    return fail(TB_EINVAL, "%s: activations are fp32 or of the cache's type", who);
  const int size = dtype_size(c->dtype);
  if (c->page_size <= 0 || (c->page_size & (c->page_size - 1)) != 0)
    return fail(TB_EINVAL, "%s: page_size %d is not a power of two", who, c->page_size);
  if (c->n_pages < 0 || c->n_pages > 0x7FFFFFFF || c->kv_heads <= 0 || c->kv_heads > 4096 || c->head_dim <= 0 ||
      c->head_dim > 4096)
    return fail(TB_EINVAL, "%s: bad cache extents", who);
  const int64_t ext[3] = {c->n_pages, c->page_size, c->kv_heads};
  const int64_t str[3] = {c->page_stride, c->token_stride, c->head_stride};
  for (int i = 0; i < 3; ++i) {
    if (ext[i] <= 1) continue;  // the stride of a single element is never used
    if (str[i] < c->head_dim || str[i] >= (int64_t(1) << 37) || str[i] * size % 16 != 0)
      return fail(TB_EINVAL, "%s: cache strides must cover head_dim and be multiples of 16 bytes", who);
  }
  if (c->n_pages > 0 && (!c->k || !c->v)) return fail(TB_EINVAL, "%s: null pool", who);
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(TB_EINVAL, "%s: the pools must be 16-byte aligned", who);
  if (b->batch < 0 || b->batch > (1 << 20) || b->max_pages < 0 ||
      b->max_pages > (0x7FFFFFFF - 65536) / c->page_size ||  // room to round a length up to a tile
      b->table_stride < b->max_pages)
    return fail(TB_EINVAL, "%s: bad batch extents", who);
  if (b->batch > 0 && (!b->lens || (b->max_pages > 0 && !b->table)))
    return fail(TB_EINVAL, "%s: null lengths or page table", who);
  if (!aligned4(b->lens) || !aligned4(b->table))
    return fail(TB_EINVAL, "%s: lengths and page table must be 4-byte aligned", who);
  *pools = paged_pools(c);
  seqs->lens = b->lens;
  seqs->table = b->table;
  seqs->table_stride = b->table_stride;
  seqs->batch = (int)b->batch;
  seqs->max_len = (int)(b->max_pages * c->page_size);
  return TB_OK;
}

tb_status paged_maps(const tb_paged_cache *c, int rows, const char *who, PagedMaps *maps, int *box_rows) {
  typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                             const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {  // the driver's host-side encoder, looked up once per process
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode) return fail(TB_ECUDA, "%s: the driver has no cuTensorMapEncodeTiled", who);
  const int size = dtype_size(c->dtype);
  const CUtensorMapDataType dt = c->dtype == TB_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : c->dtype == TB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  *box_rows = c->page_size < rows ? c->page_size : rows;
  const uint64_t row = (uint64_t)(c->head_dim * size);
  const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->kv_heads, (cuuint64_t)c->page_size,
                              (cuuint64_t)c->n_pages};
  // the stride of a single element is never used, but has to be a legal one
  const cuuint64_t strides[3] = {c->kv_heads > 1 ? (cuuint64_t)(c->head_stride * size) : row,
                                 c->page_size > 1 ? (cuuint64_t)(c->token_stride * size) : row,
                                 c->n_pages > 1 ? (cuuint64_t)(c->page_stride * size) : row};
  const cuuint32_t box[4] = {(cuuint32_t)(128 / size), 1, (cuuint32_t)*box_rows, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  for (int i = 0; i < 2; ++i) {
    const CUresult r = encode(i ? &maps->v : &maps->k, dt, 4, i ? c->v : c->k, dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TB_ECUDA, "%s: cuTensorMapEncodeTiled: error %d", who, (int)r);
  }
  return TB_OK;
}

namespace {

struct AppendArgs {
  ActRows q, k, v;
  void *q_out;
  int64_t ldq_out;
  int64_t tokens;
  int heads, kv_heads, dim;
  int per_head;   // threads per head, 16 bytes of each half
  int per_token;  // warps per token
  const int32_t *starts;
  const float *cos_t, *sin_t;  // null: no rotation
  int rope_max_seq;
  PagedPools pools;
  PagedSeqs seqs;
};

// E elements (16 bytes of activations) as type DT.
template <int DT, int E>
__device__ __forceinline__ void put(void *p, const float (&f)[E]) {
  if constexpr (DT != TB_F32 && E == 4) {
    float a = f[0], b = f[1], c = f[2], d = f[3];
    const uint32_t lo = pack_rest<DT>(a, b), hi = pack_rest<DT>(c, d);
    *static_cast<uint2 *>(p) = make_uint2(lo, hi);
  } else {
    *static_cast<uint4 *>(p) = Word<DT>::put(f);
  }
}

// ACT, CT: types of the activations and of the cache; U: groups of heads per
// warp, of one token.
template <int ACT, int CT, int U>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a, uint32_t *__restrict__ err) {
  constexpr int AS = Word<ACT>::size, CS = Word<CT>::size;
  constexpr int E = Word<ACT>::n;  // elements of each half of a head per thread
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps = a.tokens * a.per_token;
  const int half = a.dim / 2;
  // a group is 32 / per_head heads; this thread has the same elements of each
  const int span = 32 / a.per_head, sub = lane / a.per_head, i = (lane - sub * a.per_head) * E;
  const int all = sub < span ? a.heads + 2 * a.kv_heads : 0;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < warps; w += (int64_t)gridDim.x * 8) {
    const int64_t t = w / a.per_token;
    const int head0 = (int)(w - t * a.per_token) * span * U + sub;
    uint4 r0[U], r1[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int head = head0 + k * span;
      if (head >= all) continue;
      const ActRows &src = head < a.heads ? a.q : head < a.heads + a.kv_heads ? a.k : a.v;
      const int h = head < a.heads ? head : head < a.heads + a.kv_heads ? head - a.heads : head - a.heads - a.kv_heads;
      const char *at = static_cast<const char *>(src.p) + (t * src.ld + (int64_t)h * a.dim + i) * AS;
      r0[k] = *reinterpret_cast<const uint4 *>(at);
      r1[k] = *reinterpret_cast<const uint4 *>(at + half * AS);
    }
    // the token's sequence: the last b with starts[b] <= t
    int b = (int)t, pos, len;
    bool have = true;
    if (a.starts) {
      int lo = 0, n = a.seqs.batch;  // candidates lo .. lo + n - 1
      while (n > 1) {
        const int step = (n + 31) / 32;
        const int c = lo + lane * step;
        const bool le = c < lo + n && __ldg(a.starts + c) <= t;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
        lo += k * step;
        n = min(step, n - k * step);
      }
      b = lo;
      const int end = __ldg(a.starts + b + 1);
      len = __ldg(a.seqs.lens + b);
      have = t < end && t >= __ldg(a.starts + b);
      pos = (int)((unsigned)len - (unsigned)(end - t));  // (wraps round only where len < 0)
    } else {
      len = __ldg(a.seqs.lens + b);
      have = len != 0;
      pos = (int)((unsigned)len - 1u);
    }
    if (!have) continue;  // an empty slot, or a row behind the last sequence
    bool ok = len >= 0 && pos >= 0 && pos < a.seqs.max_len && (!a.cos_t || pos < a.rope_max_seq);
    int64_t row = -1;
    if (ok) {
      const int32_t id = __ldg(a.seqs.table + (int64_t)b * a.seqs.table_stride + (pos >> a.pools.shift));
      row = row_offset(a.pools, id, pos, 0);
      ok = row >= 0;
    }
    if (!ok) {
      if (lane == 0) atomicOr(err, ERR_INDEX);
      continue;
    }
    float c[E], sn[E];
    if (a.cos_t && head0 < a.heads + a.kv_heads) {
      load_act<E>(a.cos_t, (int64_t)pos * half + i, TB_F32, c);
      load_act<E>(a.sin_t, (int64_t)pos * half + i, TB_F32, sn);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int head = head0 + k * span;
      if (head >= all) continue;
      float x0[E], x1[E];
      Word<ACT>::get(r0[k], x0);
      Word<ACT>::get(r1[k], x1);
      if (a.cos_t && head < a.heads + a.kv_heads) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float y0 = __fmaf_rn(x0[e], c[e], -__fmul_rn(x1[e], sn[e]));
          x1[e] = __fmaf_rn(x0[e], sn[e], __fmul_rn(x1[e], c[e]));
          x0[e] = y0;
        }
      }
      if (head < a.heads) {
        char *d = static_cast<char *>(a.q_out) + (t * a.ldq_out + (int64_t)head * a.dim + i) * AS;
        put<ACT>(d, x0);
        put<ACT>(d + half * AS, x1);
      } else {
        const bool key = head < a.heads + a.kv_heads;
        const int h = head - a.heads - (key ? 0 : a.kv_heads);
        char *d = const_cast<char *>(key ? a.pools.k : a.pools.v) + row + h * a.pools.head_stride + i * CS;
        put<CT>(d, x0);
        put<CT>(d + half * CS, x1);
      }
    }
  }
}

// wave_grid for CTAs of 256 threads, the CTAs per SM found once per kernel and device.
template <auto KERN>
int wave_grid_of(int64_t threads, const DeviceState *st) {
  static std::atomic<int> known[64];
  int n = known[st->device].load(std::memory_order_relaxed);
  if (n == 0) {
    n = resident_ctas(reinterpret_cast<const void *>(KERN), 256, 0);
    known[st->device].store(n, std::memory_order_relaxed);
  }
  return (int)std::min<int64_t>((threads + 255) / 256, (int64_t)st->sm_count * n);
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" tb_status tb_rope_paged_append(const tb_paged_cache *cache, const tb_paged_batch *seqs, int act_dtype,
                                          const void *q_dev, int64_t ldq, const void *k_dev, int64_t ldk,
                                          const void *v_dev, int64_t ldv, int64_t tokens, int64_t heads,
                                          const int32_t *starts_dev, const float *cos_dev, const float *sin_dev,
                                          int64_t rope_max_seq, void *q_out_dev, int64_t ldq_out, tb_stream stream) {
  AppendArgs a = {};
  TB_TRY(paged_args(cache, seqs, act_dtype, "tb_rope_paged_append", &a.pools, &a.seqs));
  const int64_t D = cache->head_dim, KVH = cache->kv_heads;
  if (D % 16 != 0 || D > 256)
    return fail(TB_EINVAL, "tb_rope_paged_append: head_dim %lld (a multiple of 16, at most 256)", (long long)D);
  if (tokens < 0 || tokens > 0x7FFFFFFF || heads < 0 || heads > 65536)
    return fail(TB_EINVAL, "tb_rope_paged_append: bad extents");
  if (!starts_dev && tokens != seqs->batch)
    return fail(TB_EINVAL, "tb_rope_paged_append: without starts, tokens must equal batch");
  if (!aligned4(starts_dev)) return fail(TB_EINVAL, "tb_rope_paged_append: starts must be 4-byte aligned");
  if ((cos_dev == nullptr) != (sin_dev == nullptr))
    return fail(TB_EINVAL, "tb_rope_paged_append: one RoPE table without the other");
  if (cos_dev && (rope_max_seq <= 0 || rope_max_seq > 0x7FFFFFFF))
    return fail(TB_EINVAL, "tb_rope_paged_append: bad table length");
  if (tokens == 0 || seqs->batch == 0) return TB_OK;
  const int as = dtype_size(act_dtype);
  if (!k_dev || !v_dev || (heads > 0 && (!q_dev || !q_out_dev)))
    return fail(TB_EINVAL, "tb_rope_paged_append: null pointer");
  if (ldk < KVH * D || ldv < KVH * D || (heads > 0 && (ldq < heads * D || ldq_out < heads * D)))
    return fail(TB_EINVAL, "tb_rope_paged_append: row strides too small");
  if (!aligned16(k_dev) || !aligned16(v_dev) || ldk * as % 16 != 0 || ldv * as % 16 != 0 ||
      (heads > 0 && (!aligned16(q_dev) || !aligned16(q_out_dev) || ldq * as % 16 != 0 || ldq_out * as % 16 != 0)) ||
      !aligned16(cos_dev) || !aligned16(sin_dev))
    return fail(TB_EINVAL, "tb_rope_paged_append: rows and tables must be 16-byte aligned");
  DeviceState *st;
  TB_TRY(device_state(&st));
  a.q = {q_dev, ldq, act_dtype};
  a.k = {k_dev, ldk, act_dtype};
  a.v = {v_dev, ldv, act_dtype};
  a.q_out = q_out_dev;
  a.ldq_out = ldq_out;
  a.tokens = tokens;
  a.heads = (int)heads;
  a.kv_heads = (int)KVH;
  a.dim = (int)D;
  a.per_head = (int)(D * as / 32);
  a.starts = starts_dev;
  a.cos_t = cos_dev;
  a.sin_t = sin_dev;
  a.rope_max_seq = (int)rope_max_seq;
  // Several groups per warp (four of 16-bit activations, two of fp32) once one per warp would be more than a wave: the
  // lookups are shared and more bytes are in flight.  Measured with one and several: bf16, 12 groups a token, 256 tokens
  // 2.9 and 3.7 us, 700 tokens 5.6 and 4.1, 33k tokens 175 and 125; fp32, 24 groups, 1000 tokens 8.1 and 7.0, 8k tokens
  // 37.6 and 34.9.
  const int span = 32 / a.per_head;
  const int64_t groups = (heads + 2 * KVH + span - 1) / span;
  const bool wide = tokens * groups >= (int64_t)st->sm_count * 32;
  cudaStream_t s = as_stream(stream);
#define TB_APPEND(ACT, CT, U)                                                                                       \
  do {                                                                                                              \
    a.per_token = (int)((groups + U - 1) / U);                                                                      \
    const int ctas = wave_grid_of<paged_append_kernel<ACT, CT, U>>(tokens * a.per_token * 32, st);                  \
    return launch_pdl(paged_append_kernel<ACT, CT, U>, dim3((unsigned)ctas), 256, 0, s, "tb_rope_paged_append", a, \
                      st->err_word);                                                                                \
  } while (0)
  if (act_dtype == TB_F16) {
    if (wide) TB_APPEND(TB_F16, TB_F16, 4);
    TB_APPEND(TB_F16, TB_F16, 1);
  }
  if (act_dtype == TB_BF16) {
    if (wide) TB_APPEND(TB_BF16, TB_BF16, 4);
    TB_APPEND(TB_BF16, TB_BF16, 1);
  }
  if (cache->dtype == TB_F16) {
    if (wide) TB_APPEND(TB_F32, TB_F16, 2);
    TB_APPEND(TB_F32, TB_F16, 1);
  }
  if (cache->dtype == TB_BF16) {
    if (wide) TB_APPEND(TB_F32, TB_BF16, 2);
    TB_APPEND(TB_F32, TB_BF16, 1);
  }
  if (wide) TB_APPEND(TB_F32, TB_F32, 2);
  TB_APPEND(TB_F32, TB_F32, 1);
#undef TB_APPEND
}
