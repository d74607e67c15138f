// tb_paged_attention.cu -- attention of one query token per sequence over a
// paged key/value cache: tb_paged_attention_decode and, for a batch behind a
// common prefix, tb_paged_attention_shared.
//
// Mathematics.  Per sequence b and head: s_t = scale q.k_t, out = sum_t
// exp(s_t - m) v_t / sum_t exp(s_t - m).  Keys are taken tile by tile with the
// running maximum m and sum l, so every key and value is read once; partial
// results (m, l, acc) of key ranges join as acc = sum_i acc_i exp(m_i - M),
// l = sum_i l_i exp(m_i - M), M = max_i m_i, always in the order of the keys.
// Exponents are base 2 (scale * log2 e folded in).
//
// Accuracy.  Both products run on the tensor cores with fp32 accumulation, the
// keys and values as they are stored, queries and probabilities in parts, so
// that no rounding below 22 bits happens before the result's own:
//   fp16 cache  m16n8k16; an fp32 query is hi + lo in fp16 after a power of two
//               per row (fp16's range), a probability times 2^15 likewise
//   bf16 cache  m16n8k16; an fp32 query is three bf16 parts; probabilities
//               three parts with fp32 activations, two with bf16 ones
//   fp32 cache  m16n8k8 in tf32: queries, keys, probabilities and values all
//               as hi + lo (the leading 11 bits and the rest rounded to 11)
// The sixteen rows of the instruction are eight heads twice: row g holds one
// part and row g + 8 the next part of query (or probability) row g, which the
// same thread holds, so a second part costs no instruction where a key/value
// head has at most eight query heads, and their sum is one addition.  16-bit
// queries are exact in one part.  Products are summed inside the tensor core
// over 16 keys and then added to fp32 registers.
//
// Layout.  Each CTA's fifth warp brings tiles of T keys and values into three
// stages of shared memory by TMA, one box per page, 128 bytes of each row,
// swizzled so that every 16-byte fragment load is free of bank conflicts.  Of
// the four other warps HW take eight query heads each, KW = 4 / HW take T / KW
// keys each; each warp keeps its own (m, l, acc), joined once per item.  The
// order of head_dim inside the dot product is chosen so that each thread's
// fragments are whole 16-byte words of a key; 16-bit values are read transposed
// by ldmatrix.
//
// Bytes bound it: keys and values are read once, and four to eight heads leave
// the tensor pipe 86 % idle.  Measured (bf16, 32 heads on 8 of 128): 128
// sequences of up to 8192 keys 316 us, 6.5 TB/s of the measured 6.55; one of
// 131071 keys 93 us, 5.8 TB/s; (fp16 pages, fp32 queries, heads of 64) 32 of up
// to 4096 keys 31.5 us; one of 511 fp32 keys 7.5 to 7.9 us, all of it latency;
// fp32 pages, 128 of up to 4096 keys of 128 370 us, 5.5 TB/s.
//
// Work split.  An item is one (sequence, key/value head, group of 8 HW query
// heads); its unit of work is one tile.  The grid is one wave; CTA c takes the
// units [c U / n, (c + 1) U / n) of all U, found on the device from the
// lengths, so uneven batches and single long sequences fill the GPU alike and a
// captured launch follows the lengths.  Four computing warps per CTA and two or
// three CTAs per SM: a short item's steps (queries, one tile, joining the warps)
// then overlap with other items' (64 sequences of up to 512 keys behind a prefix
// took 37.3 us with the change from one CTA of eight warps, 40.6 before; 34.2
// with what came later).  An item cut by a CTA boundary leaves
// partial results in the workspace; the last of its CTAs to finish (a counter
// per first CTA, reset by that CTA) joins them.  Behind a prefix there are three
// kernels: the prefix's (here, or tb_paged_prefix.cu for many rows), this one
// for the sequences' own keys, and one that joins the parts of each row.  Few
// short sequences: this one joins them itself.  A short prefix: this one alone,
// reading it (from L2) before each sequence's own keys.
#include <algorithm>
#include <atomic>

#include "tb_paged.cuh"

namespace tb {
namespace {

constexpr int kMaxCtas = 448;                    // of a decode launch (counters and partial slots)
// (row, part) pairs behind a prefix that the workspace holds: two parts of every row, and more of them as long as that
// is not much memory.
constexpr int64_t prefix_pairs(int64_t rows) {
  return 2 * rows + 2 * 148 * 128 + (rows < (1 << 17) ? 2 * rows : (1 << 18));
}
constexpr int kWarps = 4;                        // computing warps
constexpr int kThreads = kWarps * 32;            // their threads
constexpr int kBlock = kThreads + 32;            // and one warp that loads
// Splits of a prefix up to which the decode kernel may join them, and with a kernel of its own.  4 sequences of up to 60
// own keys, fp32 pages and heads of 64: behind 300 keys (5 splits) 7.5 and 8.2 us, 1001 (16) 8.8 and 10.4, 2000 (37) 11.0
// and 11.8; bf16 heads of 128: behind 1001 10.0 and 10.8, 2000 (32) 13.7 and 12.8; 17 sequences behind 16387 (37) 48 and
// 34.  So it pays up to 16 everywhere, and from some 32 on only for little data.
constexpr int kJoinSplits = 16;
// ... and tiles of a sequence's own keys: with more of them its items are cut, and the joins in the kernel slow it.  Here
// and there: 4 behind 1001, own keys up to 60 (1 tile) 8.6 and 9.9 us, 200 (4) 11.8 and 11.2, 500 (8) 12.5 and 11.5; 17 x
// 8 heads behind 512, own keys up to 200 14.6 and 15.1, 500 15.8 and 15.2, 777 (13) 23.5 and 15.4.
// (Own keys count as the table has room for: the lengths are on the device.)
constexpr int kJoinTiles = 4;
// A short prefix, of up to so many tiles per item and units of work in all, is read by the decode kernel before each
// sequence's own keys: two launches fewer.  Measured so and with the prefix's kernels: 64 behind 64, 256, 512 and 1024
// keys of 64 (512, 2048, 4096, 8192 units) 15.8 and 21.4, 17.9 and 21.8, 21.5 and 22.6, 29.3 and 25.9 us; 4 with up to 300
// own keys behind 1001 (16 tiles per item) 12.3 and 11.4.
constexpr int kLeadTiles = 8;
constexpr int64_t kLeadUnits = 4096;
// Query rows of a key/value head from which the prefix runs on tcgen05.  There and here: 32 rows behind 8192 keys of 64
// (fp16, fp32 queries) 18.9 and 16.8 us, 36 rows 19.2 and 19.6, 60 rows 19.4 and 20.8; behind 32768 keys of 128 (bf16)
// 46.5 and 44.9, 46.7 and 69.7, 46.7 and 71.6; behind 4096 18.3 and 19.9, 18.5 and 20.0, 18.9 and 22.7.
constexpr int kTensorRows = 33;
constexpr float kLog2e = 1.4426950408889634f;

// x = hi + lo: hi the leading 11 bits (cut off, so that it neither overflows nor
// differs from x in sign: an infinite sum keeps its sign), lo the rest to
// nearest: |x - hi - lo| <= 2^-22 |x|.
__device__ __forceinline__ float tf32_hi(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFFE000u); }
__device__ __forceinline__ float tf32_rn(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return __uint_as_float(r);
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const float (&a)[4], float b0, float b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
        "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

template <int CT>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (CT == TB_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same with nothing to add to.
template <int CT>
__device__ __forceinline__ void mma_16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (CT == TB_F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four 8 x 8 blocks of 16-bit elements, transposed; lane i names row i % 8 of block i / 8.
__device__ __forceinline__ uint4 ldmatrix_t(uint32_t addr) {
  uint4 v;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Where a CTA stands in the list of all units: tile `tile` of item (b, i).
struct Walk {
  int b, i, tile, tiles, len;
};
// What it keeps in shared memory behind the stages and the merge buffer.
constexpr int kMaxStages = 3;
struct Control {
  uint64_t full[kMaxStages], empty[kMaxStages];
  Walk first, item[2];  // the CTA's first item; the computing warps' further ones in turn, the second in item[1]
  int warp_sum[kWarps + 1];
  int last[2];
};

// CT: cache type, D: head_dim, HW: warps across query heads, A32: fp32 activations.
template <int CT_, int D, int HW, bool A32>
struct Cfg {
  static constexpr int CT = CT_;
  // 16-bit caches: instructions per block (each takes two parts of a row)
  static constexpr int QT = CT == TB_BF16 && A32 ? 2 : 1;
  static constexpr int QR = A32 ? 4 : 2;          // registers of a query fragment (16-bit queries: no second part)
  static constexpr float PSCALE = CT == TB_F16 ? 32768.f : 1.f;  // of probabilities, for fp16's range
  static constexpr int EPC = Word<CT>::n;         // elements per 16-byte word
  static constexpr int RB = D * Word<CT>::size;   // bytes per row
  static constexpr int CPR = RB / 16;             // words per row
  static constexpr int T = RB > 256 ? 32 : 64;    // keys per tile
  static constexpr int KW = kWarps / HW;          // warps across keys
  static constexpr int KPW = T / KW;              // keys per warp and tile
  static constexpr int NT = KPW >= 16 ? 2 : 1;    // 8-key blocks per step
  static constexpr int R = 8 * HW;                // rows (query heads) per item
  static constexpr int STAGE = 2 * T * RB;
  // Measured on 32 sequences of up to 32768 keys of 128 bytes (token-major, head-major pages): 4 stages 185, 158 us;
  // 3 stages 171, 152 (fewer rows of different sequences in flight); two CTAs per SM with 6 stages 184, 182.
  static constexpr int STAGES = 3;
  static constexpr int CTAS = RB > 128 ? 2 : 3;   // per SM
  static constexpr int MERGE = kWarps * 8 * (D + 2) * 4;
  static constexpr int SMEM = STAGES * STAGE + MERGE + (int)sizeof(Control);
  static constexpr int JD = D / 4 / EPC;  // 16-byte words of a key per thread
  static constexpr int JV = D / 8 / EPC;  // 16-byte words of a value per thread and key
};

// One warp's queries (A fragments of the first product) and running state.
template <class C, int D>
struct WarpState {
  float qa[C::CT == TB_F32 ? D / 8 : 1][4];
  uint32_t qh[C::CT == TB_F32 ? 1 : D / 16][C::QT][C::QR];
  float scale2;  // scale * log2(e) over the power of two in the queries' row
  float acc[D / 8][2];
  float m, l;
};

__device__ __forceinline__ int atom_add_acq_rel(int *p, int v) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

__device__ __forceinline__ void computing_warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

// Address of 16-byte word w of row `row` of a tile of keys or values.
template <class C>
__device__ __forceinline__ uint32_t word_at(uint32_t tile, int row, int w) {
  return tile + (w >> 3) * (C::T * 128) + row * 128 + (((w ^ row) & 7) << 4);
}

// The queries of this warp's eight rows: row g at element offset `at` (-1:
// none), as loaded (fetch_q, so that a next item's arrive during this one's
// joins) and in parts (load_q).
template <class C>
__device__ __forceinline__ void fetch_q(float (&f)[C::JD][C::EPC], const ActRows &q, int64_t at) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int j = 0; j < C::JD; ++j) {
    const int c = 8 * (j >> 1) + 2 * t + (j & 1);
#pragma unroll
    for (int e = 0; e < C::EPC; ++e) f[j][e] = 0.f;
    if (at >= 0) load_act<C::EPC>(q.p, at + c * C::EPC, C::QR == 4 ? TB_F32 : C::CT, f[j]);
  }
}

template <class C, int D>
__device__ __forceinline__ void load_q(WarpState<C, D> &s, float (&f)[C::JD][C::EPC], float scale2) {
  s.scale2 = scale2;
  if constexpr (C::CT == TB_F16 && C::QR == 4) {
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < C::JD; ++j)
#pragma unroll
      for (int e = 0; e < C::EPC; ++e) mx = fmaxf(mx, fabsf(f[j][e]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int e = fp16_exp(mx);
    const float up = pow2i(e);
    s.scale2 = scale2 * pow2i(-e);
#pragma unroll
    for (int j = 0; j < C::JD; ++j)
#pragma unroll
      for (int k = 0; k < C::EPC; ++k) f[j][k] *= up;
  }
#pragma unroll
  for (int j = 0; j < C::JD; ++j) {
    if constexpr (C::CT == TB_F32) {
#pragma unroll
      for (int e = 0; e < C::EPC / 2; ++e) {
        float(&a)[4] = s.qa[j * (C::EPC / 2) + e];
        a[0] = tf32_hi(f[j][2 * e]);
        a[1] = tf32_rn(f[j][2 * e] - a[0]);
        a[2] = tf32_hi(f[j][2 * e + 1]);
        a[3] = tf32_rn(f[j][2 * e + 1] - a[2]);
      }
    } else {
      // instruction e of a 16-byte word takes its elements 4 e .. 4 e + 3
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int p = 0; p < C::QT; ++p) {
          uint32_t(&a)[C::QR] = s.qh[2 * j + e][p];
          float(&x)[C::EPC] = f[j];
          if constexpr (C::QR == 2) {
            a[0] = pack_rest<C::CT>(x[4 * e], x[4 * e + 1]);
            a[1] = pack_rest<C::CT>(x[4 * e + 2], x[4 * e + 3]);
          } else {
            a[0] = pack_rest<C::CT>(x[4 * e], x[4 * e + 1]);
            a[2] = pack_rest<C::CT>(x[4 * e + 2], x[4 * e + 3]);
            a[1] = pack_rest<C::CT>(x[4 * e], x[4 * e + 1]);
            a[3] = pack_rest<C::CT>(x[4 * e + 2], x[4 * e + 3]);
          }
        }
    }
  }
}

template <class C, int D>
__device__ __forceinline__ void reset(WarpState<C, D> &s) {
  s.m = -INFINITY;
  s.l = 0.f;
#pragma unroll
  for (int j = 0; j < D / 8; ++j) s.acc[j][0] = s.acc[j][1] = 0.f;
}

// This warp's keys of a tile in shared memory: n valid keys in the tile.
template <class C, int D>
__device__ __forceinline__ void warp_tile(WarpState<C, D> &s, uint32_t stage, int n, int kw) {
  constexpr int CT = C::CT;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int STEP = 8 * C::NT;
  const int k0 = kw * C::KPW, k1 = min(n, k0 + C::KPW);
  if (n < C::T && k1 > k0 && (k1 - k0) % STEP != 0) {
    // The rows of the last step behind the sequence's end hold whatever their page held: 0 times that has to be 0.
    // (Warps of other heads that share these keys write the same zeros before their own reads.)
    const int rows = STEP - (k1 - k0) % STEP;
    for (int i = lane; i < rows * C::CPR; i += 32)
      sts128_zero(word_at<C>(stage + C::T * C::RB, k1 + i / C::CPR, i % C::CPR));
    fence_proxy_async_smem();  // before TMA writes this stage again
    __syncwarp();
  }
  for (int k = k0; k < k1; k += STEP) {
    // scores: thread holds keys k + 8 b + 2 t, + 1 of row g (c0, c1: first part of q; c2, c3: second)
    float c[C::NT][4], lo[C::NT][4];  // lo: of fp32 keys' second parts, a chain of its own
#pragma unroll
    for (int b = 0; b < C::NT; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[b][i] = lo[b][i] = 0.f;
#pragma unroll
    for (int j = 0; j < C::JD; ++j) {
      const int w = 8 * (j >> 1) + 2 * t + (j & 1);
      uint4 u[C::NT];
#pragma unroll
      for (int b = 0; b < C::NT; ++b) {
        const int row = k + 8 * b + g;
        u[b] = lds128(word_at<C>(stage, row, w));
      }
      if constexpr (CT == TB_F32) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int b = 0; b < C::NT; ++b) {
            float f[4];
            Word<TB_F32>::get(u[b], f);
            const float(&a)[4] = s.qa[2 * j + e];
            const float h0 = tf32_hi(f[2 * e]), h1 = tf32_hi(f[2 * e + 1]);
            mma_tf32(c[b], a, h0, h1);
            mma_tf32(lo[b], a, tf32_rn(f[2 * e] - h0), tf32_rn(f[2 * e + 1] - h1));
          }
      } else {
#pragma unroll
        for (int p = 0; p < C::QT; ++p)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int b = 0; b < C::NT; ++b) {
              const uint32_t(&q)[C::QR] = s.qh[2 * j + e][p];
              uint32_t a[4];
              if constexpr (C::QR == 2) a[0] = q[0], a[1] = 0u, a[2] = q[1], a[3] = 0u;
              else a[0] = q[0], a[1] = q[1], a[2] = q[2], a[3] = q[3];
              mma_16<CT>(c[b], a, e ? u[b].z : u[b].x, e ? u[b].w : u[b].y);
            }
      }
    }
    float p[C::NT][2];
    float mx = -INFINITY;
#pragma unroll
    for (int b = 0; b < C::NT; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = C::QR == 4 ? c[b][i] + c[b][i + 2] : c[b][i];
        if (CT == TB_F32) v += lo[b][i] + lo[b][i + 2];
        v *= s.scale2;
        p[b][i] = k + 8 * b + 2 * t + i < n ? v : -INFINITY;
        mx = fmaxf(mx, p[b][i]);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m = fmaxf(s.m, mx);
    const float ms = m == -INFINITY ? 0.f : m;  // all scores -inf so far: exp2(-inf - 0) = 0, not NaN
    const float alpha = ex2(s.m - ms);
    s.m = m;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < C::NT; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[b][i] = ex2(p[b][i] - ms);
        sum += p[b][i];
      }
    s.l = fmaf(s.l, alpha, sum);
    // acc = acc alpha + p V
    const uint32_t vt = stage + C::T * C::RB;
    if constexpr (CT == TB_F32) {
      // the instruction's k index t is key 2 t, t + 4 is key 2 t + 1; output column n of block (j, e) is element
      // (n + 8 j) EPC + e
      float pa[C::NT][4];
#pragma unroll
      for (int b = 0; b < C::NT; ++b) {
        pa[b][0] = tf32_hi(p[b][0]);
        pa[b][1] = tf32_rn(p[b][0] - pa[b][0]);
        pa[b][2] = tf32_hi(p[b][1]);
        pa[b][3] = tf32_rn(p[b][1] - pa[b][2]);
      }
#pragma unroll
      for (int j = 0; j < C::JV; ++j) {
        float f[C::NT][2][4];
#pragma unroll
        for (int b = 0; b < C::NT; ++b)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = k + 8 * b + 2 * t + i;
            Word<TB_F32>::get(lds128(word_at<C>(vt, row, g + 8 * j)), f[b][i]);
          }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int b = 0; b < C::NT; ++b) {
            const float h0 = tf32_hi(f[b][0][e]), h1 = tf32_hi(f[b][1][e]);
            mma_tf32(o, pa[b], h0, h1);
            mma_tf32(o, pa[b], tf32_rn(f[b][0][e] - h0), tf32_rn(f[b][1][e] - h1));
          }
          float(&r)[2] = s.acc[j * 4 + e];
          r[0] = fmaf(r[0], alpha, o[0] + o[2]);
          r[1] = fmaf(r[1], alpha, o[1] + o[3]);
        }
      }
    } else {
      uint32_t pa[C::QT][4];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) p[b][i] *= C::PSCALE;
#pragma unroll
      for (int q = 0; q < C::QT; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int b = 0; b < 2; ++b) pa[q][2 * b + h] = pack_rest<CT>(p[b][0], p[b][1]);
      const int row = k + (lane & 15);  // blocks: keys 0-7, 8-15 of word w, then of word w + 1
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int w = 2 * j + (lane >> 4);
        const uint4 v = ldmatrix_t(word_at<C>(vt, row, w));
        float o[2][4];
        mma_16_first<CT>(o[0], pa[0], v.x, v.y);
        mma_16_first<CT>(o[1], pa[0], v.z, v.w);
#pragma unroll
        for (int q = 1; q < C::QT; ++q) {
          mma_16<CT>(o[0], pa[q], v.x, v.y);
          mma_16<CT>(o[1], pa[q], v.z, v.w);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float(&r)[2] = s.acc[2 * j + h];
          r[0] = fmaf(r[0], alpha, o[h][0] + o[h][2]);
          r[1] = fmaf(r[1], alpha, o[h][1] + o[h][3]);
        }
      }
    }
  }
}

// Leaves the warp's (m, l, acc) in the merge buffer: acc[kWarps][8 rows][D],
// then ml[kWarps][8].
template <class C, int D>
__device__ __forceinline__ void leave(const WarpState<C, D> &s, float *merge) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float l = s.l;
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  float *row = merge + (warp * 8 + g) * D;
  if constexpr (C::CT == TB_F32) {
#pragma unroll
    for (int j = 0; j < C::JV; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < C::EPC; ++e) row[(2 * t + i + 8 * j) * C::EPC + e] = s.acc[j * C::EPC + e][i];
  } else {
    constexpr float down = 1.f / C::PSCALE;
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
      *reinterpret_cast<float2 *>(row + 8 * j + 2 * t) = make_float2(s.acc[j][0] * down, s.acc[j][1] * down);
  }
  if (t == 0) reinterpret_cast<float2 *>(merge + kWarps * 8 * D)[warp * 8 + g] = make_float2(s.m, l);
}

// Running join of partial results of one row, N of its elements per thread.
template <int N>
struct Join {
  float m = -INFINITY, l = 0.f, acc[N];
  __device__ __forceinline__ Join() {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
  }
  template <class Get>
  __device__ __forceinline__ void add(float2 ml, Get get) {
    const float mn = fmaxf(m, ml.x);
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float a = ex2(m - ms), w = ex2(ml.x - ms);
    m = mn;
    l = fmaf(l, a, ml.y * w);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(acc[i], a, get(i) * w);
  }
};

// The warps' results of row `row` of an item, joined; thread `sub` of TPR
// takes elements sub + TPR i.
template <class C, int D, int N>
__device__ __forceinline__ void join_warps(Join<N> &j, const float *merge, int row, int sub) {
  constexpr int TPR = kThreads / C::R;
  const int hw = row >> 3, g = row & 7;
  const float2 *ml = reinterpret_cast<const float2 *>(merge + kWarps * 8 * D);
#pragma unroll
  for (int kw = 0; kw < C::KW; ++kw) {
    const int w = kw * (kWarps / C::KW) + hw;  // warp index: kw HW + hw
    const float *a = merge + (w * 8 + g) * D + sub;
    j.add(ml[w * 8 + g], [&](int i) { return a[i * TPR]; });
  }
}

template <class C>
__device__ __forceinline__ int tiles_of(const AttnArgs &a, int len) {
  return max(1, a.lead + (len + C::T - 1) / C::T);
}

__device__ __forceinline__ int seq_len(const PagedSeqs &s, int b) {
  const int len = s.lens[b];
  return len < 0 || len > s.max_len ? 0 : len;
}

// JOIN: it joins a prefix's parts itself (a variant, since the code for it costs the others registers: 128 ragged
// sequences 356 us with it, 322 without).
template <int CT, int D, int HW, bool A32, bool JOIN>
__global__ void __launch_bounds__(kBlock, Cfg<CT, D, HW, A32>::CTAS)
    paged_decode_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                        uint32_t *__restrict__ err) {
  using C = Cfg<CT, D, HW, A32>;
  extern __shared__ __align__(1024) unsigned char smem[];
  float *merge = reinterpret_cast<float *>(smem + C::STAGES * C::STAGE);
  Control &ctl = *reinterpret_cast<Control *>(smem + C::STAGES * C::STAGE + C::MERGE);
  const uint32_t stages = smem_addr(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int items = a.kv_heads * a.head_groups;
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], kWarps);
    }
    fence_mbar_init();
  }
  if (tid == kThreads) {
    prefetch_map(&km);
    prefetch_map(&vm);
  }

  // Behind a prefix the kernel before this one is the prefix's, whose results this one does not read: it is waited for
  // only at the end, so that this kernel's end implies it (waited for here: 4 sequences behind 1001 keys 11.9 us instead
  // of 8.2, 128 behind 32768 112 instead of 107).  Lengths, tables, pages and queries may be what any earlier kernel
  // wrote: plain loads of them, since they are ordered by the acquire.
  pdl_launch_dependents();
  if (a.prefix.splits == 0 || !earlier_kernels_seen(a.prefix)) pdl_wait();

  // ---- the units of all sequences, and this CTA's share of them: U / n for each of n CTAs, one more for the first
  // U % n (the host has made sure that U < 2^31)
  const int per = (a.seqs.batch + kBlock - 1) / kBlock;
  const int b0 = min(a.seqs.batch, tid * per), b1 = min(a.seqs.batch, b0 + per);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = a.seqs.lens[b];
    if (blockIdx.x == 0 && (len < 0 || len > a.seqs.max_len)) atomicOr(err, ERR_INDEX);
    mine += tiles_of<C>(a, seq_len(a.seqs, b)) * items;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) ctl.warp_sum[warp] = incl;
  __syncthreads();
  int before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w <= kWarps; ++w) {
    if (w < warp) before += ctl.warp_sum[w];
    total += ctl.warp_sum[w];
  }
  const int n_ctas = min(a.max_ctas, total), me = blockIdx.x;
  if (me >= n_ctas) {
    pdl_wait();
    return;
  }
  const int share = total / n_ctas, more = total - share * n_ctas;
  auto first_unit = [&](int c) { return c * share + min(c, more); };
  auto owner = [&](int u) {
    const int x = u - more * (share + 1);
    return x < 0 ? u / (share + 1) : more + x / share;
  };
  // the item after w's, whose sequence, where it is the next one, has next_len keys
  auto following = [&](Walk w, int next_len) {
    w.tile = 0;
    if (++w.i == items) w = {w.b + 1, 0, 0, tiles_of<C>(a, next_len), next_len};
    return w;
  };
  const int u0 = first_unit(me), u1 = first_unit(me + 1);
  if (u0 >= before && u0 < before + mine) {
    int u = u0 - before;
    for (int b = b0;; ++b) {
      const int len = seq_len(a.seqs, b), tiles = tiles_of<C>(a, len);
      const int n = tiles * items;
      if (u < n) {
        const int i = u / tiles;
        const Walk w = {b, i, u - i * tiles, tiles, len};
        ctl.first = w;
        ctl.item[1] = following(w, b + 1 < a.seqs.batch ? seq_len(a.seqs, b + 1) : 0);
        break;
      }
      u -= n;
    }
  }
  __syncthreads();
  Walk cur = ctl.first;
  bool dead = begin_dead(a.wait_ns, err);

  if (warp == kWarps) {  // ---- the loading warp
    int stage = 0, u = u0;
    uint32_t phase = 1;  // the stages begin empty
    asm volatile("fence.proxy.async.global;" ::: "memory");  // the pages' writers, seen by this warp, are seen by its copies
    int next_len = cur.b + 1 < a.seqs.batch ? seq_len(a.seqs, cur.b + 1) : 0;
    for (; u < u1; ++u) {
      const bool own = cur.tile >= a.lead;
      const int32_t *table = own ? a.seqs.table + (int64_t)cur.b * a.seqs.table_stride : a.prefix_table;
      const int tile = own ? cur.tile - a.lead : cur.tile;
      const TileBoxes box =  // before the wait
          tile_boxes<C::T>(a.pools, a.box_shift, table, own ? cur.len : a.prefix_len, tile);
      wait_phase(&ctl.empty[stage], phase, err, dead, a.wait_ns);
      if (__any_sync(0xffffffffu, dead)) break;
      load_rows<C::T, C::RB, Word<CT>::size>(stages + (uint32_t)stage * C::STAGE, &ctl.full[stage], &km, &vm, a.pools,
                                             a.box_shift, table, box, tile, cur.i / a.head_groups, err);
      if (++stage == C::STAGES) stage = 0, phase ^= 1;
      if (++cur.tile < cur.tiles) continue;
      cur = following(cur, next_len);
      if (cur.i == 0 && cur.b + 1 < a.seqs.batch) next_len = seq_len(a.seqs, cur.b + 1);
    }
    wait_copies<C::STAGES>(ctl.full, u - u0, err);
    pdl_wait();
    if (JOIN && me == 0 && lane == 0) *a.prefix.begun = 0;  // (a CTA that has yet to look will wait)
    return;
  }

  // ---- the computing warps
  const int hw = warp % HW, kw = warp / HW;
  constexpr int TPR = kThreads / C::R, N = D / TPR;
  const int row = tid / TPR, sub = tid % TPR;  // this thread's share of a join
  auto q_at = [&](const Walk &w) -> int64_t {
    const int kvh = w.i / a.head_groups, gi = (w.i - kvh * a.head_groups) * C::R + hw * 8 + (lane >> 2);
    return gi < a.group ? (int64_t)w.b * a.q.ld + (int64_t)(kvh * a.group + gi) * D : -1;
  };
  // results of a row of item `w`, elements e, e + step, ...: its output, joined with the prefix's parts first, or its
  // part of it
  auto put = [&](const Walk &w, int gi, int e, int step, auto &j) {
    constexpr int n = sizeof(j.acc) / sizeof(float);
    const int kvh = w.i / a.head_groups;
    if constexpr (JOIN) pdl_wait();
    if (gi >= a.group) return;
    const int64_t at_parts = ((int64_t)kvh * a.prefix.rows + (int64_t)w.b * a.group + gi) * a.prefix.parts;
    if constexpr (JOIN) {
      constexpr int P = n >= 16 ? 2 : 32 / n;
      for (int p0 = 0; p0 < a.prefix.splits; p0 += P) {
        float2 ml[P];
        float v[P][n];
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (p0 + p >= a.prefix.splits) continue;
          ml[p] = __ldcg(a.prefix.ml + at_parts + p0 + p);
#pragma unroll
          for (int i = 0; i < n; ++i) v[p][i] = __ldcg(a.prefix.acc + (at_parts + p0 + p) * D + e + i * step);
        }
#pragma unroll
        for (int p = 0; p < P; ++p)
          if (p0 + p < a.prefix.splits) j.add(ml[p], [&](int i) { return v[p][i]; });
      }
    } else if (a.prefix.splits > 0) {
      const int64_t at = at_parts + a.prefix.splits;
#pragma unroll
      for (int i = 0; i < n; ++i) a.prefix.acc[at * D + e + i * step] = j.acc[i];
      if (e == 0) a.prefix.ml[at] = make_float2(j.m, j.l);
      return;
    }
    const bool none = w.len == 0 && a.prefix_len == 0;
    const int64_t at = (int64_t)w.b * a.ldo + (int64_t)(kvh * a.group + gi) * D + e;
#pragma unroll
    for (int i = 0; i < n; ++i)
      store_act1(a.out, at + i * step, A32 ? TB_F32 : CT, none ? 0.f : __fdiv_rn(j.acc[i], j.l));
  };
  WarpState<C, D> s;
  float qf[C::JD][C::EPC];
  fetch_q<C>(qf, a.q, q_at(cur));
  int stage = 0;
  uint32_t phase = 0;
  // the items that this CTA shares with others: its first, begun before u0, and its last, unfinished at u1
  Walk cut[2];
  int cut_unit[2] = {-1, -1};  // the item's first unit
  // The items after the first are found by the first warp, one ahead of their use, and read behind the barrier of a join:
  // all warps agree on them whatever became of the tiles.
  int odd = 0, next_len = 0;  // parity of this item; keys of the sequence behind the next item's
  if (warp == 0 && ctl.item[1].b + 1 < a.seqs.batch) next_len = seq_len(a.seqs, ctl.item[1].b + 1);
  for (int u = u0; u < u1; odd ^= 1) {
    const Walk item = cur;
    const int item0 = u - item.tile, end = min(u1, item0 + item.tiles);
    if (!JOIN && a.prefix.splits > 0 && tid == 0 && item0 >= u0)
      a.prefix.own[(int64_t)item.b * items + item.i] =
          make_int2(2 * me + 1, item0 + item.tiles <= u1 ? 0 : owner(item0 + item.tiles - 1) - me + 1);
    reset(s);
    load_q(s, qf, a.scale2);
    for (; u < end; ++u) {
      wait_phase(&ctl.full[stage], phase, err, dead, a.wait_ns);
      const int tile = u - item0 - a.lead;  // of the sequence's own; below 0 of the prefix
      const int keys = tile < 0 ? a.prefix_len - (tile + a.lead) * C::T : item.len - tile * C::T;
      warp_tile(s, stages + (uint32_t)stage * C::STAGE, min(C::T, keys), kw);
      __syncwarp();
      if (lane == 0 && !dead) mbar_arrive(&ctl.empty[stage]);
      if (++stage == C::STAGES) stage = 0, phase ^= 1;
    }
    if (u < u1) {  // the next item's queries arrive during this one's joins
      cur = ctl.item[odd ^ 1];
      fetch_q<C>(qf, a.q, q_at(cur));
      if (warp == 0) {
        const Walk w = following(cur, next_len);
        if (lane == 0) ctl.item[odd] = w;
        if (w.i == 0 && w.b + 1 < a.seqs.batch) next_len = seq_len(a.seqs, w.b + 1);
      }
    }
    leave(s, merge);
    computing_warps_sync();
    Join<N> j;
    join_warps<C, D>(j, merge, row, sub);
    if (item0 >= u0 && item0 + item.tiles <= u1) {
      put(item, (item.i % a.head_groups) * C::R + row, sub, TPR, j);
    } else {
      const int k = item0 < u0 ? 0 : 1;
      const int64_t slot = 2 * me + k;
      float *acc = a.slot_acc + (slot * C::R + row) * D + sub;
#pragma unroll
      for (int i = 0; i < N; ++i) __stcg(acc + i * TPR, j.acc[i]);
      if (sub == 0) __stcg(a.slot_ml + slot * C::R + row, make_float2(j.m, j.l));
      cut[k] = item;
      cut_unit[k] = item0;
    }
    computing_warps_sync();  // the merge buffer has been read
  }

  // ---- the cut items: whoever of its CTAs comes last joins one (behind a prefix the next kernel does, JOIN apart)
  if ((cut_unit[0] < 0 && cut_unit[1] < 0) || (!JOIN && a.prefix.splits > 0)) {
    pdl_wait();
    return;
  }
  if (tid < 2) {  // (the barrier above ordered the CTA's partial results before this)
    const int unit = tid ? cut_unit[1] : cut_unit[0], tiles = tid ? cut[1].tiles : cut[0].tiles;
    int last = 0;
    if (unit >= 0) {
      const int c0 = owner(unit), parts = owner(unit + tiles - 1) - c0 + 1;
      if (atom_add_acq_rel(a.counters + c0, 1) == parts - 1) {
        a.counters[c0] = 0;  // ready for the next launch
        last = parts;
      }
    }
    ctl.last[tid] = last;
  }
  computing_warps_sync();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int parts = ctl.last[k];  // 0: not the last
    if (parts == 0) continue;
    const int c0 = owner(cut_unit[k]);
    // CTA c's slot: its first item's where the item began before it
    auto slot = [&](int p) { return (int64_t)(2 * (c0 + p) + (cut_unit[k] < first_unit(c0 + p) ? 0 : 1)) * C::R; };
    const int hg = cut[k].i % a.head_groups, rows = min(C::R, a.group - hg * C::R);
    // four elements of a row per thread; eight parts' loads at a time, joined in their order
    for (int x = tid; x < rows * (D / 4); x += kThreads) {
      const int r = x / (D / 4), e = x % (D / 4) * 4;
      Join<4> j;
      for (int p0 = 0; p0 < parts; p0 += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          if (p0 + p >= parts) continue;
          const int64_t at = slot(p0 + p) + r;
          ml[p] = __ldcg(a.slot_ml + at);
          v[p] = __ldcg(reinterpret_cast<const float4 *>(a.slot_acc + at * D + e));
        }
#pragma unroll
        for (int p = 0; p < 8; ++p)
          if (p0 + p < parts) j.add(ml[p], [&](int i) { return i == 0 ? v[p].x : i == 1 ? v[p].y : i == 2 ? v[p].z : v[p].w; });
      }
      put(cut[k], hg * C::R + r, e, 1, j);
    }
  }
  pdl_wait();
}

// The prefix: item (row tile, split, key/value head), rows = the queries of all
// sequences' heads of that key/value head, R of them per CTA.
template <int CT, int D, int HW, bool A32>
__global__ void __launch_bounds__(kBlock, Cfg<CT, D, HW, A32>::CTAS)
    paged_prefix_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                        uint32_t *__restrict__ err) {
  using C = Cfg<CT, D, HW, A32>;
  extern __shared__ __align__(1024) unsigned char smem[];
  float *merge = reinterpret_cast<float *>(smem + C::STAGES * C::STAGE);
  Control &ctl = *reinterpret_cast<Control *>(smem + C::STAGES * C::STAGE + C::MERGE);
  const uint32_t stages = smem_addr(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], kWarps);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  if (tid == 0) let_next_begin(a.prefix);
  const int split = blockIdx.y, rt = blockIdx.x, kvh = blockIdx.z;
  const int tiles = (a.prefix_len + C::T - 1) / C::T;
  const int t0 = (int)((int64_t)split * tiles / a.prefix.splits);
  const int t1 = (int)((int64_t)(split + 1) * tiles / a.prefix.splits);
  bool dead = begin_dead(a.wait_ns, err);
  if (warp == kWarps) {
    int stage = 0, t = t0;
    uint32_t phase = 1;
    for (; t < t1; ++t) {
      wait_phase(&ctl.empty[stage], phase, err, dead, a.wait_ns);
      if (__any_sync(0xffffffffu, dead)) break;
      load_rows<C::T, C::RB, Word<CT>::size>(
          stages + (uint32_t)stage * C::STAGE, &ctl.full[stage], &km, &vm, a.pools, a.box_shift, a.prefix_table,
          tile_boxes<C::T>(a.pools, a.box_shift, a.prefix_table, a.prefix_len, t), t, kvh, err);
      if (++stage == C::STAGES) stage = 0, phase ^= 1;
    }
    wait_copies<C::STAGES>(ctl.full, t - t0, err);
    return;
  }
  const int hw = warp % HW, kw = warp / HW;
  WarpState<C, D> s;
  reset(s);
  {
    const int row = rt * C::R + hw * 8 + (lane >> 2), b = row / a.group;
    float f[C::JD][C::EPC];
    fetch_q<C>(f, a.q,
               row < a.prefix.rows ? (int64_t)b * a.q.ld + (int64_t)(kvh * a.group + row - b * a.group) * D : -1);
    load_q(s, f, a.scale2);
  }
  int stage = 0;
  uint32_t phase = 0;
  for (int t = t0; t < t1; ++t) {
    wait_phase(&ctl.full[stage], phase, err, dead, a.wait_ns);
    warp_tile(s, stages + (uint32_t)stage * C::STAGE, min(C::T, a.prefix_len - t * C::T), kw);
    __syncwarp();
    if (lane == 0 && !dead) mbar_arrive(&ctl.empty[stage]);
    if (++stage == C::STAGES) stage = 0, phase ^= 1;
  }
  leave(s, merge);
  computing_warps_sync();
  constexpr int TPR = kThreads / C::R, N = D / TPR;
  const int r = tid / TPR, sub = tid % TPR, row = rt * C::R + r;
  if (row >= a.prefix.rows) return;
  Join<N> j;
  join_warps<C, D>(j, merge, r, sub);
  const int64_t at = ((int64_t)kvh * a.prefix.rows + row) * a.prefix.parts + split;
#pragma unroll
  for (int i = 0; i < N; ++i) a.prefix.acc[at * D + sub + i * TPR] = j.acc[i];
  if (sub == 0) a.prefix.ml[at] = make_float2(j.m, j.l);
}

// The outputs behind a prefix: a warp per row joins the prefix's parts and then
// its own keys', in order, P parts' loads at a time: 16 up to eight rows per SM,
// 8 beyond (fewer registers, more warps).  Measured 16 and 8: 544 rows of 38 parts
// 28.8 and 30.7 us for the whole call, 2048 rows of 19 parts 37.2 and 34.3.
template <int D, int P>
__global__ void __launch_bounds__(256) paged_combine_kernel(const AttnArgs a, int heads) {
  constexpr int E = D / 32;  // elements per lane
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.prefix.begun = 0;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);  // b * heads + h
  if (row >= (int64_t)a.seqs.batch * heads) return;
  const int b = (int)(row / heads), h = (int)(row - (int64_t)b * heads), kvh = h / a.group, gi = h - kvh * a.group;
  const int hg = gi / a.prefix.slot_rows;
  const int2 own = __ldcg(a.prefix.own + ((int64_t)b * a.kv_heads + kvh) * a.head_groups + hg);
  Join<E> j;
  // parts 0 .. n - 1, part p at index at(p) of acc and ml
  auto join = [&](const float *acc, const float2 *ml, int n, auto at) {
    for (int p0 = 0; p0 < n; p0 += P) {
      float2 m[P];
      float v[P][E];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (p0 + p >= n) continue;
        const int64_t i = at(p0 + p);
        m[p] = __ldcg(ml + i);
        const float *from = acc + i * D + lane * E;
        if constexpr (E == 2) {
          const float2 x = __ldcg(reinterpret_cast<const float2 *>(from));
          v[p][0] = x.x, v[p][1] = x.y;
        } else {
          const float4 x = __ldcg(reinterpret_cast<const float4 *>(from));
          v[p][0] = x.x, v[p][1] = x.y, v[p][2] = x.z, v[p][3] = x.w;
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (p0 + p < n) j.add(m[p], [&](int i) { return v[p][i]; });
    }
  };
  const int64_t at = ((int64_t)kvh * a.prefix.rows + (int64_t)b * a.group + gi) * a.prefix.parts;
  join(a.prefix.acc, a.prefix.ml, a.prefix.splits + (own.y == 0), [&](int p) { return at + p; });
  // CTA c's slot 2 c + 1 where the item begins in it, the others' slot 2 c
  const int r = gi - hg * a.prefix.slot_rows;
  join(a.slot_acc, a.slot_ml, own.y,
       [&](int p) { return (int64_t)(own.x + (p ? 2 * p - 1 : 0)) * a.prefix.slot_rows + r; });
  const int64_t to = (int64_t)b * a.ldo + (int64_t)h * D + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) store_act1(a.out, to + i, a.q.dtype, __fdiv_rn(j.acc[i], j.l));
}

// Warps across query heads: the fewest that take the rows in one item, so that
// as many warps as possible split the keys (up to 8 rows 1, 16: 2, 32: 4).
int head_warps(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

struct Layout {
  size_t slot_acc, slot_ml, prefix_acc, prefix_ml, own, bytes;
};
Layout layout_of(int64_t batch, int64_t heads, int64_t kv_heads, int64_t D) {
  const size_t slots = 2 * kMaxCtas * 8 * (size_t)head_warps(heads / kv_heads);
  const size_t rows = (size_t)prefix_pairs(batch * heads);
  Layout l;
  l.slot_acc = up256((kMaxCtas + 1) * sizeof(int));  // the counters and prefix.begun
  l.slot_ml = l.slot_acc + up256(slots * D * sizeof(float));
  l.prefix_acc = l.slot_ml + up256(slots * sizeof(float2));
  l.prefix_ml = l.prefix_acc + up256(rows * D * sizeof(float));
  l.own = l.prefix_ml + up256(rows * sizeof(float2));
  l.bytes = l.own + up256((size_t)(batch * heads) * sizeof(int2));
  return l;
}

// CTAs of a kernel in one wave of the current device, its shared memory limit raised; found once per device.
template <class C, auto KERN>
tb_status wave_of(const DeviceState *st, int *ctas) {
  static std::atomic<int> known[64];
  int n = known[st->device].load(std::memory_order_acquire);
  if (n == 0) {
    TB_TRY(ensure_smem_for(KERN, C::SMEM));
    n = st->sm_count * resident_ctas(reinterpret_cast<const void *>(KERN), kBlock, C::SMEM);
    known[st->device].store(n, std::memory_order_release);
  }
  *ctas = n;
  return TB_OK;
}

template <int CT, int D, int HW, bool A32>
tb_status launch_decode(AttnArgs &a, const PagedMaps &maps, const DeviceState *st, cudaStream_t s, const char *who) {
  using C = Cfg<CT, D, HW, A32>;
  int ctas;
  TB_TRY((wave_of<C, paged_decode_kernel<CT, D, HW, A32, false>>(st, &ctas)));
  a.max_ctas = std::min(ctas, kMaxCtas);
  a.prefix.join_here = a.prefix.splits > 0 && a.prefix.splits <= kJoinSplits && a.prefix.few;
  if (a.prefix.join_here) {
    TB_TRY((wave_of<C, paged_decode_kernel<CT, D, HW, A32, true>>(st, &ctas)));
    a.max_ctas = std::min(ctas, kMaxCtas);
    return launch_pdl(paged_decode_kernel<CT, D, HW, A32, true>, dim3((unsigned)a.max_ctas), kBlock, C::SMEM, s, who, a,
                      maps.k, maps.v, st->err_word);
  }
  return launch_pdl(paged_decode_kernel<CT, D, HW, A32, false>, dim3((unsigned)a.max_ctas), kBlock, C::SMEM, s, who, a,
                    maps.k, maps.v, st->err_word);
}

template <int CT, int D, int HW, bool A32>
tb_status launch_prefix(AttnArgs &a, const PagedMaps &maps, const DeviceState *st, cudaStream_t s, const char *who) {
  using C = Cfg<CT, D, HW, A32>;
  constexpr auto kern = paged_prefix_kernel<CT, D, HW, A32>;
  int ctas;
  TB_TRY((wave_of<C, paged_prefix_kernel<CT, D, HW, A32>>(st, &ctas)));
  const int row_tiles = (a.prefix.rows + C::R - 1) / C::R;
  const int64_t items = (int64_t)row_tiles * a.kv_heads;
  const int tiles = (a.prefix_len + C::T - 1) / C::T;
  set_prefix_splits(a, items, tiles, ctas);
  return launch_pdl(kern, dim3((unsigned)row_tiles, (unsigned)a.prefix.splits, (unsigned)a.kv_heads), kBlock, C::SMEM, s,
                    who, a, maps.k, maps.v, st->err_word);
}

template <int CT, int D, bool A32>
tb_status run(AttnArgs &a, const tb_paged_cache *cache, const DeviceState *st, cudaStream_t s, const char *who) {
  // every kernel here takes tiles of as many keys (one warp's 16 and more; 8 of 512 bytes)
  constexpr int T = Cfg<CT, D, 1, A32>::T;
  PagedMaps maps;
  int box;
  tb_paged_cache c = *cache;
  if (c.n_pages == 0) c.n_pages = 1, c.k = c.v = a.counters;  // an empty pool: every page id is outside it
  TB_TRY(paged_maps(&c, T, who, &maps, &box));
  a.box_shift = 0;
  while ((1 << a.box_shift) < box) ++a.box_shift;
  const int hw = head_warps(a.group);
  a.head_groups = (a.group + 8 * hw - 1) / (8 * hw);
  a.prefix.slot_rows = 8 * hw;
  const int64_t lead = (a.prefix_len + T - 1) / T;
  const int64_t items = (int64_t)a.seqs.batch * a.kv_heads * a.head_groups;
  const int64_t own = (a.seqs.max_len + T - 1) / T;  // tiles of a sequence at most
  a.prefix.few = items <= st->sm_count && own <= kJoinTiles;
  if (!a.prefix.few && lead <= kLeadTiles && lead * items <= kLeadUnits) {
    a.lead = (int)lead;
  } else if (lead > 0 && CT != TB_F32 && a.prefix.rows >= kTensorRows) {
    TB_TRY(launch_prefix_tc(a, maps, CT, D, st, s, who));
  } else if (lead > 0) {
    switch (head_warps(a.prefix.rows)) {
      case 1: TB_TRY((launch_prefix<CT, D, 1, A32>(a, maps, st, s, who))); break;
      case 2: TB_TRY((launch_prefix<CT, D, 2, A32>(a, maps, st, s, who))); break;
      default: TB_TRY((launch_prefix<CT, D, 4, A32>(a, maps, st, s, who))); break;
    }
  }
  switch (hw) {
    case 1: TB_TRY((launch_decode<CT, D, 1, A32>(a, maps, st, s, who))); break;
    case 2: TB_TRY((launch_decode<CT, D, 2, A32>(a, maps, st, s, who))); break;
    default: TB_TRY((launch_decode<CT, D, 4, A32>(a, maps, st, s, who))); break;
  }
  if (a.prefix.splits == 0 || a.prefix.join_here) return TB_OK;
  const int heads = a.kv_heads * a.group;
  const int64_t rows = (int64_t)a.seqs.batch * heads;
  auto combine = rows <= 8 * st->sm_count ? paged_combine_kernel<D, 16> : paged_combine_kernel<D, 8>;
  return launch_pdl(combine, dim3((unsigned)((rows + 7) / 8)), 256, 0, s, who, a, heads);
}

tb_status attention(const tb_paged_cache *cache, const tb_paged_batch *seqs, const int32_t *prefix_table,
                    int64_t prefix_len, int act_dtype, const void *q, int64_t ldq, int64_t heads, float scale,
                    void *out, int64_t ldo, void *ws, size_t ws_bytes, cudaStream_t stream, const char *who) {
  AttnArgs a = {};
  TB_TRY(paged_args(cache, seqs, act_dtype, who, &a.pools, &a.seqs));
  const int64_t D = cache->head_dim, KVH = cache->kv_heads, B = seqs->batch;
  if (D != 64 && D != 128) return fail(TB_EINVAL, "%s: head_dim %lld (64 or 128)", who, (long long)D);
  if (heads <= 0 || heads > 65536 || heads % KVH != 0)
    return fail(TB_EINVAL, "%s: heads must be a positive multiple of kv_heads", who);
  if (B * heads > (1 << 24)) return fail(TB_EINVAL, "%s: more than 2^24 query rows", who);
  if (prefix_len < 0 || prefix_len > 0x7FFFFFFF - 65536) return fail(TB_EINVAL, "%s: bad prefix length", who);
  if (B * heads * (a.seqs.max_len / 32 + 1) > 0x7FFFFFFF - kLeadUnits)  // units of work at most
    return fail(TB_EINVAL, "%s: batch * heads * max_pages * page_size is too large (2^36)", who);
  if (B == 0) return TB_OK;
  if (!q || !out || !ws || (prefix_len > 0 && !prefix_table)) return fail(TB_EINVAL, "%s: null pointer", who);
  if (!aligned4(prefix_table)) return fail(TB_EINVAL, "%s: the prefix's pages must be 4-byte aligned", who);
  const int as = dtype_size(act_dtype);
  if (ldq < heads * D || ldo < heads * D) return fail(TB_EINVAL, "%s: row strides too small", who);
  if (!aligned16(q) || !aligned16(out) || ldq * as % 16 != 0 || ldo * as % 16 != 0)
    return fail(TB_EINVAL, "%s: rows must be 16-byte aligned", who);
  if ((reinterpret_cast<uintptr_t>(ws) & 255) != 0) return fail(TB_EINVAL, "%s: the workspace must be 256-byte aligned", who);
  const Layout l = layout_of(B, heads, KVH, D);
  if (ws_bytes < l.bytes)
    return fail(TB_EINVAL, "%s: workspace of %zu bytes, %zu needed", who, ws_bytes, l.bytes);
  DeviceState *st;
  TB_TRY(device_state(&st));
  char *w = static_cast<char *>(ws);
  a.q = {q, ldq, act_dtype};
  a.out = out;
  a.ldo = ldo;
  a.kv_heads = (int)KVH;
  a.group = (int)(heads / KVH);
  a.scale2 = scale * kLog2e;
  a.counters = reinterpret_cast<int *>(w);
  a.slot_acc = reinterpret_cast<float *>(w + l.slot_acc);
  a.slot_ml = reinterpret_cast<float2 *>(w + l.slot_ml);
  a.prefix.acc = reinterpret_cast<float *>(w + l.prefix_acc);
  a.prefix.ml = reinterpret_cast<float2 *>(w + l.prefix_ml);
  a.prefix.own = reinterpret_cast<int2 *>(w + l.own);
  a.prefix.begun = a.counters + kMaxCtas;
  a.prefix.rows = (int)(B * a.group);
  a.prefix_table = prefix_table;
  a.prefix_len = (int)prefix_len;
  a.wait_ns = wait_limit_ns();
#define TB_RUN(CT, A32) return D == 64 ? run<CT, 64, A32>(a, cache, st, stream, who) : run<CT, 128, A32>(a, cache, st, stream, who)
  if (act_dtype == TB_F16) TB_RUN(TB_F16, false);
  if (act_dtype == TB_BF16) TB_RUN(TB_BF16, false);
  if (cache->dtype == TB_F16) TB_RUN(TB_F16, true);
  if (cache->dtype == TB_BF16) TB_RUN(TB_BF16, true);
  TB_RUN(TB_F32, true);
#undef TB_RUN
}

}  // namespace

void set_prefix_splits(AttnArgs &a, int64_t items, int64_t tiles, int64_t ctas) {
  const int64_t rows = (int64_t)a.prefix.rows * a.kv_heads;
  a.prefix.splits = (int)prefix_splits(items, tiles, ctas, prefix_pairs(rows) / rows - 1);
  a.prefix.parts = a.prefix.splits + 1;
}

}  // namespace tb

using namespace tb;

extern "C" {

tb_status tb_paged_attention_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                             size_t *bytes_out) {
  if (!bytes_out) return fail(TB_EINVAL, "tb_paged_attention_workspace_bytes: null pointer");
  if (batch < 0 || heads <= 0 || heads > 65536 || kv_heads <= 0 || heads % kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128) || batch > (1 << 20) || batch * heads > (1 << 24))
    return fail(TB_EINVAL, "tb_paged_attention_workspace_bytes: bad extents");
  *bytes_out = layout_of(batch, heads, kv_heads, head_dim).bytes;
  return TB_OK;
}

tb_status tb_paged_attention_decode(const tb_paged_cache *cache, const tb_paged_batch *seqs, int act_dtype,
                                    const void *q, int64_t ldq, int64_t heads, float scale, void *out, int64_t ldo,
                                    void *workspace, size_t workspace_bytes, tb_stream stream) {
  return attention(cache, seqs, nullptr, 0, act_dtype, q, ldq, heads, scale, out, ldo, workspace, workspace_bytes,
                   as_stream(stream), "tb_paged_attention_decode");
}

tb_status tb_paged_attention_shared(const tb_paged_cache *cache, const tb_paged_batch *seqs,
                                    const int32_t *prefix_table, int64_t prefix_len, int act_dtype, const void *q,
                                    int64_t ldq, int64_t heads, float scale, void *out, int64_t ldo, void *workspace,
                                    size_t workspace_bytes, tb_stream stream) {
  return attention(cache, seqs, prefix_table, prefix_len, act_dtype, q, ldq, heads, scale, out, ldo, workspace,
                   workspace_bytes, as_stream(stream), "tb_paged_attention_shared");
}

}  // extern "C"
