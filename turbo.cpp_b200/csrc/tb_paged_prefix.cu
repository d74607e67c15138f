// tb_paged_prefix.cu -- the common prefix of tb_paged_attention_shared on the
// fifth-generation tensor cores (16-bit caches, many query rows).
//
// All sequences' query heads of one key/value head are the rows of a matrix
// product against the prefix: S = Q K^T, P = exp2(scale S - m), O = P V, with
// the running maximum m and sum l of each row; each CTA takes a share of the
// keys and leaves (m, l, acc) per row, which are joined with the sequences' own
// keys' later.
//
// Accuracy: operands in parts as in tb_paged_attention.cu (a query in QT, a
// probability in PT parts; with 16-bit activations one and two, so that a
// sequence's results do not get coarser with the batch; fp16 probabilities are
// scaled by 2^15).  The parts are further MMAs into the same
// accumulator, the smallest first.  With fp32 activations O starts from zero for each tile and is
// added to fp32 registers (one FMA with the rescaling), so no long sum runs
// inside the tensor core, whose accumulator cuts off rather than rounds (2^-24 a
// step: some 1e-5 over a thousand keys).  With 16-bit activations, whose
// outputs are rounded to 2^-9 or 2^-12, O stays in tensor memory for KEEP tiles
// (512 steps, 2^-15 at most) before it is added to an fp32 sum in local memory
// (in registers, although untouched, it cost 3 % of every call), and is rescaled
// only where a row's maximum has grown by 2^8.
//
// Roles: two streams, each a warpgroup whose threads own one row each (TMEM
// lane = row), and one warp issuing its MMAs; one warp loading.  A stream's
// scores have two buffers: while the exponentials of one run, the products fill
// the other.  With more than 128 rows the streams are two row tiles over the
// same keys (PAIR), which halves the reads of K and V; else, or where two
// tiles' queries do not fit, they take alternate key tiles of the same rows and
// join at the end.
//   TMEM, per stream: S [64 columns, twice] with P written over it, O [D
//   columns].  Chunk c of 32 keys is read before its P is written: one part to
//   columns 16 c, two parts to 32 c and 32 c + 16, a third to 64 + 16 c (three
//   parts at head_dim 128 leave room for one buffer only).
// Bounds for 64 keys and two row tiles (cycles per SM): exponentials 1024 on the
// special function units (a polynomial on the FMA units for some of them gained
// nothing: 0, 1/8 .. 4/8 of them measured 81, 80, 81, 83, 85 us); products with
// two parts of a probability 448 at head_dim 64 and 896 at 128 per row tile (Q is
// read from shared memory at 128 bytes a cycle, 1.5 times the tensor cores' own
// time for S).  Measured, with the sequences' own keys and the joins (512 rows of
// each of 8 key/value heads behind 32768 keys): bf16 heads of 128 105 us, of 64 82
// us; with probabilities in one part, which left outputs 1.4 times as far off, 97.6
// and 74.  (The prefix's kernel by itself, cold: 84 us for those 32768 keys of 128,
// 48 for 16384, the tensor pipe 61 % and the special function units 37 % busy.)
// 64 sequences behind 8192 fp16 keys of 64, fp32 queries 34 us.  Two row
// tiles as streams or alternate keys: 80 and 127 us; 33.8 and 35.5 even where the
// second tile has 8 rows (with probabilities in one part).
#include <algorithm>

#include "tb_paged.cuh"

namespace tb {
namespace {

constexpr int kRows = 128;
constexpr int kBlock = 384;

__device__ __forceinline__ void commit_to(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One thread of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// After the wait: the registers become operands, so that no use of them moves ahead of it.
__device__ __forceinline__ void loaded(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Shared-memory descriptor, 128-byte swizzle.  K-major (queries, keys): rows of
// 128 bytes, groups of eight rows 1024 bytes apart.  MN-major (values): the same
// bytes read as 64 columns of head_dim, groups of eight keys 1024 bytes apart,
// the next 64 columns `lbo` bytes on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// CT: cache type, D: head_dim, A32: fp32 activations.
template <int CT_, int D, bool A32>
struct TC {
  static constexpr int CT = CT_;
  static constexpr int QT = !A32 ? 1 : CT == TB_F16 ? 2 : 3;  // parts of a query
  static constexpr int PT = A32 ? QT : 2;                     // parts of a probability
  static constexpr int KT = 64;                               // keys per tile
  static constexpr int NB = PT == 3 && D == 128 ? 1 : 2;      // buffers of S
  static constexpr bool SUMS = A32;                           // O summed in registers, tile by tile
  static constexpr int KEEP = SUMS ? 1 : 512 / (PT * KT / 16);  // tiles whose O is summed in tensor memory
  static constexpr bool PAIR_FITS = QT * D <= 192;            // the queries of two row tiles in shared memory
  static constexpr int RB = 2 * D, CB = D / 64;               // bytes and 128-byte columns of a row
  static constexpr int QTILE = QT * CB * kRows * 128;
  static constexpr int QBYTES = (PAIR_FITS ? 2 : 1) * QTILE;
  static constexpr int HALF = KT * RB;  // a tile of keys, or of values
  static constexpr int STAGES = 4;      // even, so that with alternate tiles a stage is always the same stream's
  static constexpr float SLACK = SUMS ? 0.f : 8.f;  // log2 by which a row may exceed its reference maximum
  static constexpr float PEXP = CT == TB_F16 ? 15.f - SLACK : 0.f;  // probabilities are scaled by 2^PEXP
  static constexpr uint32_t F = CT == TB_BF16 ? 1u : 0u;
  // D fp32, A and B of type F; N, M = 128; the second product's B is MN-major
  static constexpr uint32_t IDESC_QK = (1u << 4) | (F << 7) | (F << 10) | ((uint32_t)(KT >> 3) << 17) | (8u << 24);
  static constexpr uint32_t IDESC_PV = (1u << 4) | (F << 7) | (F << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
  static constexpr int BUF = PT == 3 ? 96 : 64;              // columns of a buffer of S and P
  static constexpr int O = PT == 3 && D == 64 ? 192 : 128;  // column of a stream's O
  static_assert(NB * BUF <= O && O + D <= 256, "");
  static __device__ __forceinline__ int pcol(int part, int chunk) {
    return part < 2 ? 32 * chunk + 16 * part : 64 + 16 * chunk;
  }
};

struct PrefixControl {
  uint64_t kfull[4], kempty[4], vfull[4], vempty[4];
  // per stream and buffer of S (a barrier then never runs a whole phase ahead of a waiter that skips one: tile j's
  // scores imply the products of tile j - NB)
  uint64_t s_full[2][2], p_full[2][2], o_full[2][2];
  uint64_t done[2];  // per stream: all products
  uint32_t tmem;
  float down[2 * kRows];  // fp32 queries of an fp16 cache: 2^-e of each row
};

template <class C>
constexpr int prefix_smem() {
  return C::QBYTES + C::STAGES * 2 * C::HALF + (int)sizeof(PrefixControl);
}

template <int CT, int D, bool A32>
__global__ void __launch_bounds__(kBlock, 1)
    paged_prefix_tc_kernel(const AttnArgs a, const int pair, const __grid_constant__ CUtensorMap km,
                           const __grid_constant__ CUtensorMap vm, uint32_t *__restrict__ err) {
  using C = TC<CT, D, A32>;
  extern __shared__ __align__(1024) unsigned char smem[];
  PrefixControl &ctl = *reinterpret_cast<PrefixControl *>(smem + C::QBYTES + C::STAGES * 2 * C::HALF);
  const uint32_t qs = smem_addr(smem), stages = qs + C::QBYTES;
  // (the warp's number by a shuffle: known to be the same in all lanes, what follows from it stays in uniform registers,
  // which the tensor core's operands come from)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int split = blockIdx.y, kvh = blockIdx.z;
  const int all = (a.prefix_len + C::KT - 1) / C::KT;
  const int t0 = (int)((int64_t)split * all / a.prefix.splits);
  const int n = (int)((int64_t)(split + 1) * all / a.prefix.splits) - t0;  // tiles of this CTA
  if (tid == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&ctl.kfull[i], 1);
      mbar_init(&ctl.kempty[i], pair ? 2 : 1);
      mbar_init(&ctl.vfull[i], 1);
      mbar_init(&ctl.vempty[i], pair ? 2 : 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&ctl.s_full[w][0], 1);
      mbar_init(&ctl.s_full[w][1], 1);
      mbar_init(&ctl.p_full[w][0], kRows);
      mbar_init(&ctl.p_full[w][1], kRows);
      mbar_init(&ctl.o_full[w][0], 1);
      mbar_init(&ctl.o_full[w][1], 1);
      mbar_init(&ctl.done[w], 1);
    }
    fence_mbar_init();
  }
  if (tid == 256) {
    prefetch_map(&km);
    prefetch_map(&vm);
  }
  if (warp == 11) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&ctl.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  pdl_wait();
  if (tid == kBlock - 1) let_next_begin(a.prefix);
  const int stream = warp >> 2, r = tid & 127;
  const int row0 = blockIdx.x * (pair ? 2 * kRows : kRows);  // of all rows of the key/value head
  // ---- queries (all warps but the loading one): D / 8 lanes per row, eight elements each
  if (warp != 8) {
    constexpr int L = D / 8, PER = (kBlock - 32) / L;  // rows at a time
    constexpr int N = 2 * kRows / PER + 1, W = A32 ? 2 : 1;
    static_assert(PER % (32 / L) == 0, "a warp's rows end together");
    const int at = tid < 256 ? tid : tid - 32, c = at % L;
    const int rows = pair ? 2 * kRows : kRows;
    uint4 raw[N][W];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = at / L + k * PER, row = row0 + i;
#pragma unroll
      for (int e = 0; e < W; ++e) raw[k][e] = make_uint4(0, 0, 0, 0);
      if (i < rows && row < a.prefix.rows) {
        const int b = row / a.group;
        const int64_t from = (int64_t)b * a.q.ld + (int64_t)(kvh * a.group + row - b * a.group) * D + 8 * c;
#pragma unroll
        for (int e = 0; e < W; ++e)
          raw[k][e] = reinterpret_cast<const uint4 *>(static_cast<const char *>(a.q.p) + from * (A32 ? 4 : 2))[e];
      }
    }
    const float sign = a.scale2 < 0.f ? -1.f : 1.f;  // a negative scale turns the queries round
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = at / L + k * PER;
      if (i >= rows) break;
      float f[8];
      if constexpr (A32) {
        float lo[4], hi[4];
        Word<TB_F32>::get(raw[k][0], lo);
        Word<TB_F32>::get(raw[k][W - 1], hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = lo[e], f[4 + e] = hi[e];
      } else {
        Word<CT>::get(raw[k][0], f);
      }
      float up = sign;
      if constexpr (A32 && CT == TB_F16) {
        float mx = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(f[e]));
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const int e = fp16_exp(mx);
        up *= pow2i(e);
        if (c == 0) ctl.down[i] = pow2i(-e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= up;
#pragma unroll
      for (int p = 0; p < C::QT; ++p) {
        uint4 w;
        w.x = pack_rest<CT>(f[0], f[1]);
        w.y = pack_rest<CT>(f[2], f[3]);
        w.z = pack_rest<CT>(f[4], f[5]);
        w.w = pack_rest<CT>(f[6], f[7]);
        const uint32_t to = qs + (i / kRows) * C::QTILE + (p * C::CB + (c >> 3)) * kRows * 128 + (i % kRows) * 128 +
                            (((c ^ i) & 7) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                     : "memory");
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync 4, %0;" ::"n"(kBlock - 32) : "memory");
  }
  const uint32_t tmem = ctl.tmem;
  bool dead = false;

  // tile j of a stream w is tile first + j * step of the CTA's n
  const int step = pair ? 1 : 2;
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 8) {  // ---- loading
      int keys = 0, values = 0;  // tiles issued
      dead = begin_dead(a.wait_ns, err);  // (the others find out by waiting)
      for (int t = 0; t < n; ++t) {
        const int s = t % C::STAGES;
        const uint32_t ph = ((t / C::STAGES) & 1) ^ 1;
        const TileBoxes box = tile_boxes<C::KT>(a.pools, a.box_shift, a.prefix_table, a.prefix_len, t0 + t);
        wait_phase(&ctl.kempty[s], ph, err, dead, a.wait_ns);
        if (__any_sync(0xffffffffu, dead)) break;
        load_rows<C::KT, C::RB, 2>(stages + s * 2 * C::HALF, &ctl.kfull[s], &km, nullptr, a.pools, a.box_shift,
                                   a.prefix_table, box, t0 + t, kvh, err);
        ++keys;
        wait_phase(&ctl.vempty[s], ph, err, dead, a.wait_ns);
        if (__any_sync(0xffffffffu, dead)) break;
        load_rows<C::KT, C::RB, 2>(stages + s * 2 * C::HALF + C::HALF, &ctl.vfull[s], &vm, nullptr, a.pools,
                                   a.box_shift, a.prefix_table, box, t0 + t, kvh, err);
        ++values;
      }
      wait_copies<C::STAGES>(ctl.kfull, keys, err);
      wait_copies<C::STAGES>(ctl.vfull, values, err);
    } else if (warp < 11) {  // ---- products of stream w
      const int w = warp - 9, first = pair ? 0 : w, mine = (n - first + step - 1) / step;
      const uint32_t ts = tmem + w * 256, q = qs + (pair ? w * C::QTILE : 0);
      const uint64_t qd = desc(q, 16);
      auto scores = [&](int j) {
        const int t = first + j * step, s = t % C::STAGES;
        const uint32_t k = stages + s * 2 * C::HALF, to = ts + (j % C::NB) * C::BUF;
        const uint64_t kd = desc(k, 16);  // 16 elements further: 32 bytes, 2 in the descriptor's address field
        wait_phase(&ctl.kfull[s], (t / C::STAGES) & 1, err, dead, a.wait_ns);
        fence_after();
        if (elect_one()) {
#pragma unroll
          for (int p = C::QT - 1; p >= 0; --p)  // the smallest part first: the accumulator cuts off at its own size
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
              mma_ss(to, qd + ((p * C::CB + i / 4) * kRows * 8 + (i % 4) * 2), kd + ((i / 4) * C::KT * 8 + (i % 4) * 2),
                     C::IDESC_QK, p < C::QT - 1 || i > 0);
          commit_to(&ctl.s_full[w][j % C::NB]);
          if (!dead) commit_to(&ctl.kempty[s]);
        }
        __syncwarp();
      };
      for (int j = 0; j < min(C::NB, mine); ++j) scores(j);
      for (int j = 0; j < mine; ++j) {
        const int t = first + j * step, s = t % C::STAGES;
        const uint32_t v = stages + s * 2 * C::HALF + C::HALF, p0 = ts + (j % C::NB) * C::BUF;
        const int keys = min(C::KT, a.prefix_len - (t0 + t) * C::KT), steps = (keys + 15) / 16;
        wait_phase(&ctl.vfull[s], (t / C::STAGES) & 1, err, dead, a.wait_ns);
        if (keys < steps * 16) {
          // the rows of the last step behind the prefix hold whatever their page held: 0 times that has to be 0
          for (int i = lane; i < (steps * 16 - keys) * (C::RB / 16); i += 32) {
            const int vr = keys + i / (C::RB / 16), c = i % (C::RB / 16);
            sts128_zero(v + (c >> 3) * C::KT * 128 + vr * 128 + (((c ^ vr) & 7) << 4));
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        wait_phase(&ctl.p_full[w][j % C::NB], (j / C::NB) & 1, err, dead, a.wait_ns);
        fence_after();
        const uint64_t vd = desc(v, C::KT * 128);  // 16 keys further: 2048 bytes
        if (elect_one()) {
#pragma unroll
          for (int p = C::PT - 1; p >= 0; --p)
#pragma unroll
            for (int i = 0; i < C::KT / 16; ++i) {
              if (i >= steps) break;
              mma_ts(ts + C::O, p0 + C::pcol(p, i / 2) + 8 * (i % 2), vd + i * 128, C::IDESC_PV,
                     p < C::PT - 1 || i > 0 || j % C::KEEP > 0);
            }
          if (!dead) commit_to(&ctl.vempty[s]);
          commit_to(&ctl.o_full[w][j % C::NB]);
        }
        __syncwarp();
        // into the buffer whose P the products just issued read: the tensor core takes them in order
        if (j + C::NB < mine) scores(j + C::NB);
      }
      // tensor memory is given back, and the CTA ends, only behind the last product, waited for elsewhere or not
      if (elect_one()) commit_to(&ctl.done[w]);
      __syncwarp();
      mbar_wait_bounded(&ctl.done[w], 0, err);
    }
  } else {  // ---- the exponentials of stream `stream`
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const uint32_t ts = tmem + stream * 256 + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes
    float scale2 = fabsf(a.scale2);
    if (A32 && CT == TB_F16) scale2 *= ctl.down[(pair ? stream * kRows : 0) + r];
    if (scale2 < 1e-37f) scale2 = 1e-37f;  // 0 in effect, but times the -inf of a masked key it is still -inf
    uint64_t acc[C::SUMS ? D / 2 : 1];  // pairs of columns
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < (C::SUMS ? D / 2 : 1); ++i) acc[i] = 0ull;
    // SUMS: adds a finished tile's O to the running sum
    auto take_o = [&](float f) {
      const uint64_t al = pack2(f, f);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(ts + C::O + 32 * c, o);
        tmem_wait_ld();
        loaded(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint64_t &x = acc[C::SUMS ? 16 * c + i : 0];
          x = fma2(x, al, pack2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])));
        }
      }
    };
    // not SUMS: O times this row's factor, in place (the products before are done, the next wait for P)
    auto scale_o = [&](float f) {
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(ts + C::O + 32 * c, o);
        tmem_wait_ld();
        loaded(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st32(ts + C::O + 32 * c, o);
      }
    };
    // not SUMS: the sum of the O before the present one, and the factor that it still needs
    float kept[C::SUMS ? 1 : D], kept_f = 0.f;
    auto keep_o = [&](bool first) {
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(ts + C::O + 32 * c, o);
        tmem_wait_ld();
        loaded(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float &x = kept[C::SUMS ? 0 : 32 * c + i];
          x = first ? __uint_as_float(o[i]) : fmaf(x, kept_f, __uint_as_float(o[i]));
        }
      }
      kept_f = 1.f;
    };
    const int first = pair ? 0 : stream, mine = (n - first + step - 1) / step;
    auto wait_o = [&](int j) { wait_phase(&ctl.o_full[stream][j % C::NB], (j / C::NB) & 1, err, dead, a.wait_ns); };
    float before = 1.f;  // SUMS: the factor that the sums before the last tile's O still need
    for (int j = 0; j < mine; ++j) {
      const uint32_t sp = ts + (j % C::NB) * C::BUF;
      wait_phase(&ctl.s_full[stream][j % C::NB], (j / C::NB) & 1, err, dead, a.wait_ns);
      fence_after();
      uint32_t u[C::KT / 32][32];  // the row's scores
#pragma unroll
      for (int c = 0; c < C::KT / 32; ++c) tmem_ld32(sp + 32 * c, u[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < C::KT / 32; ++c) loaded(u[c]);
      const int keys = a.prefix_len - (t0 + first + j * step) * C::KT;  // KT or more except in the last tile
      if (keys < C::KT) {
#pragma unroll
        for (int c = 0; c < C::KT / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (32 * c + i >= keys) u[c][i] = 0xFF800000u;  // -inf
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < C::KT / 32; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(u[c][i]), __uint_as_float(u[c][i + 1]));
      const float top = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2);
      float alpha = 1.f;
      if constexpr (C::SUMS) {
        alpha = ex2(m - (top == -INFINITY ? 0.f : top));
        l *= alpha;
        m = top;
      } else if (j == 0) {
        m = top;
      } else {
        if (j % C::KEEP == 0) {  // the next products begin a new O
          wait_o(j - 1);
          fence_after();
          keep_o(j == C::KEEP);
        }
        // the reference maximum follows only where a row has outgrown it by 2^SLACK; its O and l are then scaled down
        const bool grown = top > m + C::SLACK;
        if (__any_sync(0xffffffffu, grown)) {
          const float f = grown ? ex2(m - top) : 1.f;
          wait_o(j - 1);
          fence_after();
          scale_o(f);
          kept_f *= f;
          l *= f;
          if (grown) m = top;
        }
      }
      const float ms = m == -INFINITY ? 0.f : m;
      const uint64_t scale = pack2(scale2, scale2), shift = pack2(C::PEXP - ms, C::PEXP - ms);
      uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < C::KT / 32; ++c) {
        float p[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t x = fma2(pack2(__uint_as_float(u[c][2 * i]), __uint_as_float(u[c][2 * i + 1])), scale, shift);
          unpack2(x, p[2 * i], p[2 * i + 1]);
          p[2 * i] = ex2(p[2 * i]);
          p[2 * i + 1] = ex2(p[2 * i + 1]);
          sum[i & 1] = add2(sum[i & 1], pack2(p[2 * i], p[2 * i + 1]));
        }
#pragma unroll
        for (int k = 0; k < C::PT; ++k) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack_rest<CT>(p[2 * i], p[2 * i + 1]);
          tmem_st16(sp + C::pcol(k, c), w);
        }
      }
      float s0, s1;
      unpack2(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      if (C::SUMS && j > 0) {  // the last tile's O, before the next products overwrite it
        wait_o(j - 1);
        fence_after();
        take_o(before);
      }
      before = alpha;
      tmem_wait_st();
      fence_before();
      mbar_arrive(&ctl.p_full[stream][j % C::NB]);
    }
    float out[D];
#pragma unroll
    for (int i = 0; i < D; ++i) out[i] = 0.f;
    if (mine > 0) {
      wait_o(mine - 1);
      fence_after();
      if constexpr (C::SUMS) {
        take_o(before);
#pragma unroll
        for (int i = 0; i < D / 2; ++i) unpack2(acc[i], out[2 * i], out[2 * i + 1]);
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(ts + C::O + 32 * c, o);
          tmem_wait_ld();
          loaded(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) out[32 * c + i] = __uint_as_float(o[i]);
        }
        if (mine > C::KEEP) {
#pragma unroll
          for (int i = 0; i < D; ++i) out[i] = fmaf(kept[C::SUMS ? 0 : i], kept_f, out[i]);
        }
      }
    }
    const float down = ex2(-C::PEXP);
    l *= down;
#pragma unroll
    for (int i = 0; i < D; ++i) out[i] *= down;
    if (!pair) {
      // both streams are done with the stages once both have their last O: the second leaves its results there
      asm volatile("bar.sync 1, 256;" ::: "memory");
      float *left = reinterpret_cast<float *>(smem + C::QBYTES);  // [D + 2][128]
      if (stream == 1) {
        left[D * kRows + r] = m;
        left[(D + 1) * kRows + r] = l;
#pragma unroll
        for (int i = 0; i < D; ++i) left[i * kRows + r] = out[i];
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (stream == 0) {
        const float m1 = left[D * kRows + r];
        const float mn = fmaxf(m, m1), ms = mn == -INFINITY ? 0.f : mn;
        const float w0 = ex2(m - ms), w1 = ex2(m1 - ms);
        m = mn;
        l = l * w0 + left[(D + 1) * kRows + r] * w1;
#pragma unroll
        for (int i = 0; i < D; ++i) out[i] = fmaf(out[i], w0, left[i * kRows + r] * w1);
      }
    }
    // results through shared memory, so that rows leave whole: the stream's queries are no longer read (its last O is
    // here), and half of the columns take at most their room
    if (pair || stream == 0) {
      constexpr int H = D / 2;  // columns at a time
      static_assert(kRows * H * 4 <= C::QTILE, "");
      const int row = row0 + (pair ? stream * kRows : 0);
      if (row + r < a.prefix.rows)
        a.prefix.ml[((int64_t)kvh * a.prefix.rows + row + r) * a.prefix.parts + split] = make_float2(m, l);
      float4 *buf = reinterpret_cast<float4 *>(smem + (pair ? stream * C::QTILE : 0));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < H / 4; ++i)
          buf[r * (H / 4) + (i ^ (r & 7))] = make_float4(out[h * H + 4 * i], out[h * H + 4 * i + 1],
                                                         out[h * H + 4 * i + 2], out[h * H + 4 * i + 3]);
        asm volatile("bar.sync %0, 128;" ::"r"(2 + stream) : "memory");
        for (int i = r; i < kRows * H / 4; i += kRows) {
          const int x = i / (H / 4), c = i % (H / 4);
          if (row + x < a.prefix.rows)
            reinterpret_cast<float4 *>(a.prefix.acc + (((int64_t)kvh * a.prefix.rows + row + x) * a.prefix.parts + split) * D +
                                       h * H)[c] = buf[x * (H / 4) + (c ^ (x & 7))];
        }
        asm volatile("bar.sync %0, 128;" ::"r"(2 + stream) : "memory");
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 11)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int CT, int D, bool A32>
tb_status launch(AttnArgs &a, const PagedMaps &maps, const DeviceState *st, cudaStream_t s, const char *who) {
  using C = TC<CT, D, A32>;
  auto kern = paged_prefix_tc_kernel<CT, D, A32>;
  constexpr int smem = prefix_smem<C>();
  static_assert(smem <= 227 * 1024 && C::STAGES * 2 * C::HALF >= (D + 2) * kRows * 4, "");
  TB_TRY(ensure_smem_for(kern, smem));
  const int pair = C::PAIR_FITS && a.prefix.rows > kRows;
  const int rows = pair ? 2 * kRows : kRows;
  const int row_tiles = (a.prefix.rows + rows - 1) / rows;
  const int tiles = (a.prefix_len + C::KT - 1) / C::KT;
  const int64_t items = (int64_t)row_tiles * a.kv_heads;
  set_prefix_splits(a, items, tiles, st->sm_count);
  return launch_pdl(kern, dim3((unsigned)row_tiles, (unsigned)a.prefix.splits, (unsigned)a.kv_heads), kBlock, smem, s,
                    who, a, pair, maps.k, maps.v, st->err_word);
}

}  // namespace

tb_status launch_prefix_tc(AttnArgs &a, const PagedMaps &maps, int cache_dtype, int head_dim, const DeviceState *st,
                           cudaStream_t s, const char *who) {
  const bool wide = head_dim == 128, a32 = a.q.dtype == TB_F32;
#define TB_PREFIX(CT, A32) \
  return wide ? launch<CT, 128, A32>(a, maps, st, s, who) : launch<CT, 64, A32>(a, maps, st, s, who)
  if (cache_dtype == TB_F16) {
    if (a32) TB_PREFIX(TB_F16, true);
    TB_PREFIX(TB_F16, false);
  }
  if (a32) TB_PREFIX(TB_BF16, true);
  TB_PREFIX(TB_BF16, false);
#undef TB_PREFIX
}

}  // namespace tb
