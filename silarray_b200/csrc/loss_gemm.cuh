// The tensor-core products of the cross entropy (sm_100a), for bf16 operands
// and for fp32 ones given as exact tf32 pairs (x = hi + lo).
//
// One persistent kernel, D[M, N] = A . B with fp32 accumulation in TMEM:
//   bf16  tcgen05.mma kind::f16, one product per 16 k;
//   tf32  kind::tf32, lo.hi + hi.lo + hi.hi per 8 k (3xTF32).
// Either operand may lie in either major order (k contiguous, or the M / N
// index), so ds and W serve their products in place and nothing is transposed.
//   warp 0      TMA producer: boxes of 128-byte rows, 192 KB ring;
//   warp 1      allocates the 512 TMEM columns (two accumulators of 256) and
//               issues the MMAs from one thread;
//   warps 2-9   epilogue, two per TMEM lane quarter, 128 columns each.
// A tile is 256 x 256 on a CTA pair (cta_group::2: each CTA loads its 128 rows
// of A and 128 columns of B), or for the scores 128 x bn on one CTA, where that takes fewer
// rounds of all SMs (score_tiles): few rows, where reading W is all, and few tiles.
//
// What bounds it: the tensor pipe and, over many milliseconds, the card's
// power.  The one thread that issues the MMAs was the limit at first: with a
// commit per CTA of the pair, descriptors built per MMA and a stage of 64 k,
// the scores of 8192 x 131072 x 2048 took 3.73 ms (1181 TFLOP/s); one multicast
// commit for both CTAs 3.53; descriptors advanced by an add and the wait's
// first poll inline 3.31; stages of 128 k 3.13 (1405; torch.matmul's library
// product alone 3.35 at the same shape and load).  4 to 7 stages of 64 k gave the
// same times, and prefetching operands to the L2 made them worse.
//
// Sums: the tensor core truncates as it accumulates, so sums that need more
// than its 2^-22 per step are cut into chunks; the epilogue adds each chunk in fp32
// registers, to nearest, while the next one runs.  Chunks are 128 k of tf32, 1024 k of bf16
// scores, and 16384 k of the products of bf16 ds, whose results are rounded to bf16: of a sum of
// one sign such chunks lose 9 x 10^-5 (2^-13 at most, a chunk's sum growing evenly), where
// 211000 terms in one chunk lost 1.2 x 10^-3 and 262144 1.7 x 10^-3.
// The backward's bf16 scores take the forward's chunks although ds is rounded to bf16
// next: 8 x 10^-4 of a sum of 131072 products of one sign is lost in one chunk, 10^-5 of
// one of 4096, and where p is near 1 that much is left in p - 1.  It costs steps of D above
// 1024 1 to 2.5 % (4096 rows of 32768 x 4096 3.23 -> 3.27 ms, 16384 of 20000 x 1536 3.14 -> 3.20).
//
// Every wait is bounded; on expiry the kernel records a code, unwinds, lets what
// is in flight land, frees its TMEM and exits.  No load is multicast.
#pragma once

#include <cuda.h>

#include "elem.cuh"
#include "loss_epilogue.cuh"
#include "tc_common.cuh"

namespace silcu {
namespace lossmm {
using namespace tc;

constexpr int BM = 128, BN = 256;

enum Epilogue { kStats = 0, kScoreGrad = 1, kOut = 2, kOutT = 3 };
enum OutMode { kDirect = 0, kPlane = 1, kPlaneAdd = 2 };

// mbar_wait without its call: around a call the 128 sums of an epilogue thread
// would have to be saved.
__device__ __forceinline__ bool wait_inline(uint32_t bar, uint32_t parity, int *err, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer();
#pragma unroll 1
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); i++) {
    if ((i & 63u) == 0) {
      if (*reinterpret_cast<volatile int *>(err) != 0) return false;
      if (globaltimer() - t0 > WAIT_NS) {
        atomicCAS(err, 0, code);
        return false;
      }
    }
  }
  return true;
}

// After a wait that gave up: the loads and MMAs that this thread issued, or that
// it no longer waits for, end within microseconds; a millisecond covers them.
__device__ __forceinline__ void settle() {
  const unsigned long long t0 = globaltimer();
#pragma unroll 1
  for (int i = 0; i < (1 << 16) && globaltimer() - t0 < 1000000ull; i++) asm volatile("nanosleep.u32 1000;");
}

// Adds to an earlier launch's sum.  Nothing else adds to this element in this
// launch, so the order is fixed; done in the L2, no thread waits for the old sum
// (as loads and stores, which may alias, 32 in a row cost a tile 15 us and more).
__device__ __forceinline__ void red_add4(float *p, const uint4 &v) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(__uint_as_float(v.x)),
               "f"(__uint_as_float(v.y)), "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w))
               : "memory");
}

__device__ __forceinline__ void red_add(float *p, float v) {
  asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(p), "f"(v) : "memory");
}

__device__ __forceinline__ void store_as(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_as(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// x rounded to tf32 as cvt.rna.tf32 does (halves away from zero), on the
// integer pipe: the conversion took 70 of 660 us of the score gradients.
__device__ __forceinline__ float tf32_rna_bits(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
}

// What the tensor core reads of x as a tf32 operand.
__device__ __forceinline__ float tf32_trunc(float x) {
  return __uint_as_float(__float_as_uint(x) & 0xffffe000u);
}

// x - tf32_trunc(x) for the tensor core, which cuts it to 11 bits of 13: 2^-12 of itself more is a
// quarter to half a step of those, so that what is cut is off by half a step at most and an
// eighth on average, as if it had been rounded (three eighths without, all of them toward
// zero).  The epilogue warps' instructions are what a stage of few rows waits for: 4 rows of 50000 x
// 2048 take 154 us with this, 152 without, 162 with a conversion that rounds.
__device__ __forceinline__ float remainder_of(float x) {
  return __fmul_rn(__fsub_rn(x, tf32_trunc(x)), 1.0f + 1.0f / 4096.0f);
}

// Whether a row with this target is not left out.
__device__ __forceinline__ bool counts(int y, int V) { return y >= 0 && y < V; }

struct Bf16 {
  using T = __nv_bfloat16;
  static constexpr int PARTS = 1, KROW = 64, KMMA = 16;  // k in a 128-byte row, and of one MMA
  static constexpr uint32_t FORMAT = (1u << 7) | (1u << 10);
};
struct Tf32 {
  using T = float;
  static constexpr int PARTS = 2, KROW = 32, KMMA = 8;
  static constexpr uint32_t FORMAT = (2u << 7) | (2u << 10);
};

template <typename Ty, int EPI, bool PAIR, bool RAW = false>
struct Cfg {
  static_assert(!RAW || (Ty::PARTS == 2 && !PAIR), "raw operands: tf32 on single CTAs");
  static_assert(PAIR || EPI == kStats || EPI == kScoreGrad || (EPI == kOutT && RAW), "single CTAs");
  static constexpr int TM = PAIR ? 2 * BM : BM;
  static constexpr int ROWS_B = PAIR ? BN / 2 : BN;  // B columns held per CTA
  static constexpr int SUBS = PAIR && Ty::PARTS == 1 ? 2 : 1;  // 128-byte-row tiles of each operand per stage
  static constexpr int BK = SUBS * Ty::KROW;
  static constexpr int TILE_A = BM * 128, TILE_B = ROWS_B * 128;
  static constexpr int STAGE_BYTES = SUBS * Ty::PARTS * (TILE_A + TILE_B);
  static constexpr int RING_BYTES = 192 * 1024;
  static constexpr int STAGES = RAW ? 8 : RING_BYTES / STAGE_BYTES;  // RAW: at most, see Params::stages
  static constexpr int EPI_WARPS = 8;
  static constexpr int SMEM_BYTES = RING_BYTES + EPI_WARPS * 4096 + 1024 + 512;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int NBUF = 2;
  // Stages per accumulation chunk; a tile may take several, which meet in registers.
  // SUMS: every tile's sums pass through registers; else those of one chunk stay in TMEM.
  static constexpr bool SUMS = Ty::PARTS == 2 || EPI == kStats;
  // Columns that join the sums at a time: 32 leave the tf32 sums no registers, and
  // what spills there every chunk pays for (score gradients 660 -> 477 us with 16).  What
  // still spills, outside that loop: 48 bytes a thread of the tf32 score gradients
  // (not RAW), 36 of the bf16 scores.
  static constexpr int LD = EPI == kStats && Ty::PARTS == 1 ? 32 : 16;
  // The sums go back to TMEM for the epilogues that have no registers beside
  // them (with the 128 sums in registers the tf32 score gradients spill 2.8 KB a thread).
  static constexpr bool BACK = !SUMS || EPI == kScoreGrad || EPI == kOut;
  // The scores' chunks are the same in both passes, which so see the same scores:
  // (p - 1) of a target that is all but certain is what is left of them.
  static constexpr int CHUNK =
      (Ty::PARTS == 2 ? 128 : EPI == kStats || EPI == kScoreGrad ? 1024 : 16384) / BK;
  // Rows of tiles that are walked together, column by column.  The scores read W once
  // (their H stays in the L2); kOut's tiles of one row of them follow one another and share its
  // ds: against groups of 8 the DRAM reads of 4096 x 8192 x 768 fp32 fall from 1018 to 783 MB.
  // Backward passes of 19 shapes (both types, 200 to 32768 rows, D 512 to 4096) take 1 to 3 %
  // less than with groups of 16 where ds is the larger operand, as long where tiles are few, and
  // 1 to 2.4 % more where W is much the larger one (bf16, 1024 and 2048 rows, D 2048 and 4096).
  static constexpr int GROUP_M = EPI == kOut ? 1 : 16;
  static constexpr uint32_t MN_BOX = Ty::KROW * 128;       // KROW elements of M / N x KROW k
  static constexpr uint32_t MN_STEP = Ty::KMMA * 128;      // one MMA's k inside it
  static constexpr int MN_BOXES_A = BM / Ty::KROW, MN_BOXES_B = ROWS_B / Ty::KROW;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// Division of 0 <= n < 2^31 by a divisor known on the host: with 2^l >= d, m =
// floor(2^(31 + l) / d) + 1 is off by less than 1 and n m / 2^(31 + l) by less than 1 / d.
struct Divisor {
  uint32_t m, shift;
  void set(int d) {
    int l = 0;
    while ((int64_t(1) << l) < d) l++;
    shift = uint32_t(31 + l);
    m = uint32_t((uint64_t(1) << shift) / uint64_t(d) + 1);
  }
  __device__ __forceinline__ int operator()(int n) const { return int((uint64_t(uint32_t(n)) * m) >> shift); }
};

struct Problem {
  CUtensorMap a[2], b[2];  // [part]: hi, lo (tf32)
  int M, N, K, tiles_m, tiles_n;
  // What tile_of divides by (set in launch): the epilogue of a short tile waits for it,
  // and three divisions at run time take 900 cycles.
  Divisor by_split, by_group, by_last;
  int ksplit;              // each tile's K range in this many parts (kOut; part i -> plane i)
  int amn;                 // kOut: A is stored with the M index contiguous (kOutT: it always is)
  int mode, vec;           // vec: kDirect rows are 16-byte aligned
  int of_rows;             // kOut: the result is dH, with a row for each target (kOutT: always)
  void *out;
  int64_t ldo, plane;      // row stride; elements from one plane to the next
};

struct __align__(64) Params {
  Problem p[2];  // kOut: up to two products in one launch
  void *ds[2];       // score gradients [part]: [M, lds], lds a multiple of 64
  int64_t lds;
  int bn;            // tile columns (of the scores on CTA pairs: BN)
  int rows_a;        // rows of A's boxes (single CTAs; the rest of a tile is never stored)
  int half;          // columns of an epilogue warp (RAW and kOut; else 128)
  int stages;        // ring stages (RAW)
  // Work items n0 of p[0] and n1 of p[1] over `units` CTAs (pairs); see work_at.
  int units, n0, n1, rounds, tail, extra;  // rounds = n0 / units, tail = n0 % units
  const float *alpha;  // kOut, kOutT: factor of kDirect results in bf16, 0 for rows that are left out; or null = 1
  LossArgs loss;
  int part0;  // index of this launch's first part
  int *err;
};

struct Work {
  int prob, item;
};

// The k-th item of unit u.  The first product's items go round the units; if
// the last round leaves units tail.. without one, those start with `extra` rounds of
// the second product's (about one item of the first in cost), and the rest goes
// round all units.
__device__ __forceinline__ bool work_at(const Params &p, int u, int k, Work &w) {
  if (u + k * p.units < p.n0) {
    w = Work{0, u + k * p.units};
    return true;
  }
  k -= p.rounds + (u < p.tail);  // the unit's items of the first product
  const int low = p.units - p.tail;  // units short of one item
  int j;
  if (p.tail && u >= p.tail) j = k < p.extra ? k * low + u - p.tail : p.extra * low + (k - p.extra) * p.units + u;
  else j = p.extra * low + k * p.units + u;
  w = Work{1, j};
  return j < p.n1;
}

struct Tile {
  int m0, n0, kb0, kb1, part;
};

template <typename C>
__device__ __forceinline__ Tile tile_of(const Problem &q, int bn, int item) {
  const int t = q.by_split(item), part = item - t * q.ksplit;
  const int group = q.by_group(t);
  const int first = group * C::GROUP_M;
  const int gm = q.tiles_m - first < C::GROUP_M ? q.tiles_m - first : C::GROUP_M;
  const int r = t - group * C::GROUP_M * q.tiles_n;
  const int nk = (q.K + C::BK - 1) / C::BK;
  const int col = gm == C::GROUP_M ? r / C::GROUP_M : q.by_last(r), row = first + r - col * gm;
  // at most 64 parts of 2^24 k, 32 or more to a block: the products stay below 2^31
  return Tile{row * C::TM, col * bn, q.by_split(part * nk), q.by_split((part + 1) * nk), part};
}

template <typename Ty, typename C>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn) {
  if (!mn) return make_desc(addr);
  return Ty::PARTS == 1 ? make_desc_mn16(addr, C::MN_BOX) : make_desc_mn32(addr, C::MN_BOX);
}

// The scores' operands both have k contiguous; of kOut's, B has the N index contiguous
// (BMN) and A what Problem::amn says.
//
// kOutT stores its result transposed, D[m, n] at out[n][m]: dH of few rows as
// (W^T ds^T)^T.  W, with the M index contiguous, then fills the tile's 128 or 256 rows
// and ds its few columns, and an MMA takes the time of the columns that exist.  As
// ds . W the few rows were padded to a whole tile: 30 rows of 60000 x 3000
// took 185 us in bf16 and 580 in fp32; so they take 56 (6.4 TB/s) and 280.
//
// RAW: one operand may be plain fp32.  Its tile is the hi operand as it stands (the
// tensor core reads the upper 19 bits of a value), and the epilogue warps, idle
// while the MMAs run, write the remainders beside it.  Two buffers for those and more
// stages in their place gave nothing, nor did halves of the warps that take turns: twelve
// MMAs per 32 k that each read 128 rows of A are what a stage costs.  For few rows, where the
// time is that of reading W, this spares writing and reading a split copy.
// Stages are as large as the tile needs.
template <typename Ty, int EPI, bool PAIR, bool RAW>
__global__ void __launch_bounds__(Cfg<Ty, EPI, PAIR, RAW>::THREADS, 1) gemm(const __grid_constant__ Params p) {
  using C = Cfg<Ty, EPI, PAIR, RAW>;
  using T = typename Ty::T;
  constexpr bool BMN = EPI == kOut, RAW_A = EPI == kOutT;
  constexpr int NBUF = C::NBUF, PARTS = Ty::PARTS, SUBS = C::SUBS;
  const int TILE_A = RAW ? p.rows_a * 128 : C::TILE_A, TILE_B = RAW ? p.bn * 128 : C::TILE_B;
  const int SUB_BYTES = PARTS * (TILE_A + TILE_B), STAGE_BYTES = SUBS * SUB_BYTES;
  const uint32_t STAGES = RAW ? uint32_t(p.stages) : uint32_t(C::STAGES);
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::RING_BYTES + C::EPI_WARPS * 4096);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 3 * C::STAGES + 2 * NBUF);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + C::STAGES);
  const uint32_t tfull0 = smem_u32(bars + 2 * C::STAGES), tempty0 = smem_u32(bars + 2 * C::STAGES + NBUF);
  const uint32_t ready0 = smem_u32(bars + 2 * C::STAGES + 2 * NBUF);  // RAW: the stage's remainders are written

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int unit = PAIR ? int(blockIdx.x >> 1) : int(blockIdx.x);
  const int bn = PAIR && (EPI == kStats || EPI == kScoreGrad) ? BN : p.bn;

  let_next_start();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
      if (RAW) mbar_init(ready0 + 8 * s, C::EPI_WARPS);
    }
    for (int j = 0; j < NBUF; j++) {
      mbar_init(tfull0 + 8 * j, 1);
      mbar_init(tempty0 + 8 * j, C::EPI_WARPS * (PAIR ? 2 : 1));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // the peer's barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_previous();
  if (EPI == kStats && blockIdx.x == 0 && threadIdx.x == 0) *p.loss.done = 0u;
  Work w;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t kbg = 0;
      bool ok = true;
      const uint32_t bytes =
          SUBS * PARTS * ((PAIR ? TILE_A : p.rows_a * 128) * (PAIR ? 2 : 1) + bn * 128);  // a pair's, on the even CTA
      const int boxes_b = (PAIR ? bn / 2 : bn) / Ty::KROW;
      for (int k = 0; ok && work_at(p, unit, k, w); k++) {
        const Problem &q = p.p[w.prob];
        const Tile tl = tile_of<C>(q, bn, w.item);
        const int am = tl.m0 + BM * int(rank), nb = tl.n0 + (PAIR ? bn / 2 : 0) * int(rank);
        const bool amn = EPI == kOutT || (EPI == kOut && q.amn);
        for (int kb = tl.kb0; kb < tl.kb1; kb++, kbg++) {
          const uint32_t s = kbg % STAGES, ph = (kbg / STAGES) & 1;
          if (kbg >= STAGES && !mbar_try_wait(empty0 + 8 * s, ph ^ 1) &&
              !mbar_wait(empty0 + 8 * s, ph ^ 1, p.err, 21)) {
            ok = false;
            break;
          }
          // a pair's bytes all complete on the even CTA's barrier
          const uint32_t bar = PAIR ? mapa_shared(full0 + 8 * s, 0) : full0 + 8 * s;
          if (rank == 0) mbar_expect_tx(full0 + 8 * s, RAW ? bytes - (RAW_A ? TILE_A : TILE_B) : bytes);
          auto load = [&](uint32_t dst, const CUtensorMap *map, int c0, int c1) {
            if (PAIR) tma_load_2d_pair(dst, map, bar, c0, c1);
            else tma_load_2d(dst, map, bar, c0, c1);
          };
#pragma unroll
          for (int u = 0; u < SUBS; u++) {
            const int kc = kb * C::BK + u * Ty::KROW;
            uint32_t dst = smem_u32(smem + s * STAGE_BYTES + u * SUB_BYTES);
#pragma unroll
            for (int h = 0; h < PARTS; h++, dst += TILE_A) {
              if (RAW && RAW_A && h == 1) continue;
              if (amn) {
#pragma unroll
                for (int i = 0; i < C::MN_BOXES_A; i++) load(dst + i * C::MN_BOX, &q.a[h], am + Ty::KROW * i, kc);
              } else {
                load(dst, &q.a[h], kc, am);
              }
            }
#pragma unroll
            for (int h = 0; h < PARTS; h++, dst += TILE_B) {
              if (RAW && !RAW_A && h == 1) break;
              if (BMN) {
#pragma unroll
                for (int i = 0; i < C::MN_BOXES_B; i++)
                  if (i < boxes_b) load(dst + i * C::MN_BOX, &q.b[h], nb + Ty::KROW * i, kc);
              } else {
                load(dst, &q.b[h], kc, nb);
              }
            }
          }
        }
      }
      if (!ok) settle();
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {  // the pair's MMAs are issued by the even CTA
      uint32_t kbg = 0, cg = 0;
      bool ok = true;
      const uint32_t base = smem_u32(smem);
      for (int k = 0; ok && work_at(p, unit, k, w); k++) {
        const Problem &q = p.p[w.prob];
        const Tile tl = tile_of<C>(q, bn, w.item);
        const bool amn = EPI == kOutT || (EPI == kOut && q.amn);
        const uint64_t adesc = operand_desc<Ty, C>(base, amn), bdesc = operand_desc<Ty, C>(base + PARTS * TILE_A, BMN);
        const uint32_t astep = (amn ? C::MN_STEP : 32u) >> 4, bstep = (BMN ? C::MN_STEP : 32u) >> 4;
        const uint32_t idesc = (1u << 4) | Ty::FORMAT | (uint32_t(amn) << 15) | (uint32_t(BMN) << 16) |
                               (uint32_t(bn >> 3) << 17) | (uint32_t(C::TM >> 4) << 24);
        for (int c0 = tl.kb0; c0 < tl.kb1 && ok; c0 += C::CHUNK, cg++) {
          const int c1 = tl.kb1 - c0 < C::CHUNK ? tl.kb1 : c0 + C::CHUNK;
          const uint32_t j = cg % NBUF, use = cg / NBUF;
          if (cg >= uint32_t(NBUF) && !mbar_wait(tempty0 + 8 * j, (use & 1) ^ 1, p.err, 24)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t acc = tmem + j * BN;
          for (int kb = c0; kb < c1; kb++, kbg++) {
            const uint32_t s = kbg % STAGES, ph = (kbg / STAGES) & 1;
            if ((!mbar_try_wait(full0 + 8 * s, ph) && !mbar_wait(full0 + 8 * s, ph, p.err, 22)) ||
                (RAW && !mbar_try_wait(ready0 + 8 * s, ph) && !mbar_wait(ready0 + 8 * s, ph, p.err, 26))) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int u = 0; u < SUBS; u++) {
              const uint32_t off = (s * STAGE_BYTES + u * SUB_BYTES) >> 4;
#pragma unroll
              for (int kk = 0; kk < Ty::KROW / Ty::KMMA; kk++) {
                const uint64_t a = adesc + uint64_t(off + kk * astep), b = bdesc + uint64_t(off + kk * bstep);
                const uint32_t first = (kb == c0 && u == 0 && kk == 0) ? 0u : 1u;
                if constexpr (PARTS == 1) {
                  if (PAIR) mma_f16_pair(acc, a, b, idesc, first);
                  else mma_f16(acc, a, b, idesc, first);
                } else {  // small terms first
                  const uint64_t al = a + uint64_t(TILE_A >> 4), bl = b + uint64_t(TILE_B >> 4);
                  if (PAIR) {
                    mma_tf32_pair(acc, al, b, idesc, first);
                    mma_tf32_pair(acc, a, bl, idesc, 1u);
                    mma_tf32_pair(acc, a, b, idesc, 1u);
                  } else {
                    mma_tf32(acc, al, b, idesc, first);
                    mma_tf32(acc, a, bl, idesc, 1u);
                    mma_tf32(acc, a, b, idesc, 1u);
                  }
                }
              }
            }
            if (PAIR) mma_commit_both(empty0 + 8 * s);  // the stage is free in both CTAs
            else mma_commit(empty0 + 8 * s);
          }
          if (PAIR) mma_commit_both(tfull0 + 8 * j);
          else mma_commit(tfull0 + 8 * j);
        }
      }
      if (!ok) settle();
    }
  } else {
    const int qr = warp & 3, h = (warp - 2) >> 2;
    float *st = reinterpret_cast<float *>(smem + C::RING_BYTES) + (warp - 2) * 1024;
    const int half = RAW || EPI == kOut ? p.half : 128;
    const float alpha = (EPI == kOut || EPI == kOutT) && p.alpha ? *p.alpha : 1.0f;
    uint32_t cg = 0, kbe = 0;
    bool ok = true;
    for (int k = 0; ok && work_at(p, unit, k, w); k++) {
      const Problem &q = p.p[w.prob];
      const Tile tl = tile_of<C>(q, bn, w.item);
      const int r0 = tl.m0 + BM * int(rank) + 32 * qr, c0 = tl.n0 + half * h;
      const int row = r0 + lane;
      // this warp's columns of the tile (may be <= 0)
      const int cols = min(min(q.N, tl.n0 + bn), c0 + half) - c0;
      // RAW: the next `n` stages' remainders x - tf32(x) of the raw operand, for the MMAs.
      // Every warp sees every use of a slot, so no barrier is ever more than one phase ahead
      // of it.
      auto remainders = [&](int n) {
        for (int i = 0; i < n; i++, kbe++) {
          const uint32_t s = kbe % STAGES;
          if (!__all_sync(0xffffffffu, wait_inline(full0 + 8 * s, (kbe / STAGES) & 1, p.err, 25))) return false;
          const int tile = RAW_A ? TILE_A : TILE_B;
          float4 *hi = reinterpret_cast<float4 *>(smem + s * STAGE_BYTES + (RAW_A ? 0 : 2 * TILE_A)), *lo = hi + tile / 16;
          for (int e = int(threadIdx.x) - 64; e < tile / 16; e += 32 * C::EPI_WARPS) {
            float4 x = hi[e];
            x.x = remainder_of(x.x);
            x.y = remainder_of(x.y);
            x.z = remainder_of(x.z);
            x.w = remainder_of(x.w);
            lo[e] = x;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(ready0 + 8 * s);
        }
        return true;
      };
      auto finished = [&](uint32_t t) {  // the accumulator of chunk t is complete
        const uint32_t j = t % NBUF, use = t / NBUF;
        const bool got = __all_sync(0xffffffffu, wait_inline(tfull0 + 8 * j, use & 1, p.err, 23));
        tc_fence_after();
        return got;
      };
      auto release = [&](uint32_t t) {  // the MMAs may write it again
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          const uint32_t bar = tempty0 + 8 * (t % NBUF);
          if (PAIR) mbar_arrive_cluster_relaxed(mapa_shared(bar, 0));
          else mbar_arrive(bar);
        }
      };
      // What the epilogue needs of the row: asked for while the MMAs run, where
      // three registers are left beside the sums.
      constexpr bool EARLY = PARTS == 1 || !C::BACK;
      int y = -1;
      float lse = 0.f, g = 0.f;
      auto row_data = [&] {
        if ((EPI == kStats || EPI == kScoreGrad) && row < q.M) {
          y = max(p.loss.targets[row], -1);  // any negative one; differences with it do not overflow
          if (EPI == kScoreGrad) {
            lse = p.loss.lse[row] * kLog2e;
            g = p.loss.scale ? p.loss.scale[p.loss.per_row ? row : 0] : 1.0f;
          }
        }
        if (EPI == kOut && PARTS == 1) y = p.alpha && q.of_rows && row < q.M ? p.loss.targets[row] : 0;
      };
      if (EARLY) row_data();
      const uint32_t src0 = tmem + (uint32_t(32 * qr) << 16) + half * h;
      float acc[128];
      if (C::SUMS || tl.kb1 - tl.kb0 > C::CHUNK) {
        int kc = tl.kb0;
        if constexpr (C::SUMS && PARTS == 1) {  // the first chunk lands in the sums' registers
          ok = finished(cg);
          if (ok && cols > 0) {
#pragma unroll
            for (int cb = 0; cb < 128; cb += 32) tmem_ld_cols<32>(src0 + (cg % NBUF) * BN + cb, acc, cb);
            tmem_ld_done(acc);
          }
          if ((kc += C::CHUNK) < tl.kb1) release(cg++);
        } else {
#pragma unroll
          for (int i = 0; i < 128; i++) acc[i] = 0.f;
        }
        if (RAW) ok = remainders(min(C::CHUNK, tl.kb1 - kc));
        while (ok && kc < tl.kb1) {
          // the next chunk's remainders before this chunk's sums: its MMAs can start
          if (RAW && kc + C::CHUNK < tl.kb1) ok = remainders(min(C::CHUNK, tl.kb1 - kc - C::CHUNK));
          ok = ok && finished(cg);
          if (ok && cols > 0) {
#pragma unroll
            for (int cb = 0; cb < 128; cb += C::LD) {
              if (EPI == kOutT && cb >= cols) break;
              float r[C::LD];
              tmem_ld_cols<C::LD>(src0 + (cg % NBUF) * BN + cb, r);
              tmem_ld_done(r);
#pragma unroll
              for (int i = 0; i < C::LD; i++) acc[cb + i] = __fadd_rn(acc[cb + i], r[i]);
            }
          }
          if ((kc += C::CHUNK) < tl.kb1) release(cg++);
        }
        if constexpr (C::BACK) {
          if (ok && cols > 0) {
#pragma unroll
            for (int cb = 0; cb < 4; cb++) {
              if (32 * cb >= cols) break;  // the other warp's columns may still hold its last chunk
              uint32_t r[32];
#pragma unroll
              for (int i = 0; i < 32; i++) r[i] = __float_as_uint(acc[32 * cb + i]);
              tmem_st32_cols(src0 + (cg % NBUF) * BN + 32 * cb, r);
            }
            tmem_st_wait();
          }
        } else {
          release(cg);
        }
      } else {
        ok = finished(cg);
      }
      cg++;
      if (!ok) break;  // a wait gave up; ok is the same in all lanes
      if (!EARLY) row_data();
      constexpr bool IN_REGS = !C::BACK;
      // Columns 32 cb .. 32 cb + 31 of this thread's row, for cb = 0, 1, 2, 3 in
      // turn; from TMEM the next ones are on their way while these are used.
      float ahead[IN_REGS ? 1 : 32];
      if constexpr (!IN_REGS) tmem_ld_cols<32>(src0 + ((cg - 1) % NBUF) * BN, ahead);
      auto block = [&](int cb, float (&v)[32]) {
        if constexpr (IN_REGS) {
#pragma unroll
          for (int i = 0; i < 32; i++) v[i] = acc[32 * cb + i];
        } else {
          tmem_ld_done(ahead);
#pragma unroll
          for (int i = 0; i < 32; i++) v[i] = ahead[i];
          if (cb < 3) tmem_ld_cols<32>(src0 + ((cg - 1) % NBUF) * BN + 32 * (cb + 1), ahead);
        }
      };
      // 16-byte chunk i of this lane's row in the staging block: 32 rows of 128
      // bytes, chunks swizzled by the row.
      auto put = [&](int i, uint4 v) {
        *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(st) + lane * 128 + 16 * (i ^ (lane & 7))) = v;
      };
      // The staged block to rows r0.. of `out` from column col0 on, 8 lanes a row.  A
      // lane with at least `whole` columns from its own on writes vector(address, 16
      // bytes), one with fewer single(address, 16 bytes, columns).  Several vectors are
      // read before the first is written: one by one they took 150 cycles each, and
      // the epilogue of a short product was all there was (dW of 30 rows of 60000 x
      // 3000, bf16: 156 us).
      constexpr int AT_ONCE = PARTS == 2 && EPI == kScoreGrad ? 4 : 8;  // eight spill there
      const int rows_left = q.M - r0 - (lane >> 3);
      auto send = [&](auto *out, int64_t ld, int col0, int whole, auto &&vector, auto &&single) {
        constexpr int W = 16 / int(sizeof(*out));
        const int ch = lane & 7, left = c0 + cols - col0 - W * ch;
        auto *dst = out + int64_t(r0 + (lane >> 3)) * ld + col0 + W * ch;
        const char *src = reinterpret_cast<const char *>(st) + (lane >> 3) * 128;
        const int even = 16 * (ch ^ (lane >> 3)), odd = 16 * (ch ^ ((lane >> 3) + 4));
        __syncwarp();
#pragma unroll
        for (int i0 = 0; i0 < 8; i0 += AT_ONCE) {
          uint4 x[AT_ONCE];
#pragma unroll
          for (int i = 0; i < AT_ONCE; i++)
            x[i] = *reinterpret_cast<const uint4 *>(src + 512 * (i0 + i) + (i & 1 ? odd : even));
          if (i0 + AT_ONCE == 8) __syncwarp();
          if (left >= whole) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++, dst += 4 * ld)
              if (4 * (i0 + i) < rows_left) vector(dst, x[i]);
          } else if (left > 0) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++, dst += 4 * ld)
              if (4 * (i0 + i) < rows_left) single(dst, x[i], left);
          }
        }
      };
      constexpr int UNROLL = IN_REGS ? 4 : 1;

      if constexpr (EPI == kStats) {
        if (r0 < q.M) {
          float m, l;
          if (cols >= 128) softmax_part(acc, 128, m, l);
          else softmax_part(acc, cols, m, l);
          const int at = y - p.loss.v0 - c0;  // the target among this thread's columns
          if (counts(y, p.loss.V) && at >= 0 && at < min(cols, 128)) {
#pragma unroll
            for (int i = 0; i < 128; i++)
              if (i == at) p.loss.target_score[row] = acc[i];
          }
          if (row < q.M) p.loss.part[int64_t(p.part0 + 2 * (tl.n0 / bn) + h) * q.M + row] = make_float2(m, l);
        }
      } else if constexpr (EPI == kScoreGrad) {
        if (r0 < q.M) {
          const bool used = counts(y, p.loss.V);
          const int at = y - p.loss.v0 - c0;
          // plain stores need no wait before the next block; rows of ds end on whole vectors
          auto store = [](T *dst, const uint4 &x) { *reinterpret_cast<uint4 *>(dst) = x; };
          auto none = [](T *, const uint4 &, int) {};
#pragma unroll UNROLL
          for (int cb = 0; cb < 4; cb++) {
            if (32 * cb < cols) {
              float v[32];
              block(cb, v);
              score_gradient(v, lse, g, at - 32 * cb, used);
              if constexpr (PARTS == 1) {  // 64 bf16 columns per 128-byte row: two blocks a store
#pragma unroll
                for (int i = 0; i < 4; i++)
                  put(4 * (cb & 1) + i, make_uint4(pack_bf16(v[8 * i], v[8 * i + 1]), pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                                                   pack_bf16(v[8 * i + 4], v[8 * i + 5]),
                                                   pack_bf16(v[8 * i + 6], v[8 * i + 7])));
                if ((cb & 1) || 32 * (cb + 1) >= cols) send(static_cast<T *>(p.ds[0]), p.lds, c0 + 32 * (cb & ~1), 1, store, none);
              } else {  // the exact tf32 pair, 32 columns per row each
#pragma unroll
                for (int part = 0; part < 2; part++) {
#pragma unroll
                  for (int i = 0; i < 8; i++) {
                    uint32_t e[4];
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                      const float x = v[4 * i + t], hi = tf32_rna_bits(x);
                      e[t] = __float_as_uint(part ? __fsub_rn(x, hi) : hi);
                    }
                    put(i, make_uint4(e[0], e[1], e[2], e[3]));
                  }
                  send(static_cast<T *>(p.ds[part]), p.lds, c0 + 32 * cb, 1, store, none);
                }
              }
            }
          }
        }
      } else if constexpr (EPI == kOutT) {  // 32 lanes hold 32 neighbours of an output row
#pragma unroll UNROLL
        for (int cb = 0; cb < 4; cb++) {
          if (32 * cb < cols) {
            float v[32];
            block(cb, v);
            uint32_t left_out = 0;  // of the block's 32 output rows
            if (PARTS == 1 && q.mode == kDirect && p.alpha)
              left_out = __ballot_sync(0xffffffffu, lane < cols - 32 * cb &&
                                                        !counts(p.loss.targets[c0 + 32 * cb + lane], p.loss.V));
            if (row < q.M) {
              const int64_t at = int64_t(c0 + 32 * cb) * q.ldo + row;
#pragma unroll
              for (int i = 0; i < 32; i++) {
                if (32 * cb + i < cols) {
                  if (q.mode == kDirect) store_as(static_cast<T *>(q.out) + at + i * q.ldo, left_out >> i & 1 ? 0.f : alpha * v[i]);
                  else if (q.mode == kPlane) static_cast<float *>(q.out)[tl.part * q.plane + at + i * q.ldo] = v[i];
                  else red_add(static_cast<float *>(q.out) + tl.part * q.plane + at + i * q.ldo, v[i]);
                }
              }
            }
          }
        }
      } else if (r0 < q.M) {
        const int mode = q.mode;
        if (PARTS == 1) g = p.alpha && !counts(y, p.loss.V) ? 0.f : alpha;
        const bool direct16 = mode == kDirect && PARTS == 1;
        const int64_t ldo = q.ldo;
        float *out = static_cast<float *>(q.out) + tl.part * q.plane;
        // planes' rows hold whole vectors; results' may end or lie elsewhere
        const int whole = mode != kDirect ? 1 : q.vec ? 16 / int(sizeof(T)) : 1 << 30;
#pragma unroll UNROLL
        for (int cb = 0; cb < 4; cb++) {
          if (32 * cb < cols) {
            float v[32];
            block(cb, v);
            if (direct16) {  // 64 bf16 columns per staged row: two blocks a store
#pragma unroll
              for (int i = 0; i < 4; i++)
                put(4 * (cb & 1) + i,
                    make_uint4(pack_bf16(g * v[8 * i], g * v[8 * i + 1]), pack_bf16(g * v[8 * i + 2], g * v[8 * i + 3]),
                               pack_bf16(g * v[8 * i + 4], g * v[8 * i + 5]), pack_bf16(g * v[8 * i + 6], g * v[8 * i + 7])));
              if ((cb & 1) || 32 * (cb + 1) >= cols)
                send(
                    static_cast<unsigned short *>(q.out), ldo, c0 + 32 * (cb & ~1), whole,
                    [](unsigned short *dst, const uint4 &x) { *reinterpret_cast<uint4 *>(dst) = x; },
                    [](unsigned short *dst, const uint4 &x, int left) {
                      const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                      for (int t = 0; t < 8; t++)
                        if (t < left) dst[t] = static_cast<unsigned short>(e[t >> 1] >> (16 * (t & 1)));
                    });
            } else {  // 32 fp32 columns
#pragma unroll
              for (int i = 0; i < 8; i++)
                put(i, make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                                  __float_as_uint(v[4 * i + 3])));
              auto single = [](float *dst, const uint4 &x, int left) {
                const uint32_t e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int t = 0; t < 4; t++)
                  if (t < left) dst[t] = __uint_as_float(e[t]);
              };
              if (mode == kPlaneAdd)
                send(out, ldo, c0 + 32 * cb, whole, [](float *dst, const uint4 &x) { red_add4(dst, x); }, single);
              else
                send(out, ldo, c0 + 32 * cb, whole, [](float *dst, const uint4 &x) { *reinterpret_cast<uint4 *>(dst) = x; },
                     single);
            }
          }
        }
      }
      if constexpr (!IN_REGS) {
        tmem_ld_wait();  // a load that no block took
        release(cg - 1);
      }
    }
    if (!ok) settle();
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();  // no CTA frees TMEM or leaves while its peer may still use the pair
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------- host side
// An operand in memory: [MN, k] rows, or with `mn` [k, MN] rows; the row
// stride in elements.  Pointers and row strides are multiples of 16 bytes.
struct Operand {
  const void *p, *lo;  // lo: the tf32 pair's (null for bf16 and raw fp32)
  int64_t ld, ldlo;
  bool mn;
};

template <typename Ty>
bool operand_map(CUtensorMap (&m)[2], const Operand &o, int64_t extent, int64_t K, int rows) {
  for (int h = 0; h < (o.lo ? 2 : 1); h++) {
    const void *p = h ? o.lo : o.p;
    const int64_t ld = h ? o.ldlo : o.ld;
    const bool ok = o.mn ? make_map2<typename Ty::T>(&m[h], p, extent, K, ld, Ty::KROW, Ty::KROW, Ty::PARTS == 2)
                         : make_map2<typename Ty::T>(&m[h], p, K, extent, ld, Ty::KROW, rows, false);
    if (!ok) return false;
  }
  return true;
}

template <typename Ty>
bool set_problem(Problem &q, bool pair, int bn, int rows_a, int64_t M, int64_t N, int64_t K, const Operand &a,
                 const Operand &b) {
  q.M = int(M);
  q.N = int(N);
  q.K = int(K);
  const int TM = pair ? 2 * BM : BM;
  q.tiles_m = int((M + TM - 1) / TM);
  q.tiles_n = int((N + bn - 1) / bn);
  q.ksplit = 1;
  q.amn = a.mn;
  return operand_map<Ty>(q.a, a, M, K, rows_a) && operand_map<Ty>(q.b, b, N, K, pair ? bn / 2 : bn);
}

inline int64_t items_of(const Problem &q) { return int64_t(q.tiles_m) * q.tiles_n * q.ksplit; }

template <typename Ty, int EPI, bool PAIR, bool RAW = false>
silcu_status launch(Params &p, int problems, cudaStream_t s) {
  using C = Cfg<Ty, EPI, PAIR, RAW>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm<Ty, EPI, PAIR, RAW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               C::SMEM_BYTES);
    if (e != cudaSuccess) return fail(SILCU_CUDA_ERROR, "cross_entropy: smem attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int64_t n0 = items_of(p.p[0]), n1 = problems > 1 ? items_of(p.p[1]) : 0;
  if (n0 + n1 > 0x3FFFFFFF) return fail(SILCU_UNSUPPORTED, "cross_entropy: too many tiles");
  const int64_t most = PAIR ? sm_count() / 2 : sm_count();
  p.n0 = int(n0);
  p.n1 = int(n1);
  p.units = int(n0 + n1 < most ? n0 + n1 : most);
  p.rounds = int(n0 / p.units);
  p.tail = int(n0 % p.units);
  for (int i = 0; i < problems; i++) {
    Problem &q = p.p[i];
    q.by_split.set(q.ksplit);
    q.by_group.set(C::GROUP_M * q.tiles_n);
    q.by_last.set(q.tiles_m % C::GROUP_M ? q.tiles_m % C::GROUP_M : C::GROUP_M);
  }
  p.extra = 0;
  if (n1 && p.tail) {  // an item of the first product in items of the second, by their k
    const double c0 = double(p.p[0].K) / p.p[0].ksplit, c1 = double(p.p[1].K) / p.p[1].ksplit;
    p.extra = int(c0 / c1 + 0.5);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t(p.units * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = PAIR ? 2 : 1;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // see launch_after
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm<Ty, EPI, PAIR, RAW>, p);
  if (e != cudaSuccess) return fail(SILCU_CUDA_ERROR, "cross_entropy: launch: %s", cudaGetErrorString(e));
  return check_launch("cross_entropy");
}

}  // namespace lossmm
}  // namespace silcu
