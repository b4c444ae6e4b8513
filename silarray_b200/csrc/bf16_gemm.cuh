// The bf16 tensor-core products of the cross entropy (sm_100a).
//
// One persistent kernel, D[M, N] = A . B in tcgen05.mma kind::f16 with fp32
// accumulation in TMEM, for operands in either major order (AMN / BMN: the M /
// N index is the contiguous one in memory, else k is):
//   warp 0      TMA producer: 64-k stages, 128-byte swizzle;
//   warp 1      allocates the 512 TMEM columns (two accumulators of 256) and
//               issues the MMAs from one thread;
//   warps 2-9   epilogue, two per TMEM lane quarter, 128 columns each, on one
//               accumulator while the MMAs fill the other.
// Tiles are 128 x 256 per CTA, or 256 x 256 per CTA pair (cta_group::2: each
// CTA loads its 128 rows of A and 128 columns of B).
// Epilogues: the cross entropy's statistics, its score gradients (bf16, TMA
// stores), or a plain result: bf16, or fp32 planes that later launches add to.
// Every wait is bounded; on expiry the kernel records a code, unwinds, frees
// its TMEM and exits.
#pragma once

#include <cuda.h>

#include "elem.cuh"
#include "loss_epilogue.cuh"
#include "tc_common.cuh"

namespace silcu {
namespace bf16 {
using namespace tc;

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int GROUP_M = 8;

enum Epilogue { kStats = 0, kScoreGrad = 1, kOut = 2 };
enum OutMode { kOutBf16 = 0, kOutPlane = 1, kOutPlaneAdd = 2 };

template <bool PAIR>
struct Cfg {
  static constexpr int TM = PAIR ? 2 * BM : BM;
  static constexpr int ROWS_B = PAIR ? BN / 2 : BN;
  static constexpr int TILE_A = BM * BK * 2;
  static constexpr int TILE_B = ROWS_B * BK * 2;
  static constexpr int STAGE_BYTES = TILE_A + TILE_B;
  static constexpr int STAGES = 192 * 1024 / STAGE_BYTES;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES;
  static constexpr int EPI_WARPS = 8;
  static constexpr int STAGING = EPI_WARPS * 4096;
  static constexpr int SMEM_BYTES = RING_BYTES + STAGING + 1024 + 512;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int NBUF = 2;
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

struct __align__(64) Params {
  CUtensorMap a, b, c;  // c: the score gradients' stores
  int M, N, K, tiles_m, tiles_n;
  int ksplit;  // each tile's K range in this many parts (kOut; part p -> plane p)
  LossArgs loss;
  void *out;
  int64_t ldo, plane;  // row stride; elements from one plane to the next
  int mode;
  int vec;  // kOutBf16: rows are 16-byte aligned
  int *err;
};

struct Tile {
  int m0, n0;
};

template <int TM>
__device__ __forceinline__ Tile tile_at(const Params &p, int t) {
  const int group = t / (GROUP_M * p.tiles_n);
  const int first = group * GROUP_M;
  const int gm = p.tiles_m - first < GROUP_M ? p.tiles_m - first : GROUP_M;
  const int r = t - group * GROUP_M * p.tiles_n;
  return Tile{(first + r % gm) * TM, (r / gm) * BN};
}

template <bool AMN, bool BMN, int EPI, bool PAIR>
__global__ void __launch_bounds__(Cfg<PAIR>::THREADS, 1) gemm(const __grid_constant__ Params p) {
  using C = Cfg<PAIR>;
  constexpr int STAGES = C::STAGES, NBUF = C::NBUF, TILE_A = C::TILE_A, STAGE_BYTES = C::STAGE_BYTES;
  constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(AMN) << 15) | (uint32_t(BMN) << 16) |
                             (uint32_t(BN >> 3) << 17) | (uint32_t(C::TM >> 4) << 24);
  constexpr uint32_t MN_BOX = 64 * BK * 2;  // bytes of one 64-element x BK box of an MN-major operand
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::RING_BYTES + C::STAGING);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 2 * NBUF);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
  const uint32_t tfull0 = smem_u32(bars + 2 * STAGES), tempty0 = smem_u32(bars + 2 * STAGES + NBUF);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int items = p.tiles_m * p.tiles_n * p.ksplit;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const int first = PAIR ? int(blockIdx.x >> 1) : int(blockIdx.x);
  const int step = PAIR ? int(gridDim.x >> 1) : int(gridDim.x);
  const int nk = (p.K + BK - 1) / BK;
  auto k_range = [&](int item, int &kb0, int &kb1) {
    const int64_t part = item % p.ksplit;
    kb0 = int(part * nk / p.ksplit);
    kb1 = int((part + 1) * nk / p.ksplit);
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
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
  if (PAIR) cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t kbg = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step) {
        const Tile tl = tile_at<C::TM>(p, item / p.ksplit);
        const int am = tl.m0 + BM * int(rank), bn = tl.n0 + C::ROWS_B * int(rank);
        int kb0, kb1;
        k_range(item, kb0, kb1);
        for (int kb = kb0; kb < kb1; kb++, kbg++) {
          const uint32_t s = kbg % STAGES, ph = (kbg / STAGES) & 1;
          if (kbg >= uint32_t(STAGES) && !mbar_wait(empty0 + 8 * s, ph ^ 1, p.err, 21)) { ok = false; break; }
          const uint32_t bar = PAIR ? mapa_shared(full0 + 8 * s, 0) : full0 + 8 * s;
          const uint32_t da = smem_u32(smem + s * STAGE_BYTES), db = da + TILE_A;
          const int k = kb * BK;
          // a pair's bytes all complete on the even CTA's barrier
          if (rank == 0) mbar_expect_tx(full0 + 8 * s, (PAIR ? 2 : 1) * STAGE_BYTES);
          auto load = [&](uint32_t dst, const CUtensorMap *map, int c0, int c1) {
            if (PAIR) tma_load_2d_pair(dst, map, bar, c0, c1);
            else tma_load_2d(dst, map, bar, c0, c1);
          };
          if (AMN) {
            load(da, &p.a, am, k);
            load(da + MN_BOX, &p.a, am + 64, k);
          } else {
            load(da, &p.a, k, am);
          }
          if (BMN) {
#pragma unroll
            for (int i = 0; i < C::ROWS_B / 64; i++) load(db + i * MN_BOX, &p.b, bn + 64 * i, k);
          } else {
            load(db, &p.b, k, bn);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      uint32_t kbg = 0, cg = 0;
      bool ok = true;
      for (int item = first; item < items && ok; item += step, cg++) {
        int kb0, kb1;
        k_range(item, kb0, kb1);
        const uint32_t j = cg % NBUF, use = cg / NBUF;
        if (cg >= uint32_t(NBUF) && !mbar_wait(tempty0 + 8 * j, (use & 1) ^ 1, p.err, 24)) break;
        tc_fence_after();
        const uint32_t acc = tmem + j * BN;
        for (int kb = kb0; kb < kb1; kb++, kbg++) {
          const uint32_t s = kbg % STAGES, ph = (kbg / STAGES) & 1;
          if (!mbar_wait(full0 + 8 * s, ph, p.err, 22)) { ok = false; break; }
          tc_fence_after();
          const uint32_t da = smem_u32(smem + s * STAGE_BYTES), db = da + TILE_A;
#pragma unroll
          for (int kk = 0; kk < BK / 16; kk++) {
            // 16 k: 32 bytes along a K-major row, two 8-k groups of an MN-major tile
            const uint64_t a = AMN ? make_desc_mn16(da + kk * 2048, MN_BOX) : make_desc(da + kk * 32);
            const uint64_t b = BMN ? make_desc_mn16(db + kk * 2048, MN_BOX) : make_desc(db + kk * 32);
            const uint32_t accum = (kb == kb0 && kk == 0) ? 0u : 1u;
            if (PAIR) mma_f16_pair(acc, a, b, IDESC, accum);
            else mma_f16(acc, a, b, IDESC, accum);
          }
          if (PAIR) {
            mma_commit_pair(empty0 + 8 * s);
            mma_commit_pair(mapa_shared(empty0 + 8 * s, 1));
          } else {
            mma_commit(empty0 + 8 * s);
          }
        }
        if (PAIR) {
          mma_commit_pair(tfull0 + 8 * j);
          mma_commit_pair(mapa_shared(tfull0 + 8 * j, 1));
        } else {
          mma_commit(tfull0 + 8 * j);
        }
      }
    }
  } else {
    const int q = warp & 3, h = (warp - 2) >> 2;
    float *st = reinterpret_cast<float *>(smem + C::RING_BYTES) + (warp - 2) * 1024;
    uint32_t cg = 0;
    for (int item = first; item < items; item += step, cg++) {
      const Tile tl = tile_at<C::TM>(p, item / p.ksplit);
      const int r0 = tl.m0 + BM * int(rank) + 32 * q, c0 = tl.n0 + 128 * h;
      const int row = r0 + lane;
      const uint32_t j = cg % NBUF, use = cg / NBUF;
      // what the epilogue needs of the row arrives while the MMAs run
      int y = -1;
      float lse = 0.f, g = 0.f;
      if (EPI != kOut && row < p.M) {
        y = p.loss.targets[row];
        if (EPI == kScoreGrad) {
          lse = p.loss.lse[row] * kLog2e;
          g = p.loss.scale[row];
        }
      }
      const bool w = __all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * j, use & 1, p.err, 23));
      if (!w || !__all_sync(0xffffffffu, *reinterpret_cast<volatile int *>(p.err) == 0)) break;
      tc_fence_after();
      const uint32_t src = tmem + (uint32_t(32 * q) << 16) + j * BN + 128 * h;
      const bool live = r0 < p.M && c0 < p.N;  // warp-uniform: something of this block exists
      if (EPI == kStats) {
        if (live) {
          float m = -INFINITY, l = 0.f;
          const int at = y - p.loss.v0 - c0;  // the target among this thread's 128 columns
          const bool mine = row < p.M && y >= 0 && y < p.loss.V && at >= 0 && at < 128;
#pragma unroll 1
          for (int cb = 0; cb < 4 && c0 + 32 * cb < p.N; cb++) {
            uint32_t r[32];
            tmem_ld32_nowait(src + 32 * cb, r);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
            const int valid = p.N - c0 - 32 * cb;
            if (valid >= 32) softmax_fold(v, 0, 32, m, l);
            else softmax_fold(v, 0, valid, m, l);
            const int d = at - 32 * cb;
            if (__any_sync(0xffffffffu, mine && d >= 0 && d < 32)) {
#pragma unroll
              for (int i = 0; i < 32; i++)
                if (mine && i == d) p.loss.target_score[row] = v[i];
            }
          }
          if (row < p.M) p.loss.part[int64_t((p.loss.v0 + c0) >> 7) * p.M + row] = make_float2(m, l);
        }
      } else if (EPI == kScoreGrad) {
        if (live) {
          const bool counts = y >= 0 && y < p.loss.V;
          const int at = y - p.loss.v0 - c0;
#pragma unroll 1
          for (int cb = 0; cb < 4 && c0 + 32 * cb < p.N; cb += 2) {
            uint32_t r[32], packed[32];
#pragma unroll
            for (int half = 0; half < 2; half++) {
              tmem_ld32_nowait(src + 32 * (cb + half), r);
              tmem_ld_wait();
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
              score_gradient(v, 0, lse, g, at - 32 * (cb + half), counts);
#pragma unroll
              for (int i = 0; i < 16; i++) packed[16 * half + i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            }
            if (lane == 0) bulk_wait_read0();  // the staging block's last store has read it
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; i++)
              *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(st) + lane * 128 + 16 * (i ^ (lane & 7))) =
                  make_uint4(packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&p.c, smem_u32(st), c0 + 32 * cb, r0);
              bulk_commit();
            }
          }
        }
      } else if (live) {
        const bool f32 = p.mode != kOutBf16;
        const int part = item % p.ksplit;
#pragma unroll 1
        for (int cb = 0; cb < 4 && c0 + 32 * cb < p.N; cb++) {
          uint32_t r[32];
          tmem_ld32_nowait(src + 32 * cb, r);
          tmem_ld_wait();
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; i++)
            *reinterpret_cast<uint4 *>(st + lane * 32 + 4 * (i ^ (lane & 7))) =
                make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
          __syncwarp();
          const int col0 = c0 + 32 * cb;
          if (f32) {  // 8 lanes per row, 16 bytes each
            float *plane = static_cast<float *>(p.out) + part * p.plane;
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int rr = 4 * i + (lane >> 3), ch = lane & 7;
              float4 v = *reinterpret_cast<const float4 *>(st + rr * 32 + 4 * (ch ^ (rr & 7)));
              if (r0 + rr < p.M && col0 + 4 * ch < p.N) {
                float4 *dst = reinterpret_cast<float4 *>(plane + int64_t(r0 + rr) * p.ldo + col0 + 4 * ch);
                if (p.mode == kOutPlaneAdd) {
                  const float4 o = *dst;
                  v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
                }
                *dst = v;
              }
            }
          } else {  // 4 lanes per row, 8 columns each
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int rr = 8 * i + (lane >> 2), ch = 2 * (lane & 3);
              const float4 v = *reinterpret_cast<const float4 *>(st + rr * 32 + 4 * (ch ^ (rr & 7)));
              const float4 u = *reinterpret_cast<const float4 *>(st + rr * 32 + 4 * ((ch + 1) ^ (rr & 7)));
              const int col = col0 + 4 * ch;
              if (r0 + rr < p.M && col < p.N) {
                __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(p.out) + int64_t(r0 + rr) * p.ldo + col;
                if (p.vec && col + 8 <= p.N) {
                  *reinterpret_cast<uint4 *>(dst) = make_uint4(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w),
                                                               pack_bf16(u.x, u.y), pack_bf16(u.z, u.w));
                } else {
                  const float e[8] = {v.x, v.y, v.z, v.w, u.x, u.y, u.z, u.w};
#pragma unroll
                  for (int k = 0; k < 8; k++)
                    if (col + k < p.N) dst[k] = __float2bfloat16_rn(e[k]);
                }
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive_cluster(mapa_shared(tempty0 + 8 * j, 0));
        else mbar_arrive(tempty0 + 8 * j);
      }
    }
    if (EPI == kScoreGrad) {
      if (lane == 0) bulk_wait_all0();
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------- host side
struct Operand {
  const void *p;
  int64_t ld;
  bool mn;  // stored [k, MN] (the M / N index contiguous), else [MN, k]
};

// Fills the operand maps and the tiling.  Operands' pointers and row strides
// are multiples of 16 bytes.
inline bool set_operands(Params &p, bool pair, int64_t M, int64_t N, int64_t K, const Operand &a, const Operand &b) {
  p.M = int(M);
  p.N = int(N);
  p.K = int(K);
  const int TM = pair ? 2 * BM : BM;
  p.tiles_m = int((M + TM - 1) / TM);
  p.tiles_n = int((N + BN - 1) / BN);
  p.ksplit = 1;
  const int rows_b = pair ? BN / 2 : BN;
  return (a.mn ? make_map2_bf16(&p.a, a.p, M, K, a.ld, 64, BK) : make_map2_bf16(&p.a, a.p, K, M, a.ld, BK, BM)) &&
         (b.mn ? make_map2_bf16(&p.b, b.p, N, K, b.ld, 64, BK) : make_map2_bf16(&p.b, b.p, K, N, b.ld, BK, rows_b));
}

template <bool AMN, bool BMN, int EPI, bool PAIR>
silcu_status launch(const Params &p, cudaStream_t s) {
  using C = Cfg<PAIR>;
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(gemm<AMN, BMN, EPI, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               C::SMEM_BYTES);
    if (e != cudaSuccess) return fail(SILCU_CUDA_ERROR, "cross_entropy: smem attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int64_t units = PAIR ? sm_count() / 2 : sm_count();
  const int64_t items = int64_t(p.tiles_m) * p.tiles_n * p.ksplit;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t((items < units ? items : units) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = PAIR ? 2 : 1;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm<AMN, BMN, EPI, PAIR>, p);
  if (e != cudaSuccess) return fail(SILCU_CUDA_ERROR, "cross_entropy: launch: %s", cudaGetErrorString(e));
  return check_launch("cross_entropy");
}

}  // namespace bf16
}  // namespace silcu
