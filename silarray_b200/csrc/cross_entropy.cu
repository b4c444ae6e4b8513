// Softmax cross entropy of a vocabulary projection, forward and backward,
// without the logits in memory.
//
//   s = H . W^T,  lse_t = log sum_v exp(s_tv),  loss_t = lse_t - s_t,y(t)
//   ds_tv = g_t (exp(s_tv - lse_t) - [v = y(t)]),  dH = ds . W,  dW = ds^T . H
//
// Forward: one tensor-core product whose epilogue keeps, for every row and each half of a
// tile's columns, the maximum and the sum of exponentials (8 bytes in place of 128
// scores; tiles of fewer than 256 columns keep the same two parts) and the target's score;
// loss_finish joins them.
// Backward: piece by piece of the vocabulary, the same product again with the
// score gradients as its epilogue (ds of one piece is all that is kept), then
// dH += ds . W_piece and dW_piece = ds^T . H.  Recomputing the scores costs
// 2 T V D operations on top of the 6 T V D of the forward and the gradients;
// keeping them would take T V values.
// Bound by the tensor cores except for few rows, where reading W is all.
//
// The products run on loss_gemm.cuh: bf16 operands as they are, fp32 ones as
// exact tf32 pairs (3xTF32), split once per call (H) and per piece (W; for few
// rows inside the products, see kRawRows).  With
// bf16, ds is rounded to bf16, the operand type of its two products, once per
// element; the factor that all rows share (the gradient of the mean or the
// sum) multiplies the results instead, so that its own rounding does not.
//
// Rows whose target lies outside [0, V) are left out: the backward pass works
// on a copy of H with those rows zero and gives them ds = 0 by selection, so
// nothing that H holds there reaches dW.
#include <stdlib.h>
#include <string.h>

#include <utility>

#include "loss_gemm.cuh"

namespace silcu {
namespace {

using Args = silcu_cross_entropy_args;

// ------------------------------------------------------------ small kernels
__device__ __forceinline__ double cta_sum(double v, double *sm) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < int(blockDim.x >> 5); i++) s += sm[i];
  __syncthreads();
  return s;
}

// Number of rows that count, in every thread of the CTA.
__device__ __forceinline__ double count_rows(const int32_t *targets, int64_t rows, int V, double *sm) {
  int n = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) {
    const int y = targets[i];
    n += y >= 0 && y < V;
  }
  return cta_sum(double(n), sm);
}

// Joins a row's parts, lse = M + log sum l_i exp(m_i - M), and with `total`
// the rows' losses to their sum, or their mean over the rows that count (0 when
// none does).  A CTA takes 8 rows and has 128 threads for the parts of each;
// 8 rows of 294 parts took 4.6 us with 32 threads a row and a chain of 31 joins at its
// end.  The CTA that finishes last adds the losses, in row order whichever it
// is: `done` counts the CTAs, and the scores' launch has set it to 0.
constexpr int kFinishRows = 8;
__global__ void __launch_bounds__(1024) loss_finish(const float2 *part, int nparts, int64_t rows, const int32_t *targets,
                                                    int V, const float *target_score, float *lse, float *loss, int mean,
                                                    unsigned *done, float *total) {
  __shared__ float2 sm[32][kFinishRows];
  __shared__ double sums[32];
  __shared__ int counts[32];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row0 = int64_t(blockIdx.x) * kFinishRows, row = row0 + (lane & 7);
  let_next_start();
  wait_for_previous();
  // what the row's result needs of it, on its way early (an unwritten score is not used)
  const int64_t mine = row0 + warp;
  int y = -1;
  float score = 0.f;
  if (warp < kFinishRows && mine < rows) {
    y = targets[mine];
    score = target_score[mine];
  }
  float m = -INFINITY, l = 0.f;
  auto join = [&](float om, float ol) {
    const float mx = fmaxf(m, om);
    const float ref = mx == -INFINITY ? 0.f : mx;
    l = l * ex2((m - ref) * kLog2e) + ol * ex2((om - ref) * kLog2e);
    m = mx;
  };
  if (row < rows) {
#pragma unroll 4
    for (int i = threadIdx.x >> 3; i < nparts; i += 128) {
      const float2 x = load_streaming(part + int64_t(i) * rows + row);
      join(x.x, x.y);
    }
  }
  auto across = [&](int step) {
    const float om = __shfl_xor_sync(0xffffffffu, m, step), ol = __shfl_xor_sync(0xffffffffu, l, step);
    join(om, ol);
  };
  across(8);
  across(16);
  if (lane < kFinishRows) sm[warp][lane] = make_float2(m, l);
  __syncthreads();
  if (warp < kFinishRows) {
    m = sm[lane][warp].x, l = sm[lane][warp].y;
#pragma unroll
    for (int step = 1; step < 32; step *= 2) across(step);
    if (lane == 0 && mine < rows) {
      const float v = m + logf(l);
      lse[mine] = v;
      loss[mine] = y >= 0 && y < V ? v - score : 0.f;
    }
  }
  if (!total) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(done, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
  double s = 0.0;
  int n = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    const int t = targets[i];
    s += double(load_l2(loss + i));
    n += t >= 0 && t < V;
  }
  s = warp_sum(s);
  n = warp_sum(n);
  if (lane == 0) sums[warp] = s, counts[warp] = n;
  __syncthreads();
  if (warp == 0) {
    s = warp_sum(sums[lane]);
    n = warp_sum(counts[lane]);
    if (mean) s = n > 0 ? s / double(n) : 0.0;
    if (lane == 0) *total = float(s);
  }
}

// The factor that the gradients of a mean or a sum share: 0 when no row counts.
struct Shared {
  const float *dloss;
  int reduction;
  float *factor;  // null: not wanted
};
__device__ __forceinline__ void shared_factor(const Shared &c, const int32_t *targets, int64_t rows, int V) {
  __shared__ double sm[32];
  const double d = c.dloss ? double(*c.dloss) : 1.0;
  double f = d;
  // of a sum only a factor that is not finite would make something of the zeros of no rows
  if (c.reduction == SILCU_REDUCE_MEAN || !isfinite(d)) {
    const double n = count_rows(targets, rows, V, sm);
    f = n == 0.0 ? 0.0 : c.reduction == SILCU_REDUCE_MEAN ? d / n : d;
  }
  if (threadIdx.x == 0) *c.factor = float(f);
}

// dst [rows, dp] = src [rows, D] (row stride ld), columns D.. zero; with
// targets, rows that are left out are zero as well.  With `lo`, dst and lo
// take the exact tf32 pair; with `lo` alone, src itself is to be the hi operand (the
// tensor core reads its upper 19 bits) and lo takes what that leaves.  The first CTA
// writes the shared factor where it is wanted.
template <typename T>
__global__ void __launch_bounds__(256) copy_rows(const T *src, int64_t ld, int64_t rows, int D, int dp,
                                                 const int32_t *targets, int V, T *dst, float *lo, const Shared shared) {
  constexpr int W = 16 / sizeof(T);
  const int per_row = dp / W;
  const bool vec = ld % W == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  const int64_t n = rows * per_row;
  const int first = shared.factor ? 1 : 0;
  let_next_start();
  wait_for_previous();
  if (first && blockIdx.x == 0) {
    shared_factor(shared, targets, rows, V);
    return;
  }
  for (int64_t i = int64_t(blockIdx.x - first) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x - first) * 256) {
    const int64_t r = i / per_row;
    const int c = int(i - r * per_row) * W;
    Raw<T, W> v = raw_zero<T, W>();
    bool keep = true;
    if (targets) {
      const int y = targets[r];
      keep = y >= 0 && y < V;
    }
    if (keep) {
      if (vec && c + W <= D) {
        v = raw_load<T, W>(src + r * ld + c);
      } else {
        T e[W] = {};
#pragma unroll
        for (int k = 0; k < W; k++)
          if (c + k < D) e[k] = src[r * ld + c + k];
        memcpy(&v, e, sizeof(v));
      }
    }
    if constexpr (sizeof(T) == 4) {
      float x[4], l[4];
      unpack(v, x);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float h = dst ? tc::tf32_rna(x[k]) : lossmm::tf32_trunc(x[k]);
        l[k] = __fsub_rn(x[k], h);
        if (!dst) l[k] = tc::tf32_rna(l[k]);  // 13 bits, of which the tensor core would cut two
        x[k] = h;
      }
      pack(x, v);
      store_f32<4>(lo + r * dp + c, l);
    }
    if (sizeof(T) == 2 || dst) *reinterpret_cast<decltype(v.r) *>(dst + r * dp + c) = v.r;
  }
}

// out [rows, D] = alpha times the sum of the fp32 planes [rows, ldp] (with targets, 0 for rows
// that are left out, whatever alpha is), in plane order, or for few elements of many planes by WAYS neighbouring lanes
// that take turns at the planes (16 planes of 100 x 1024: 9 us by one thread).
template <typename T, int WAYS>
__global__ void __launch_bounds__(256) planes_finish(const float *planes, int nplanes, int64_t plane, int64_t rows, int D,
                                                     int ldp, const float *alpha, const int32_t *targets, int V, T *out,
                                                     int64_t ldo, int vec) {
  constexpr int W = 16 / sizeof(T);
  const int per_row = (D + W - 1) / W;
  const int64_t n = rows * per_row;
  const int way = threadIdx.x % WAYS;
  let_next_start();
  wait_for_previous();
  const float k0 = alpha ? *alpha : 1.0f;
  for (int64_t i0 = int64_t(blockIdx.x) * (256 / WAYS); i0 < n; i0 += int64_t(gridDim.x) * (256 / WAYS)) {
    const int64_t i = i0 + threadIdx.x / WAYS, r = i / per_row;
    const int c = int(i - r * per_row) * W;
    float f[W] = {};
    int y = 0;
    if (i < n) {
      if (targets) y = targets[r];
      const float *src = planes + r * ldp + c;  // ldp is a multiple of W: the last vectors stay inside the row
      constexpr int AHEAD = 32 / W;             // planes on their way at a time
      for (int p = way; p < nplanes; p += AHEAD * WAYS) {
        float v[AHEAD][W];
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
          if (p + j * WAYS < nplanes) load_f32<W>(src + (p + j * WAYS) * plane, v[j]);
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
          if (p + j * WAYS < nplanes) {
#pragma unroll
            for (int k = 0; k < W; k++) f[k] += v[j][k];
          }
      }
    }
#pragma unroll
    for (int step = 1; step < WAYS; step *= 2) {
#pragma unroll
      for (int k = 0; k < W; k++) f[k] += __shfl_xor_sync(0xffffffffu, f[k], step);
    }
    if (i >= n || way) continue;
    const float factor = lossmm::counts(y, V) ? k0 : 0.0f;
#pragma unroll
    for (int k = 0; k < W; k++) f[k] *= factor;
    T *dst = out + r * ldo + c;
    Raw<T, W> o;
    pack(f, o);
    if (vec && c + W <= D) {
      *reinterpret_cast<decltype(o.r) *>(dst) = o.r;
    } else {
      T e[W];
      memcpy(e, &o, sizeof(o));
#pragma unroll
      for (int k = 0; k < W; k++)
        if (c + k < D) dst[k] = e[k];
    }
  }
}

uint32_t stream_grid(int64_t items) {
  const int64_t g = (items + 255) / 256, cap = int64_t(sm_count()) * 16;
  return uint32_t(g < 1 ? 1 : g < cap ? g : cap);
}

// --------------------------------------------------------------------- plan
using lossmm::Bf16;
using lossmm::Operand;
using lossmm::Tf32;

// Elements of a piece's ds, and of its copied weights: 128 MB of bf16, 512 MB of tf32 pairs.
// Each piece ends its two launches on a round of tiles that is not full, and adds to dH's planes;
// 2^26 scores are 1024 tiles of 256 x 256, 14 rounds of 74 pairs.  The L2 plays no part.  The
// backward passes of 16 shapes (both types, 512 to 32768 rows, 20000 to 131072 columns, D 512
// to 4096) took, against each one's best piece, 6 % more on average with 2^25 scores, 3 % with 2^26
// (11 % at most), 2 % with 2^27, which would double the memory.
constexpr int64_t kPieceElements = int64_t(1) << 26;

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }

// Columns per piece at most, from SILCU_LOSS_PIECE (tests, tuning).  An entry point reads
// it once and plans once: the plan whose size it checks is the one it runs.
int64_t piece_limit() {
  const char *e = getenv("SILCU_LOSS_PIECE");
  if (!e) return INT64_MAX;
  const int64_t want = atoll(e);
  return up(want < 1 ? 1 : want < (1 << 24) ? want : 1 << 24, 256);
}

// Vocabulary columns per piece: a multiple of 256 that stays within the limit at
// `elements` per column, and pieces of about equal size.
int64_t piece_of(int64_t V, int64_t elements, int64_t limit) {
  int64_t p = kPieceElements / elements / 256 * 256;
  if (p < 256) p = 256;
  if (limit < p) p = limit;
  if (p >= V) return V;
  return up(ceil_div(V, ceil_div(V, p)), 256);
}

// Tiles of the scores: 256 x 256 on CTA pairs, or 128 x bn on single CTAs.
// Whichever takes the shortest rounds of all SMs, counting a tile by its columns
// (below 128 an MMA costs more than its share) and single CTAs, which read B
// once per 128 rows, at 1.1: 32768 columns of 8 rows run as 147 tiles of 224
// instead of 128 of 256; 333 x 10007 as one round of 147 tiles of 128 x 208
// instead of two of pairs.
struct ScoreTiles {
  bool pair, raw;
  int bn;
};
ScoreTiles score_tiles(int64_t rows, int64_t n, bool raw) {
  const int64_t sms = sm_count();
  if (raw) {  // each tile reads its A from shared memory again: wide ones, and 16 columns' time for starting
    ScoreTiles best{false, true, 32};
    double cost = 0.0;
    for (int bn = 32; bn <= lossmm::BN; bn += 16) {
      const double c = double(ceil_div(ceil_div(rows, lossmm::BM) * ceil_div(n, bn), sms)) * (bn + 16);
      if (bn == 32 || c < cost) cost = c, best.bn = bn;
    }
    return best;
  }
  ScoreTiles best{true, false, lossmm::BN};
  double cost = double(ceil_div(ceil_div(rows, 2 * lossmm::BM) * ceil_div(n, lossmm::BN), sms / 2)) * lossmm::BN;
  for (int bn = lossmm::BN; bn >= 16; bn -= 16) {
    const int64_t rounds = ceil_div(ceil_div(rows, lossmm::BM) * ceil_div(n, bn), sms);
    const double c = 1.1 * double(rounds) * (bn >= 128 ? bn : 0.5 * (bn + 128));
    if (c < cost) cost = c, best = ScoreTiles{false, false, bn};
  }
  return best;
}

bool rows16(const void *p, int64_t ld, int dtype) {
  return aligned16(p) && (ld * int64_t(dtype_bytes(dtype))) % 16 == 0;
}

// fp32 W is read as it is, and split inside the products, where few rows make
// reading it the larger part of the work: forward and backward of 30 rows of
// 60000 x 3000 took 2.18 ms with a split copy and 1.15 without (0.97 since dH is
// transposed).  Every 128 rows split W again, so more rows are better off with the copy:
// 200 rows of the same 1.30 ms with it, 1.34 without; 333 of 10007 x 768 173 and 256 us.
constexpr int64_t kRawRows = 128;
template <typename Ty>
bool raw_w(const Args &a) {
  return Ty::PARTS == 2 && a.rows <= kRawRows && rows16(a.W, a.ldw, a.dtype);
}

// A bump allocator over the workspace (or, with none, its size).
struct Space {
  char *base;
  size_t used = 0;
  template <typename T>
  T *take(int64_t n) {
    used = (used + 255) / 256 * 256;
    T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
    used += size_t(n) * sizeof(T);
    return p;
  }
};

// An operand's copy in the workspace: aligned rows (bf16), the tf32 pair, or for fp32
// rows that TMA can read in place the pair's lo alone, a third less to move (W of
// 10007 x 768: 15 us with both).  In place the hi operand is cut, not rounded, and lo has the
// sign of x: that is for W only, since the products drop lo lo, which would have the
// sign of the product if H were cut as well (-5.9 x 10^-8 of every score at D 768).
template <typename Ty>
struct Copy {
  typename Ty::T *p = nullptr;
  float *lo = nullptr;
  int64_t dp = 0;
  void take(Space &sp, int64_t rows, int64_t D, bool in_place = false) {
    dp = up(D, 16 / int64_t(sizeof(typename Ty::T)));
    if (!in_place) p = sp.take<typename Ty::T>(rows * dp);
    if (Ty::PARTS == 2) lo = sp.take<float>(rows * dp);
  }
  silcu_status fill(const void *src, int64_t ld, int64_t rows, int64_t D, const int32_t *targets, int64_t V,
                    cudaStream_t s, const Shared &shared = {}) const {
    using T = typename Ty::T;
    launch_after(copy_rows<T>, stream_grid(rows * dp * int64_t(sizeof(T)) / 16) + (shared.factor ? 1 : 0), 256, 0, s,
                 static_cast<const T *>(src), ld, rows, int(D), int(dp), targets, int(V), p, lo, shared);
    return check_launch("cross_entropy copy");
  }
  Operand operand(bool mn) const { return Operand{p, lo, dp, dp, mn}; }
  Operand operand(bool mn, const void *src, int64_t ld) const {  // of src, in place where it is not copied
    return p || !lo ? operand(mn) : Operand{src, lo, ld, dp, mn};
  }
};

template <typename Ty>
struct Forward {
  int64_t piece;
  ScoreTiles tiles;
  int nparts;
  bool copy_h, copy_w;  // operands that are not read in place
  Copy<Ty> h, w;
  float2 *part;
  float *target_score, *row_loss;
  unsigned *done;  // CTAs of loss_finish so far

  Forward(const Args &a, Space &sp, int64_t limit) {
    copy_h = Ty::PARTS == 2 || !rows16(a.H, a.ldh, a.dtype);
    copy_w = Ty::PARTS == 2 ? !raw_w<Ty>(a) : !rows16(a.W, a.ldw, a.dtype);
    piece = copy_w ? piece_of(a.V, up(a.D, 8), limit) : a.V;
    tiles = score_tiles(a.rows, piece, raw_w<Ty>(a));
    nparts = 0;
    for (int64_t v0 = 0; v0 < a.V; v0 += piece) nparts += parts(a, v0);
    part = sp.take<float2>(int64_t(nparts) * a.rows);
    target_score = sp.take<float>(a.rows);
    row_loss = a.reduction == SILCU_REDUCE_NONE ? a.loss : sp.take<float>(a.rows);
    done = sp.take<unsigned>(1);
    if (copy_h) h.take(sp, a.rows, a.D);
    if (copy_w) w.take(sp, piece, a.D, Ty::PARTS == 2 && rows16(a.W, a.ldw, a.dtype));
  }
  int64_t columns(const Args &a, int64_t v0) const { return a.V - v0 < piece ? a.V - v0 : piece; }
  int parts(const Args &a, int64_t v0) const { return 2 * int(ceil_div(columns(a, v0), tiles.bn)); }
};

// One of the two products of ds, with M x N results from sums of K: its K is
// cut into `split` parts whose sums are fp32 planes, and `direct` results
// need no planes at all.
struct Gradient {
  int64_t M, N, K;
  int split = 1;
  bool wanted, direct;
  bool transposed = false;    // computed as its transpose (kOutT): the N x M tiles hold all of M
  float *planes = nullptr;
  int tile = 2 * lossmm::BM;  // rows of a tile (CTA pairs: 256; single CTAs: 128)
  int bn = lossmm::BN;        // and its columns
  int64_t tiles() const { return transposed ? ceil_div(N, tile) : ceil_div(M, tile) * ceil_div(N, bn); }
  int64_t units() const { return tile == lossmm::BM ? sm_count() : sm_count() / 2; }
};

// Time of both products in one launch, in k of one tile: the slowest SM pair's
// items (work_at; `first` has the longer ones), each with its epilogue, and
// the planes' traffic.  One k of a tile takes 131072 flops of a pair's share of
// the measured 1.4 PFLOP/s (7 ns; half that for a tile of 128 on one SM; six
// times that in 3xTF32).
double out_time(const Gradient &first, const Gradient &second, bool tf32) {
  const int64_t units = first.units();
  const int64_t n0 = first.wanted ? first.tiles() * first.split : 0;
  const int64_t n1 = second.wanted ? second.tiles() * second.split : 0;
  if (n0 + n1 == 0) return 0.0;
  const int64_t u = n0 + n1 < units ? n0 + n1 : units, tail = n0 % u, low = u - tail;
  const double epilogue = tf32 ? 128.0 : 512.0;
  const double ns = (tf32 ? 42.0 : 7.0) * (first.tile == lossmm::BM ? 0.5 : first.bn / 256.0);
  const double c0 = double(first.K) / first.split, c1 = double(second.K) / second.split;
  const int64_t extra = n1 && tail ? int64_t(c0 / c1 + 0.5) : 0;
  auto rounds = [&](int64_t begin, int64_t step) { return begin < n1 ? ceil_div(n1 - begin, step) : 0; };
  const int64_t after = tail ? extra * low : 0;
  const int64_t high = rounds(after, u);  // unit 0: after the short units' extra rounds
  double time = double(ceil_div(n0, u)) * (c0 + epilogue) + double(high) * (c1 + epilogue);
  if (tail) {
    const int64_t own = rounds(0, low) < extra ? rounds(0, low) : extra;
    const double t = double(n0 / u) * (c0 + epilogue) + double(own + rounds(after + tail, u)) * (c1 + epilogue);
    if (t > time) time = t;
  }
  double bytes = 0.0;
  for (const Gradient *g : {&first, &second})
    if (g->wanted) bytes += 8.0 * (g->split - 1) * double(g->M) * double(g->N);
  return time * ns + bytes / 6500.0;
}

// Columns of the products' tiles, whose N is D: the width that wastes the fewest
// columns of D (16 more stand for a tile's fixed share).  Each CTA of a pair loads half
// of them in boxes of 32 fp32 or 64 bf16 columns.
int columns_of_tile(int64_t D, bool tf32) {
  int best = lossmm::BN;
  for (int bn = lossmm::BN; bn >= 64; bn -= tf32 ? 64 : 128)
    if (ceil_div(D, bn) * (bn + 16) < ceil_div(D, best) * (best + 16)) best = bn;
  return best;
}

// Cuts the products' K so that the launch ends evenly: long sums of few tiles
// (few rows, or a short vocabulary) and the last round of many.  At least 512 k
// a part, and 32 parts at most but for the few tiles of a transposed product.
void choose_splits(Gradient &dh, Gradient &dw, bool tf32) {
  static const int counts[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64};
  double best = -1.0;
  int bh = 1, bw = 1;
  for (const int h : counts) {
    if (h > 1 && (!dh.wanted || dh.K < 512 * int64_t(h) || (h > 32 && !dh.transposed))) break;
    for (const int w : counts) {
      if (w > 1 && (!dw.wanted || dw.K < 512 * int64_t(w) || w > 32)) break;
      dh.split = h;
      dw.split = w;
      const bool dw_first = dw.K / w > dh.K / h;
      const double t = out_time(dw_first ? dw : dh, dw_first ? dh : dw, tf32);
      if (best < 0.0 || t < best) best = t, bh = h, bw = w;
    }
  }
  dh.split = bh;
  dw.split = bw;
}

template <typename Ty>
struct Backward {
  int64_t piece, lds;  // lds: row stride of ds
  ScoreTiles score;
  bool copy_w;
  float *factor;       // that all rows share (mean, sum)
  Copy<Ty> h, w;       // H with left-out rows zero; a piece of W
  Copy<Ty> ds;
  Gradient dh, dw;

  Backward(const Args &a, Space &sp, int64_t limit) {
    copy_w = Ty::PARTS == 2 ? !raw_w<Ty>(a) : !rows16(a.W, a.ldw, a.dtype);
    const int64_t of_w = copy_w ? up(a.D, 8) : 0;
    piece = piece_of(a.V, a.rows > of_w ? a.rows : of_w, limit);
    score = score_tiles(a.rows, piece, raw_w<Ty>(a));
    factor = a.reduction == SILCU_REDUCE_NONE ? nullptr : sp.take<float>(1);
    h.take(sp, a.rows, a.D);
    if (copy_w) w.take(sp, piece, a.D, Ty::PARTS == 2 && rows16(a.W, a.ldw, a.dtype));
    ds.take(sp, a.rows, up(piece, 64));
    lds = ds.dp;
    dh.M = a.rows, dh.N = a.D, dh.K = piece, dh.wanted = a.dH;
    dw.M = piece, dw.N = a.D, dw.K = a.rows, dw.wanted = a.dW;
    dh.bn = dw.bn = columns_of_tile(a.D, Ty::PARTS == 2);
    dh.transposed = a.rows <= lossmm::BM;
    if (score.raw) dh.tile = lossmm::BM;  // and transposed, having few rows
    if (dh.transposed) {  // a launch of its own
      Gradient none = {};
      none.K = 1, none.wanted = false;
      choose_splits(dh, none, Ty::PARTS == 2);
      choose_splits(none, dw, Ty::PARTS == 2);
    } else {
      choose_splits(dh, dw, Ty::PARTS == 2);
    }
    dh.direct = dh.split == 1 && piece == a.V;  // else pieces add up in the planes
    dw.direct = dw.split == 1;
    for (Gradient *g : {&dh, &dw})
      if (g->wanted && !g->direct) g->planes = sp.take<float>(int64_t(g->split) * g->M * up(a.D, 8));
  }
};

// ---------------------------------------------------------------------- run
silcu_status map_error() { return fail(SILCU_CUDA_ERROR, "cross_entropy: cuTensorMapEncodeTiled failed"); }

// The ring and the epilogue warps' columns of a RAW launch with p.bn and p.rows_a.
void set_raw(lossmm::Params &p) {
  const int stages = 192 * 1024 / (2 * 128 * (p.rows_a + p.bn));
  p.stages = stages < 8 ? stages : 8;
  p.half = int(up((p.bn + 1) / 2, 32));
}

// Few rows need no whole tile of A: 8 rows of 32768 x 4096 bf16 take 51 us with
// boxes of 8 rows, 60 with boxes of 128 that are zeros for the most part.
template <typename Ty>
bool set_scores(lossmm::Params &p, const ScoreTiles &t, int64_t rows, int64_t n, int64_t D, const Operand &h,
                const Operand &w) {
  p.bn = t.bn;
  p.rows_a = !t.pair && rows < lossmm::BM ? int(up(rows, 8)) : lossmm::BM;
  if (t.raw) set_raw(p);
  return lossmm::set_problem<Ty>(p.p[0], t.pair, t.bn, p.rows_a, rows, n, D, h, w);
}

template <typename Ty, int EPI>
silcu_status scores(lossmm::Params &p, const ScoreTiles &t, cudaStream_t s) {
  if constexpr (Ty::PARTS == 2)
    if (t.raw) return lossmm::launch<Ty, EPI, false, true>(p, 1, s);
  return t.pair ? lossmm::launch<Ty, EPI, true>(p, 1, s) : lossmm::launch<Ty, EPI, false>(p, 1, s);
}

template <typename T>
const T *row_of(const void *base, int64_t row, int64_t ld) {
  return static_cast<const T *>(base) + row * ld;
}

template <typename Ty>
silcu_status forward(const Args &a, const Forward<Ty> &f, cudaStream_t s) {
  using T = typename Ty::T;
  silcu_status st;
  Operand h{a.H, nullptr, a.ldh, 0, false};
  if (f.copy_h) {
    if ((st = f.h.fill(a.H, a.ldh, a.rows, a.D, nullptr, 0, s)) != SILCU_OK) return st;
    h = f.h.operand(false);
  }
  int part0 = 0;
  for (int64_t v0 = 0; v0 < a.V; v0 += f.piece) {
    const int64_t n = f.columns(a, v0);
    const T *src = row_of<T>(a.W, v0, a.ldw);
    Operand w{src, nullptr, a.ldw, 0, false};
    if (f.copy_w) {
      if ((st = f.w.fill(src, a.ldw, n, a.D, nullptr, 0, s)) != SILCU_OK) return st;
      w = f.w.operand(false, src, a.ldw);
    }
    lossmm::Params p;
    memset(&p, 0, sizeof(p));
    if (!set_scores<Ty>(p, f.tiles, a.rows, n, a.D, h, w)) return map_error();
    p.part0 = part0;
    p.err = device_error_ptr();
    p.loss.targets = a.targets;
    p.loss.V = int32_t(a.V);
    p.loss.v0 = int32_t(v0);
    p.loss.part = f.part;
    p.loss.target_score = f.target_score;
    p.loss.done = f.done;
    if ((st = scores<Ty, lossmm::kStats>(p, f.tiles, s)) != SILCU_OK) return st;
    part0 += f.parts(a, v0);
  }
  launch_after(loss_finish, uint32_t(ceil_div(a.rows, kFinishRows)), 1024, 0, s, f.part, f.nparts, a.rows, a.targets,
               int(a.V), f.target_score, a.lse, f.row_loss, int(a.reduction == SILCU_REDUCE_MEAN), f.done,
               a.reduction == SILCU_REDUCE_NONE ? nullptr : a.loss);
  return check_launch("cross_entropy finish");
}

// Where a product of ds goes: the result itself, or planes that earlier
// pieces may have begun.
void set_output(lossmm::Problem &q, const Gradient &g, bool add, void *out, int64_t ldo, int vec, int64_t D,
                int64_t nk) {
  q.ksplit = int(g.split < nk ? g.split : nk);  // a short last piece adds to the first planes only
  if (g.direct) {
    q.mode = lossmm::kDirect;
    q.out = out;
    q.ldo = ldo;
    q.vec = vec;
  } else {
    q.mode = add ? lossmm::kPlaneAdd : lossmm::kPlane;
    q.out = g.planes;
    q.ldo = up(D, 8);
    q.plane = g.M * q.ldo;
  }
}

template <typename Ty>
silcu_status finish_planes(const Gradient &g, int64_t rows, int64_t D, const float *alpha, const int32_t *targets, int64_t V,
                           void *out, int64_t ldo, int vec, cudaStream_t s) {
  using T = typename Ty::T;
  const int64_t ldp = up(D, 8);
  const int64_t vectors = rows * ceil_div(D * int64_t(sizeof(T)), 16);
  const bool few = g.split >= 8 && vectors * 8 <= int64_t(sm_count()) * 2048;  // eight lanes each fill the SMs at most once
  launch_after(few ? planes_finish<T, 8> : planes_finish<T, 1>, stream_grid(vectors * (few ? 8 : 1)), 256, 0, s, g.planes,
               g.split, g.M * ldp, rows, int(D), int(ldp), alpha, targets, int(V), static_cast<T *>(out), ldo, vec);
  return check_launch("cross_entropy planes");
}

template <typename Ty>
silcu_status backward(const Args &a, const Backward<Ty> &b, cudaStream_t s) {
  using T = typename Ty::T;
  constexpr int BK = lossmm::Cfg<Ty, lossmm::kOut, true>::BK;
  silcu_status st;
  if ((st = b.h.fill(a.H, a.ldh, a.rows, a.D, a.targets, a.V, s, Shared{a.dloss, a.reduction, b.factor})) != SILCU_OK)
    return st;
  // A factor that all rows share leaves ds alone where ds is rounded, and multiplies the results;
  // dH's rows that are left out stay 0 whatever it is.
  const float *alpha = Ty::PARTS == 1 ? b.factor : nullptr;
  const int dh_vec = rows16(a.dH, a.lddh, a.dtype), dw_vec = rows16(a.dW, a.lddw, a.dtype);
  for (int64_t v0 = 0; v0 < a.V; v0 += b.piece) {
    const int64_t n = a.V - v0 < b.piece ? a.V - v0 : b.piece;
    const T *src = row_of<T>(a.W, v0, a.ldw);
    Operand w{src, nullptr, a.ldw, 0, false};
    if (b.copy_w) {
      if ((st = b.w.fill(src, a.ldw, n, a.D, nullptr, 0, s)) != SILCU_OK) return st;
      w = b.w.operand(false, src, a.ldw);
    }
    lossmm::Params p;
    memset(&p, 0, sizeof(p));
    p.err = device_error_ptr();
    if (!set_scores<Ty>(p, b.score, a.rows, n, a.D, b.h.operand(false), w)) return map_error();
    p.ds[0] = b.ds.p;
    p.ds[1] = b.ds.lo;
    p.lds = b.lds;
    p.loss.targets = a.targets;
    p.loss.V = int32_t(a.V);
    p.loss.v0 = int32_t(v0);
    p.loss.lse = a.lse;
    p.loss.scale = a.reduction == SILCU_REDUCE_NONE ? a.dloss : alpha ? nullptr : b.factor;
    p.loss.per_row = a.reduction == SILCU_REDUCE_NONE;
    if ((st = scores<Ty, lossmm::kScoreGrad>(p, b.score, s)) != SILCU_OK) return st;

    const bool pairs = !b.score.raw;
    w.mn = true;
    auto clear = [&](int bn) {
      memset(&p, 0, sizeof(p));
      p.err = device_error_ptr();
      p.bn = bn;
      p.rows_a = lossmm::BM;
      p.alpha = alpha;
      p.loss.targets = a.targets;
      p.loss.V = int32_t(a.V);
    };
    if (b.dh.wanted && b.dh.transposed) {
      clear(int(up(a.rows, 32)));
      if (!pairs) set_raw(p);
      if (!lossmm::set_problem<Ty>(p.p[0], pairs, p.bn, lossmm::BM, a.D, a.rows, n, w, b.ds.operand(false))) return map_error();
      set_output(p.p[0], b.dh, v0 != 0, a.dH, a.lddh, dh_vec, a.D, ceil_div(n, BK));
      if constexpr (Ty::PARTS == 2)
        st = pairs ? lossmm::launch<Ty, lossmm::kOutT, true>(p, 1, s) : lossmm::launch<Ty, lossmm::kOutT, false, true>(p, 1, s);
      else
        st = lossmm::launch<Ty, lossmm::kOutT, true>(p, 1, s);
      if (st != SILCU_OK) return st;
    }
    // Both products of ds in one launch, the one with the longer items first.
    clear(b.dw.bn);
    p.half = int(up(p.bn / 2, 32));
    int count = 0;
    const bool dw_first = b.dw.K / b.dw.split > b.dh.K / b.dh.split;
    for (const bool is_dw : {dw_first, !dw_first}) {
      if (is_dw ? !b.dw.wanted : !b.dh.wanted || b.dh.transposed) continue;
      lossmm::Problem &q = p.p[count++];
      if (is_dw) {
        if (!lossmm::set_problem<Ty>(q, true, p.bn, lossmm::BM, n, a.D, a.rows, b.ds.operand(true), b.h.operand(true)))
          return map_error();
        set_output(q, b.dw, false, static_cast<T *>(a.dW) + v0 * a.lddw, a.lddw, dw_vec, a.D,
                   ceil_div(a.rows, BK));
      } else {
        if (!lossmm::set_problem<Ty>(q, true, p.bn, lossmm::BM, a.rows, a.D, n, b.ds.operand(false), w)) return map_error();
        set_output(q, b.dh, v0 != 0, a.dH, a.lddh, dh_vec, a.D, ceil_div(n, BK));
        q.of_rows = 1;
      }
    }
    if (count && (st = lossmm::launch<Ty, lossmm::kOut, true>(p, count, s)) != SILCU_OK) return st;
    if (b.dw.wanted && !b.dw.direct) {
      st = finish_planes<Ty>(b.dw, n, a.D, alpha, nullptr, a.V, static_cast<T *>(a.dW) + v0 * a.lddw, a.lddw, dw_vec, s);
      if (st != SILCU_OK) return st;
    }
  }
  if (b.dh.wanted && !b.dh.direct) return finish_planes<Ty>(b.dh, a.rows, a.D, alpha, alpha ? a.targets : nullptr, a.V, a.dH, a.lddh, dh_vec, s);
  return SILCU_OK;
}

// ------------------------------------------------------------------- checks
silcu_status check_shape(const char *what, const Args *ap) {
  if (!ap) return fail(SILCU_INVALID_ARGUMENT, "%s: null args", what);
  const Args &a = *ap;
  if (!dtype_known(a.dtype)) return fail(SILCU_INVALID_ARGUMENT, "%s: unknown dtype %d", what, a.dtype);
  if (a.reduction < SILCU_REDUCE_MEAN || a.reduction > SILCU_REDUCE_NONE)
    return fail(SILCU_INVALID_ARGUMENT, "%s: unknown reduction %d", what, a.reduction);
  if (a.rows < 0 || a.V <= 0 || a.D <= 0) return fail(SILCU_INVALID_ARGUMENT, "%s: bad extent", what);
  if (a.rows > (1 << 20) || a.V > (1 << 24) || a.D > (1 << 17))
    return fail(SILCU_UNSUPPORTED, "%s: extent too large (rows 2^20, V 2^24, D 2^17 at most)", what);
  if (a.ldh < a.D || a.ldw < a.D) return fail(SILCU_INVALID_ARGUMENT, "%s: ldh or ldw < D", what);
  if (a.ldh > (int64_t(1) << 32) || a.ldw > (int64_t(1) << 32))
    return fail(SILCU_UNSUPPORTED, "%s: row stride too large", what);
  return SILCU_OK;
}

silcu_status check_gradients(const char *what, const Args &a) {
  for (const auto &g : {std::make_pair(a.dH, a.lddh), std::make_pair(a.dW, a.lddw)}) {
    if (g.first && g.second < a.D) return fail(SILCU_INVALID_ARGUMENT, "%s: lddh or lddw < D", what);
    if (g.first && g.second > (int64_t(1) << 32)) return fail(SILCU_UNSUPPORTED, "%s: row stride too large", what);
  }
  return SILCU_OK;
}

silcu_status check_pointers(const char *what, const Args &a) {
  const uintptr_t mask = dtype_bytes(a.dtype) - 1;
  if (!a.H || !a.W || !a.targets || !a.lse) return fail(SILCU_INVALID_ARGUMENT, "%s: null pointer", what);
  for (const void *p : {a.H, a.W, static_cast<const void *>(a.dH), static_cast<const void *>(a.dW)})
    if (reinterpret_cast<uintptr_t>(p) & mask) return fail(SILCU_INVALID_ARGUMENT, "%s: misaligned pointer", what);
  for (const void *p : {static_cast<const void *>(a.targets), static_cast<const void *>(a.lse),
                        static_cast<const void *>(a.loss), static_cast<const void *>(a.dloss)})
    if (reinterpret_cast<uintptr_t>(p) & 3) return fail(SILCU_INVALID_ARGUMENT, "%s: misaligned pointer", what);
  return SILCU_OK;
}

constexpr size_t kAlign = 256;  // the caller's workspace need not be aligned
char *aligned(void *p) { return reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(p) + kAlign - 1) & ~uintptr_t(kAlign - 1)); }

// The plan of a call, Forward or Backward, laid out in its workspace, once that is known to hold it.
template <template <typename> class Plan, typename Ty, typename F>
silcu_status with_plan(const char *what, const Args &a, void *ws, size_t bytes, F &&run) {
  Space sp{aligned(ws)};
  const Plan<Ty> plan(a, sp, piece_limit());
  const size_t need = sp.used + kAlign;
  if (!ws || bytes < need) return fail(SILCU_WORKSPACE_TOO_SMALL, "%s: workspace %zu < %zu", what, bytes, need);
  if (!device_error_ptr()) return fail(SILCU_CUDA_ERROR, "%s: no device error word", what);
  return run(plan);
}

}  // namespace
}  // namespace silcu

extern "C" {

size_t silcu_linear_cross_entropy_workspace_bytes(const silcu_cross_entropy_args *ap, int backward) {
  using namespace silcu;
  if (check_shape("linear_cross_entropy_workspace_bytes", ap) != SILCU_OK || ap->rows == 0) return 0;
  Space f{nullptr}, b{nullptr};
  const int64_t limit = piece_limit();
  if (ap->dtype == SILCU_BF16) {
    Forward<Bf16> plan(*ap, f, limit);
    if (backward) Backward<Bf16> plan_b(*ap, b, limit);
  } else {
    Forward<Tf32> plan(*ap, f, limit);
    if (backward) Backward<Tf32> plan_b(*ap, b, limit);
  }
  return (f.used > b.used ? f.used : b.used) + kAlign;
}

silcu_status silcu_linear_cross_entropy(const silcu_cross_entropy_args *ap, void *workspace, size_t workspace_bytes,
                                        silcu_stream stream) {
  using namespace silcu;
  silcu_status st = check_shape("linear_cross_entropy", ap);
  if (st != SILCU_OK) return st;
  const Args &a = *ap;
  cudaStream_t s = as_stream(stream);
  if (!a.loss && (a.rows || a.reduction != SILCU_REDUCE_NONE))
    return fail(SILCU_INVALID_ARGUMENT, "linear_cross_entropy: null pointer");
  if (a.rows == 0) {
    if (a.reduction == SILCU_REDUCE_NONE) return SILCU_OK;
    const cudaError_t r = cudaMemsetAsync(a.loss, 0, sizeof(float), s);
    return r == cudaSuccess ? SILCU_OK : fail(SILCU_CUDA_ERROR, "linear_cross_entropy: %s", cudaGetErrorString(r));
  }
  if ((st = check_pointers("linear_cross_entropy", a)) != SILCU_OK) return st;
  const int64_t e = int64_t(dtype_bytes(a.dtype));
  const Span outs[] = {flat(a.loss, a.reduction == SILCU_REDUCE_NONE ? 4 * a.rows : 4), flat(a.lse, 4 * a.rows)};
  const Span ins[] = {{a.H, a.rows, a.D * e, a.ldh * e}, {a.W, a.V, a.D * e, a.ldw * e}, flat(a.targets, 4 * a.rows)};
  if (outputs_overlap(outs, 2, ins, 3))
    return fail(SILCU_INVALID_ARGUMENT, "linear_cross_entropy: a result overlaps an operand");
  auto run = [&](const auto &plan) { return forward(a, plan, s); };
  return a.dtype == SILCU_BF16 ? with_plan<Forward, Bf16>("linear_cross_entropy", a, workspace, workspace_bytes, run)
                               : with_plan<Forward, Tf32>("linear_cross_entropy", a, workspace, workspace_bytes, run);
}

silcu_status silcu_linear_cross_entropy_backward(const silcu_cross_entropy_args *ap, void *workspace,
                                                 size_t workspace_bytes, silcu_stream stream) {
  using namespace silcu;
  const char *what = "linear_cross_entropy_backward";
  silcu_status st = check_shape(what, ap);
  if (st != SILCU_OK) return st;
  const Args &a = *ap;
  cudaStream_t s = as_stream(stream);
  if (!a.dH && !a.dW) return SILCU_OK;
  if ((st = check_gradients(what, a)) != SILCU_OK) return st;
  if (a.rows == 0) {  // no terms: dW is zero
    if (a.dW) {
      const size_t e = dtype_bytes(a.dtype);
      const cudaError_t r = cudaMemset2DAsync(a.dW, a.lddw * e, 0, a.D * e, a.V, s);
      if (r != cudaSuccess) return fail(SILCU_CUDA_ERROR, "%s: %s", what, cudaGetErrorString(r));
    }
    return SILCU_OK;
  }
  if ((st = check_pointers(what, a)) != SILCU_OK) return st;
  const int64_t e = int64_t(dtype_bytes(a.dtype));
  const Span outs[] = {{a.dH, a.rows, a.D * e, a.lddh * e}, {a.dW, a.V, a.D * e, a.lddw * e}};
  const Span ins[] = {{a.H, a.rows, a.D * e, a.ldh * e},
                      {a.W, a.V, a.D * e, a.ldw * e},
                      flat(a.targets, 4 * a.rows),
                      flat(a.lse, 4 * a.rows),
                      flat(a.dloss, a.reduction == SILCU_REDUCE_NONE ? 4 * a.rows : 4)};
  if (outputs_overlap(outs, 2, ins, 5)) return fail(SILCU_INVALID_ARGUMENT, "%s: a gradient overlaps an operand", what);
  auto run = [&](const auto &plan) { return backward(a, plan, s); };
  return a.dtype == SILCU_BF16 ? with_plan<Backward, Bf16>(what, a, workspace, workspace_bytes, run)
                               : with_plan<Backward, Tf32>(what, a, workspace, workspace_bytes, run);
}

}  // extern "C"
