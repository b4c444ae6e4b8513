// Softmax cross entropy of a vocabulary projection, forward and backward,
// without the logits in memory.
//
//   s = H . W^T,  lse_t = log sum_v exp(s_tv),  loss_t = lse_t - s_t,y(t)
//   ds_tv = g_t (exp(s_tv - lse_t) - [v = y(t)]),  dH = ds . W,  dW = ds^T . H
//
// Forward: one tensor-core product whose epilogue keeps, for every row and
// every 128 columns, the maximum and the sum of exponentials (8 bytes in place
// of 128 scores) and the target's score; loss_finish joins them.
// Backward: piece by piece of the vocabulary, the same product again with the
// score gradients as its epilogue (ds of one piece is all that is kept), then
// dH += ds . W_piece and dW_piece = ds^T . H.  Recomputing the scores costs
// 2 T V D operations on top of the 6 T V D of the forward and the gradients;
// keeping them would take T V values.
// Bound by the tensor cores except for few rows, where reading W is all.
//
// fp32 operands go through the 3xTF32 GEMM (tc_gemm.cu), bf16 ones through
// bf16_gemm.cuh; there ds is rounded to bf16, the operand type of its two
// products, once per element (2^-9 relative, the rounding that the gradients
// themselves take when they are stored).
//
// Rows whose target lies outside [0, V) are left out: the backward pass works
// on a copy of H with those rows zero and gives them ds = 0 by selection, so
// nothing that H holds there reaches dW.
#include <stdlib.h>
#include <string.h>

#include <utility>

#include "bf16_gemm.cuh"
#include "gemm_internal.cuh"

namespace silcu {
namespace {

using Args = silcu_cross_entropy_args;

// ------------------------------------------------------------ small kernels
// Joins a row's parts: lse = M + log sum l_i exp(m_i - M).  A CTA takes 32
// rows, 8 warps the parts in 8 interleaved slices.
__global__ void __launch_bounds__(256) loss_finish(const float2 *__restrict__ part, int nparts, int64_t rows,
                                                   const int32_t *__restrict__ targets, int V,
                                                   const float *__restrict__ target_score, float *__restrict__ lse,
                                                   float *__restrict__ loss) {
  __shared__ float2 sm[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t row = int64_t(blockIdx.x) * 32 + lane;
  float m = -INFINITY, l = 0.f;
  auto join = [&](float2 x) {
    const float mx = fmaxf(m, x.x);
    const float ref = mx == -INFINITY ? 0.f : mx;
    l = l * ex2((m - ref) * kLog2e) + x.y * ex2((x.x - ref) * kLog2e);
    m = mx;
  };
  if (row < rows) {
#pragma unroll 4
    for (int i = slice; i < nparts; i += 8) join(__ldcs(part + int64_t(i) * rows + row));
  }
  sm[slice][lane] = make_float2(m, l);
  __syncthreads();
  if (slice == 0 && row < rows) {
#pragma unroll
    for (int i = 1; i < 8; i++) join(sm[i][lane]);
    const float v = m + logf(l);
    lse[row] = v;
    const int y = targets[row];
    loss[row] = y >= 0 && y < V ? v - target_score[row] : 0.f;
  }
}

__device__ __forceinline__ double cta_sum(double v, double *sm) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < int(blockDim.x >> 5); i++) s += sm[i];
  __syncthreads();
  return s;
}

// Number of rows that count, in every thread of the (one) CTA.
__device__ __forceinline__ double count_rows(const int32_t *targets, int64_t rows, int V, double *sm) {
  int n = 0;
  for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) {
    const int y = targets[i];
    n += y >= 0 && y < V;
  }
  return cta_sum(double(n), sm);
}

// The scalar loss: the sum of the rows' losses, or their mean over the rows
// that count (0 when none does).
__global__ void __launch_bounds__(1024) loss_reduce(const float *__restrict__ row_loss,
                                                    const int32_t *__restrict__ targets, int64_t rows, int V, int mean,
                                                    float *__restrict__ loss) {
  __shared__ double sm[32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) s += double(row_loss[i]);
  s = cta_sum(s, sm);
  if (mean) {
    const double n = count_rows(targets, rows, V, sm);
    s = n > 0.0 ? s / n : 0.0;
  }
  if (threadIdx.x == 0) *loss = float(s);
}

// The gradient of every row's loss.
__global__ void __launch_bounds__(1024) row_scales(const float *__restrict__ dloss,
                                                   const int32_t *__restrict__ targets, int64_t rows, int V,
                                                   int reduction, float *__restrict__ scale) {
  __shared__ double sm[32];
  float g = 1.0f;
  if (reduction == SILCU_REDUCE_MEAN) {
    const double n = count_rows(targets, rows, V, sm);
    g = float((dloss ? double(*dloss) : 1.0) / (n > 0.0 ? n : 1.0));
  } else if (reduction == SILCU_REDUCE_SUM && dloss) {
    g = *dloss;
  }
  for (int64_t i = threadIdx.x; i < rows; i += 1024)
    scale[i] = reduction == SILCU_REDUCE_NONE && dloss ? dloss[i] : g;
}

// dst [rows, dp] = src [rows, D] (row stride ld), columns D.. zero; with
// targets, rows that are left out are zero as well.
template <typename T>
__global__ void __launch_bounds__(256) copy_rows(const T *__restrict__ src, int64_t ld, int64_t rows, int D, int dp,
                                                 const int32_t *__restrict__ targets, int V, T *__restrict__ dst) {
  constexpr int W = 16 / sizeof(T);
  const int per_row = dp / W;
  const bool vec = ld % W == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  const int64_t n = rows * per_row;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t r = i / per_row;
    const int c = int(i - r * per_row) * W;
    Raw<T, W> v = raw_zero<T, W>();
    bool keep = true;
    if (targets) {
      const int y = __ldg(targets + r);
      keep = y >= 0 && y < V;
    }
    if (keep) {
      if (vec && c + W <= D) {
        v = raw_load<T, W>(src + r * ld + c);
      } else {
        T *e = reinterpret_cast<T *>(&v);
#pragma unroll
        for (int k = 0; k < W; k++)
          if (c + k < D) e[k] = src[r * ld + c + k];
      }
    }
    *reinterpret_cast<decltype(v.r) *>(dst + r * dp + c) = v.r;
  }
}

// out [rows, D] bf16 = the sum of the fp32 planes [rows, ldp], in plane order.
__global__ void __launch_bounds__(256) planes_finish(const float *__restrict__ planes, int nplanes, int64_t plane,
                                                     int64_t rows, int D, int ldp, __nv_bfloat16 *__restrict__ out,
                                                     int64_t ldo, int vec) {
  const int per_row = (D + 7) / 8;
  const int64_t n = rows * per_row;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t r = i / per_row;
    const int c = int(i - r * per_row) * 8;
    float f[8] = {};
    for (int p = 0; p < nplanes; p++) {  // ldp is a multiple of 8: the last vectors stay inside the row
      float v[8];
      load_f32<8>(planes + p * plane + r * ldp + c, v);
#pragma unroll
      for (int k = 0; k < 8; k++) f[k] += v[k];
    }
    __nv_bfloat16 *dst = out + r * ldo + c;
    if (vec && c + 8 <= D) {
      Raw<__nv_bfloat16, 8> o;
      pack(f, o);
      *reinterpret_cast<uint4 *>(dst) = o.r;
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (c + k < D) dst[k] = __float2bfloat16_rn(f[k]);
    }
  }
}

uint32_t stream_grid(int64_t items) {
  const int64_t g = (items + 255) / 256, cap = int64_t(sm_count()) * 16;
  return uint32_t(g < 1 ? 1 : g < cap ? g : cap);
}

// --------------------------------------------------------------------- plan
constexpr int64_t kPieceBytes = int64_t(256) << 20;  // of ds, and of a piece's copied weights

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Vocabulary columns per piece: a multiple of 256 whose `bytes` per column
// stay within kPieceBytes, and pieces of about equal size.
int64_t piece_of(int64_t V, int64_t bytes) {
  int64_t p = kPieceBytes / bytes / 256 * 256;
  if (p < 256) p = 256;
  if (p > (1 << 20)) p = 1 << 20;  // the packing passes' grids
  if (const char *e = getenv("SILCU_LOSS_PIECE")) {  // columns per piece at most (tests, tuning)
    const int64_t want = up(atoll(e) > 0 ? atoll(e) : 256, 256);
    if (want < p) p = want;
  }
  if (p >= V) return V;
  const int64_t n = (V + p - 1) / p;
  return up((V + n - 1) / n, 256);
}

bool rows16(const void *p, int64_t ld, int dtype) {
  return aligned16(p) && (ld * int64_t(dtype_bytes(dtype))) % 16 == 0;
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

struct Forward {
  int64_t piece, dp;
  bool copy_h, copy_w;  // operands whose rows TMA cannot read in place (bf16)
  float2 *part;
  float *target_score, *row_loss;
  __nv_bfloat16 *h, *w;
  float *h_hi, *h_lo;
  void *gemm;
  size_t gemm_bytes;
};

silcu_gemm_args f32_args(int64_t M, int64_t N, int64_t K) {
  silcu_gemm_args g;
  memset(&g, 0, sizeof(g));
  g.M = M;
  g.N = N;
  g.K = K;
  g.batch = 1;
  g.alpha = 1.0f;
  g.algo = SILCU_GEMM_TC3XTF32;
  return g;
}

// Scores of a vocabulary piece (fp32): A = the split H, B = W's rows, plain.
silcu_gemm_args score_args(const Args &a, const float *hi, const float *lo, int64_t dp, int64_t v0, int64_t n) {
  silcu_gemm_args g = f32_args(a.rows, n, a.D);
  g.A_hi = hi;
  g.A_lo = lo;
  g.lda = dp;
  g.B = static_cast<const float *>(a.W) + v0 * a.ldw;
  g.ldb = a.ldw;
  g.trans_b = 1;
  g.ldc = n;
  return g;
}

// Not null, for workspace sizes: only whether an operand is given matters.
float *given() { return reinterpret_cast<float *>(uintptr_t(256)); }

template <typename F>
size_t most_over_pieces(int64_t V, int64_t piece, F &&f) {
  size_t most = f(piece);
  if (V % piece) {
    const size_t last = f(V % piece);
    if (last > most) most = last;
  }
  return most;
}

Forward plan_forward(const Args &a, Space &sp) {
  Forward f = {};
  f.part = sp.take<float2>((a.V + 127) / 128 * a.rows);
  f.target_score = sp.take<float>(a.rows);
  f.row_loss = a.reduction == SILCU_REDUCE_NONE ? a.loss : sp.take<float>(a.rows);
  if (a.dtype == SILCU_BF16) {
    f.dp = up(a.D, 8);
    f.copy_h = !rows16(a.H, a.ldh, a.dtype);
    f.copy_w = !rows16(a.W, a.ldw, a.dtype);
    f.piece = f.copy_w ? piece_of(a.V, 2 * f.dp) : a.V;
    if (f.copy_h) f.h = sp.take<__nv_bfloat16>(a.rows * f.dp);
    if (f.copy_w) f.w = sp.take<__nv_bfloat16>(f.piece * f.dp);
  } else {
    f.dp = up(a.D, 4);
    f.piece = piece_of(a.V, 8 * f.dp);
    f.h_hi = sp.take<float>(a.rows * f.dp);
    f.h_lo = sp.take<float>(a.rows * f.dp);
    f.gemm_bytes = most_over_pieces(a.V, f.piece, [&](int64_t n) {
      return tc_loss_workspace_bytes(score_args(a, given(), given(), f.dp, 0, n));
    });
    f.gemm = sp.take<char>(int64_t(f.gemm_bytes));
  }
  return f;
}

// A bf16 product's split of K: parts for idle SMs when the tiles are few, at
// least 8 stages of 64 k in each.
int split_k(int64_t M, int64_t N, int64_t K) {
  const bool pair = M > bf16::BM;
  const int64_t units = pair ? sm_count() / 2 : sm_count();
  const int64_t tiles = (M + (pair ? 255 : 127)) / (pair ? 256 : 128) * ((N + 255) / 256);
  int64_t ks = units / tiles;
  const int64_t most = (K + 64 * 8 - 1) / (64 * 8);
  if (ks > most) ks = most;
  return int(ks < 1 ? 1 : ks);
}

struct Backward {
  int64_t piece, dp, lds;  // lds: row stride of ds
  float *scale;
  void *h;                  // masked copy of H [rows, dp]
  __nv_bfloat16 *w;         // a piece of W [piece, dp], when its rows are not aligned
  void *ds;                 // [rows, lds]
  bool copy_w;
  float *dh_planes, *dw_planes;
  int dh_split, dw_split;
  bool dh_direct, dw_direct;
  float *h_hi, *h_lo;
  void *gemm;
  size_t gemm_bytes;
};

silcu_gemm_args dh_args(const Args &a, const float *ds, int64_t lds, int64_t v0, int64_t n) {
  silcu_gemm_args g = f32_args(a.rows, a.D, n);
  g.A = ds;
  g.lda = lds;
  g.B = static_cast<const float *>(a.W) + v0 * a.ldw;
  g.ldb = a.ldw;
  g.C = static_cast<float *>(a.dH);
  g.ldc = a.lddh;
  if (v0) {  // earlier pieces' sum
    g.residual = g.C;
    g.ldr = a.lddh;
  }
  return g;
}

silcu_gemm_args dw_args(const Args &a, const float *ds, int64_t lds, const float *h, int64_t dp, int64_t v0,
                        int64_t n) {
  silcu_gemm_args g = f32_args(n, a.D, a.rows);
  g.A = ds;
  g.lda = lds;
  g.trans_a = 1;
  g.B = h;
  g.ldb = dp;
  g.C = static_cast<float *>(a.dW) + v0 * a.lddw;
  g.ldc = a.lddw;
  return g;
}

Backward plan_backward(const Args &a, Space &sp) {
  Backward b = {};
  b.scale = sp.take<float>(a.rows);
  if (a.dtype == SILCU_BF16) {
    b.dp = up(a.D, 8);
    b.copy_w = !rows16(a.W, a.ldw, a.dtype);
    const int64_t per_col = 2 * a.rows > 2 * b.dp || !b.copy_w ? 2 * a.rows : 2 * b.dp;
    b.piece = piece_of(a.V, per_col);
    b.lds = up(b.piece, 64);
    b.h = sp.take<__nv_bfloat16>(a.rows * b.dp);
    if (b.copy_w) b.w = sp.take<__nv_bfloat16>(b.piece * b.dp);
    b.ds = sp.take<__nv_bfloat16>(a.rows * b.lds);
    if (a.dH) {
      b.dh_split = split_k(a.rows, a.D, b.piece);
      b.dh_direct = b.dh_split == 1 && b.piece == a.V;
      if (!b.dh_direct) b.dh_planes = sp.take<float>(b.dh_split * a.rows * b.dp);
    }
    if (a.dW) {
      b.dw_split = split_k(b.piece, a.D, a.rows);
      b.dw_direct = b.dw_split == 1;
      if (!b.dw_direct) b.dw_planes = sp.take<float>(b.dw_split * b.piece * b.dp);
    }
  } else {
    b.dp = up(a.D, 4);
    b.piece = piece_of(a.V, 4 * a.rows > 8 * b.dp ? 4 * a.rows : 8 * b.dp);
    b.lds = up(b.piece, 4);
    b.h = sp.take<float>(a.rows * b.dp);
    b.h_hi = sp.take<float>(a.rows * b.dp);
    b.h_lo = sp.take<float>(a.rows * b.dp);
    b.ds = sp.take<float>(a.rows * b.lds);
    b.gemm_bytes = most_over_pieces(a.V, b.piece, [&](int64_t n) {
      silcu_gemm_args s = score_args(a, given(), given(), b.dp, 0, n);
      s.C = given();
      size_t most = tc_loss_workspace_bytes(s);
      for (const bool first : {true, false}) {  // with and without an earlier sum to add
        silcu_gemm_args g = dh_args(a, given(), b.lds, first ? 0 : 256, n);
        g.C = given();
        const size_t w = tc_workspace_bytes(g);
        if (w > most) most = w;
      }
      silcu_gemm_args g = dw_args(a, given(), b.lds, given(), b.dp, 0, n);
      g.C = given();
      const size_t w = tc_workspace_bytes(g);
      return w > most ? w : most;
    });
    b.gemm = sp.take<char>(int64_t(b.gemm_bytes));
  }
  return b;
}

// ---------------------------------------------------------------------- run
silcu_status copy_bf16(const void *src, int64_t ld, int64_t rows, int64_t D, int64_t dp, const int32_t *targets,
                       int64_t V, __nv_bfloat16 *dst, cudaStream_t s) {
  copy_rows<__nv_bfloat16><<<stream_grid(rows * dp / 8), 256, 0, s>>>(
      static_cast<const __nv_bfloat16 *>(src), ld, rows, int(D), int(dp), targets, int(V), dst);
  return check_launch("cross_entropy copy");
}

template <int EPI>
silcu_status bf16_scores(bf16::Params &p, bool pair, cudaStream_t s) {
  return pair ? bf16::launch<false, false, EPI, true>(p, s) : bf16::launch<false, false, EPI, false>(p, s);
}

silcu_status map_error() { return fail(SILCU_CUDA_ERROR, "cross_entropy: cuTensorMapEncodeTiled failed"); }

silcu_status forward(const Args &a, const Forward &f, cudaStream_t s) {
  silcu_status st;
  LossArgs loss = {};
  loss.targets = a.targets;
  loss.V = int32_t(a.V);
  loss.part = f.part;
  loss.target_score = f.target_score;
  if (a.dtype == SILCU_BF16) {
    bf16::Operand h{a.H, a.ldh, false};
    if (f.copy_h) {
      if ((st = copy_bf16(a.H, a.ldh, a.rows, a.D, f.dp, nullptr, 0, f.h, s)) != SILCU_OK) return st;
      h = {f.h, f.dp, false};
    }
    for (int64_t v0 = 0; v0 < a.V; v0 += f.piece) {
      const int64_t n = a.V - v0 < f.piece ? a.V - v0 : f.piece;
      const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(a.W) + v0 * a.ldw;
      bf16::Operand w{src, a.ldw, false};
      if (f.copy_w) {
        if ((st = copy_bf16(src, a.ldw, n, a.D, f.dp, nullptr, 0, f.w, s)) != SILCU_OK) return st;
        w = {f.w, f.dp, false};
      }
      bf16::Params p;
      memset(&p, 0, sizeof(p));
      const bool pair = a.rows > bf16::BM;
      if (!bf16::set_operands(p, pair, a.rows, n, a.D, h, w)) return map_error();
      p.loss = loss;
      p.loss.v0 = int32_t(v0);
      p.err = device_error_ptr();
      if ((st = bf16_scores<bf16::kStats>(p, pair, s)) != SILCU_OK) return st;
    }
  } else {
    st = split_rows(static_cast<const float *>(a.H), a.ldh, 1, a.rows, a.D, f.dp, f.h_hi, f.h_lo, s);
    if (st != SILCU_OK) return st;
    for (int64_t v0 = 0; v0 < a.V; v0 += f.piece) {
      const int64_t n = a.V - v0 < f.piece ? a.V - v0 : f.piece;
      loss.v0 = int32_t(v0);
      st = tc_run_loss(score_args(a, f.h_hi, f.h_lo, f.dp, v0, n), kLossStats, loss, f.gemm, f.gemm_bytes, s);
      if (st != SILCU_OK) return st;
    }
  }
  loss_finish<<<uint32_t((a.rows + 31) / 32), 256, 0, s>>>(f.part, int((a.V + 127) / 128), a.rows, a.targets,
                                                           int(a.V), f.target_score, a.lse, f.row_loss);
  if ((st = check_launch("cross_entropy finish")) != SILCU_OK || a.reduction == SILCU_REDUCE_NONE) return st;
  loss_reduce<<<1, 1024, 0, s>>>(f.row_loss, a.targets, a.rows, int(a.V), a.reduction == SILCU_REDUCE_MEAN, a.loss);
  return check_launch("cross_entropy reduce");
}

silcu_status backward_bf16(const Args &a, const Backward &b, cudaStream_t s) {
  silcu_status st;
  __nv_bfloat16 *hm = static_cast<__nv_bfloat16 *>(b.h), *ds = static_cast<__nv_bfloat16 *>(b.ds);
  if ((st = copy_bf16(a.H, a.ldh, a.rows, a.D, b.dp, a.targets, a.V, hm, s)) != SILCU_OK) return st;
  const bool dh_vec = rows16(a.dH, a.lddh, a.dtype), dw_vec = rows16(a.dW, a.lddw, a.dtype);
  const bool pair = a.rows > bf16::BM;
  for (int64_t v0 = 0; v0 < a.V; v0 += b.piece) {
    const int64_t n = a.V - v0 < b.piece ? a.V - v0 : b.piece;
    const void *w = static_cast<const __nv_bfloat16 *>(a.W) + v0 * a.ldw;
    int64_t ldw = a.ldw;
    if (b.copy_w) {
      if ((st = copy_bf16(w, a.ldw, n, a.D, b.dp, nullptr, 0, b.w, s)) != SILCU_OK) return st;
      w = b.w;
      ldw = b.dp;
    }
    bf16::Params p;
    memset(&p, 0, sizeof(p));
    p.err = device_error_ptr();
    if (!bf16::set_operands(p, pair, a.rows, n, a.D, {hm, b.dp, false}, {w, ldw, false}) ||
        !tc::make_map2_bf16(&p.c, ds, n, a.rows, b.lds, 64, 32))
      return map_error();
    p.loss.targets = a.targets;
    p.loss.V = int32_t(a.V);
    p.loss.v0 = int32_t(v0);
    p.loss.lse = a.lse;
    p.loss.scale = b.scale;
    if ((st = bf16_scores<bf16::kScoreGrad>(p, pair, s)) != SILCU_OK) return st;
    if (a.dH) {
      if (!bf16::set_operands(p, pair, a.rows, a.D, n, {ds, b.lds, false}, {w, ldw, true})) return map_error();
      const int nk = int((n + bf16::BK - 1) / bf16::BK);
      p.ksplit = b.dh_split < nk ? b.dh_split : nk;  // a short last piece adds to the first planes only
      if (b.dh_direct) {
        p.mode = bf16::kOutBf16;
        p.out = a.dH;
        p.ldo = a.lddh;
        p.vec = dh_vec;
      } else {
        p.mode = v0 ? bf16::kOutPlaneAdd : bf16::kOutPlane;
        p.out = b.dh_planes;
        p.ldo = b.dp;
        p.plane = a.rows * b.dp;
      }
      st = pair ? bf16::launch<false, true, bf16::kOut, true>(p, s) : bf16::launch<false, true, bf16::kOut, false>(p, s);
      if (st != SILCU_OK) return st;
    }
    if (a.dW) {
      const bool wide = n > bf16::BM;
      if (!bf16::set_operands(p, wide, n, a.D, a.rows, {ds, b.lds, true}, {hm, b.dp, true})) return map_error();
      __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(a.dW) + v0 * a.lddw;
      p.ksplit = b.dw_split;
      if (b.dw_direct) {
        p.mode = bf16::kOutBf16;
        p.out = out;
        p.ldo = a.lddw;
        p.vec = dw_vec;
      } else {
        p.mode = bf16::kOutPlane;
        p.out = b.dw_planes;
        p.ldo = b.dp;
        p.plane = b.piece * b.dp;
      }
      st = wide ? bf16::launch<true, true, bf16::kOut, true>(p, s) : bf16::launch<true, true, bf16::kOut, false>(p, s);
      if (st != SILCU_OK) return st;
      if (!b.dw_direct) {
        planes_finish<<<stream_grid(n * b.dp / 8), 256, 0, s>>>(b.dw_planes, b.dw_split, p.plane, n, int(a.D),
                                                                int(b.dp), out, a.lddw, dw_vec);
        if ((st = check_launch("cross_entropy planes")) != SILCU_OK) return st;
      }
    }
  }
  if (a.dH && !b.dh_direct) {
    planes_finish<<<stream_grid(a.rows * b.dp / 8), 256, 0, s>>>(b.dh_planes, b.dh_split, a.rows * b.dp, a.rows,
                                                                 int(a.D), int(b.dp),
                                                                 static_cast<__nv_bfloat16 *>(a.dH), a.lddh, dh_vec);
    return check_launch("cross_entropy planes");
  }
  return SILCU_OK;
}

silcu_status backward_f32(const Args &a, const Backward &b, cudaStream_t s) {
  silcu_status st;
  float *hm = static_cast<float *>(b.h), *ds = static_cast<float *>(b.ds);
  copy_rows<float><<<stream_grid(a.rows * b.dp / 4), 256, 0, s>>>(static_cast<const float *>(a.H), a.ldh, a.rows,
                                                                  int(a.D), int(b.dp), a.targets, int(a.V), hm);
  if ((st = check_launch("cross_entropy copy")) != SILCU_OK) return st;
  if ((st = split_rows(hm, b.dp, 1, a.rows, a.D, b.dp, b.h_hi, b.h_lo, s)) != SILCU_OK) return st;
  LossArgs loss = {};
  loss.targets = a.targets;
  loss.V = int32_t(a.V);
  loss.lse = a.lse;
  loss.scale = b.scale;
  for (int64_t v0 = 0; v0 < a.V; v0 += b.piece) {
    const int64_t n = a.V - v0 < b.piece ? a.V - v0 : b.piece;
    loss.v0 = int32_t(v0);
    silcu_gemm_args g = score_args(a, b.h_hi, b.h_lo, b.dp, v0, n);
    g.C = ds;
    g.ldc = b.lds;
    if ((st = tc_run_loss(g, kLossGrad, loss, b.gemm, b.gemm_bytes, s)) != SILCU_OK) return st;
    if (a.dH && (st = tc_run(dh_args(a, ds, b.lds, v0, n), b.gemm, b.gemm_bytes, s)) != SILCU_OK) return st;
    if (a.dW && (st = tc_run(dw_args(a, ds, b.lds, hm, b.dp, v0, n), b.gemm, b.gemm_bytes, s)) != SILCU_OK) return st;
  }
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
  return SILCU_OK;
}

silcu_status check_space(const char *what, const Args &a, int backward, void *ws, size_t bytes) {
  const size_t need = silcu_linear_cross_entropy_workspace_bytes(&a, backward);
  if (!ws || bytes < need) return fail(SILCU_WORKSPACE_TOO_SMALL, "%s: workspace %zu < %zu", what, bytes, need);
  if (!device_error_ptr()) return fail(SILCU_CUDA_ERROR, "%s: no device error word", what);
  return SILCU_OK;
}

char *align256(void *p) { return reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(p) + 255) & ~uintptr_t(255)); }

}  // namespace
}  // namespace silcu

extern "C" {

size_t silcu_linear_cross_entropy_workspace_bytes(const silcu_cross_entropy_args *ap, int backward) {
  using namespace silcu;
  if (check_shape("linear_cross_entropy_workspace_bytes", ap) != SILCU_OK || ap->rows == 0) return 0;
  Space f{nullptr}, b{nullptr};
  plan_forward(*ap, f);
  if (backward) plan_backward(*ap, b);
  return (f.used > b.used ? f.used : b.used) + 256;  // the caller's pointer need not be aligned
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
    loss_reduce<<<1, 1024, 0, s>>>(nullptr, nullptr, 0, int(a.V), 0, a.loss);
    return check_launch("linear_cross_entropy");
  }
  if ((st = check_pointers("linear_cross_entropy", a)) != SILCU_OK) return st;
  if ((st = check_space("linear_cross_entropy", a, 0, workspace, workspace_bytes)) != SILCU_OK) return st;
  Space sp{align256(workspace)};
  return forward(a, plan_forward(a, sp), s);
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
  if ((st = check_space(what, a, 1, workspace, workspace_bytes)) != SILCU_OK) return st;
  Space sp{align256(workspace)};
  const Backward b = plan_backward(a, sp);
  row_scales<<<1, 1024, 0, s>>>(a.dloss, a.targets, a.rows, int(a.V), a.reduction, b.scale);
  if ((st = check_launch(what)) != SILCU_OK) return st;
  return a.dtype == SILCU_BF16 ? backward_bf16(a, b, s) : backward_f32(a, b, s);
}

}  // extern "C"
