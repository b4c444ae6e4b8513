// layer_norm for training: the forward pass that keeps each row's statistics,
// and the backward pass with the reduction of gamma's and beta's gradients.
//
//   mu = avg(x), r = 1 / sqrt(avg((x - mu)^2) + eps), xh = (x - mu) r, y = xh gamma + beta
//   a = dy gamma,  dx = r (a - avg(a) - xh avg(a xh)) (+ residual gradient)
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// Both are bound by HBM: the forward reads x and writes y, the backward reads
// dy, x (and the residual gradient) and writes dx, each once.  A row lives in
// the registers of a warp (short rows) or of a CTA, 4 to 32 elements a thread;
// beyond 16384 columns a CTA re-reads its row.  Elements move as 16-byte
// vectors where columns and pointers allow (4 fp32 / 8 bf16), else one by one.
//
// Three kernels, by what keeps the memory busy (measured, rows rotating
// through more than the L2):
//   ln_forward         a group of threads per row, many short-lived CTAs: fp32
//                      rows, 8192 x 4096 in 43.3 us (6.2 TB/s; persistent with
//                      prefetch 47.4).
//   ln_forward_stream  bf16 vectors: persistent, the next row's loads in flight
//                      during this row's sums, gamma and beta in shared memory.
//                      At 8 elements a vector the parameters weigh twice the
//                      row, and read from global memory with a 32-byte lane
//                      stride they keep the L1 77 % busy: 4096 x 8192 39.2 us
//                      with ln_forward, 31.4 persistent, 28.5 with shared memory.
//                      Started early behind its predecessor (launch_after) 24.9, 26.8
//                      without; for ln_forward's many CTAs the waits cost more than
//                      that gives (16384 x 768 19.4 us, 16.5 without).
//   ln_backward        persistent, prefetching; each thread adds its columns'
//                      dgamma / dbeta terms in registers over all rows of its CTA,
//                      one partial row per CTA, added in CTA order by ln_finish.
//                      16384 x 768 fp32 with residual: 34 us (5.9 TB/s), 48 with a
//                      warp per row (151 registers, one CTA per SM); 8190 x 4096
//                      bf16: 72 us with the sums in shared memory instead.
// All sums are fp32 in an order fixed by the shape and the SM count.
#include <initializer_list>

#include "elem.cuh"

namespace silcu {
namespace {

struct LnArgs {
  const void *in, *dout, *dres;
  void *out;
  float *mean_out, *rstd_out;
  const float *mean, *rstd, *gamma, *beta;
  float *part;
  uint64_t rows;
  uint32_t cols;
  float eps;
};

constexpr uint32_t kMaxRegCols = 16384;

template <int NT>
__device__ __forceinline__ float group_sum(float v, float *smem) {
  v = warp_sum(v);
  if (NT == 32) return v;
  constexpr int NW = NT / 32;
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < NW; i++) r += smem[i];
  return r;
}

// ------------------------------------------------------------------ forward
template <typename T, int VEC, int VPT, int NT, int GROUPS>
__global__ void __launch_bounds__(NT *GROUPS) ln_forward(const LnArgs a) {
  __shared__ float sm[2][NT / 32];
  const uint32_t t = threadIdx.x % NT;
  const uint64_t row = uint64_t(blockIdx.x) * GROUPS + threadIdx.x / NT;
  if (row >= a.rows) return;  // a whole group: only GROUPS > 1 has partial CTAs, and those use no CTA barrier
  const T *src = static_cast<const T *>(a.in) + row * a.cols;
  T *dst = static_cast<T *>(a.out) + row * a.cols;
  Raw<T, VEC> raw[VPT];
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const uint32_t c = (t + j * NT) * VEC;
    raw[j] = c < a.cols ? raw_load<T, VEC>(src + c) : raw_zero<T, VEC>();
  }
  const float inv_n = 1.0f / float(a.cols);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    float v[VEC];
    unpack(raw[j], v);
#pragma unroll
    for (int k = 0; k < VEC; k++) s += v[k];
  }
  const float mu = group_sum<NT>(s, sm[0]) * inv_n;
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    if ((t + j * NT) * VEC < a.cols) {
      float v[VEC];
      unpack(raw[j], v);
#pragma unroll
      for (int k = 0; k < VEC; k++) {
        const float d = v[k] - mu;
        ss = fmaf(d, d, ss);
      }
    }
  }
  const float rstd = rsqrtf(group_sum<NT>(ss, sm[1]) * inv_n + a.eps);
  if (t == 0) {
    if (a.mean_out) a.mean_out[row] = mu;
    if (a.rstd_out) a.rstd_out[row] = rstd;
  }
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const uint32_t c = (t + j * NT) * VEC;
    if (c < a.cols) {
      float v[VEC], gm[VEC], bt[VEC];
      unpack(raw[j], v);
      load_f32<VEC>(a.gamma + c, gm);
      load_f32<VEC>(a.beta + c, bt);
#pragma unroll
      for (int k = 0; k < VEC; k++) v[k] = fmaf((v[k] - mu) * rstd, gm[k], bt[k]);
      Raw<T, VEC> o;
      pack(v, o);
      raw_store<T, VEC>(dst + c, o);
    }
  }
}

// Parameters in shared memory, laid out so that the float4 h of a thread's
// vectors are NT apart: conflict-free for VEC = 8, where global loads would
// step 32 bytes per lane.
template <int VEC, int VPT, int NT>
__device__ __forceinline__ void params_to_smem(float4 *s, const float *g, uint32_t cols, uint32_t t) {
#pragma unroll
  for (int j = 0; j < VPT; j++) {
    const uint32_t i = t + j * NT, c = i * VEC;
    if (c < cols) {
#pragma unroll
      for (int h = 0; h < VEC / 4; h++) s[h * VPT * NT + i] = *reinterpret_cast<const float4 *>(g + c + 4 * h);
    }
  }
}
template <int VEC, int VPT, int NT>
__device__ __forceinline__ void params_from_smem(const float4 *s, int j, uint32_t t, float (&f)[VEC]) {
#pragma unroll
  for (int h = 0; h < VEC / 4; h++) {
    const float4 v = s[h * VPT * NT + t + j * NT];
    f[4 * h] = v.x, f[4 * h + 1] = v.y, f[4 * h + 2] = v.z, f[4 * h + 3] = v.w;
  }
}

// One CTA per row at a time, persistent, the next row in flight.
template <typename T, int VEC, int VPT, int NT, int MIN_CTAS>
__global__ void __launch_bounds__(NT, MIN_CTAS) ln_forward_stream(const LnArgs a) {
  constexpr int NW = NT / 32;
  extern __shared__ __align__(16) float4 ps[];  // gamma, beta
  __shared__ float sm[2][2][NW];
  const float4 *gs = ps, *bs = ps + VPT * NT * VEC / 4;
  const uint32_t t = threadIdx.x;
  let_next_start();
  wait_for_previous();
  params_to_smem<VEC, VPT, NT>(ps, a.gamma, a.cols, t);  // each thread reads back what it wrote
  params_to_smem<VEC, VPT, NT>(ps + VPT * NT * VEC / 4, a.beta, a.cols, t);
  const float inv_n = 1.0f / float(a.cols);
  Raw<T, VEC> raw[VPT], next[VPT];
  auto load = [&](uint64_t r) {
    const T *src = static_cast<const T *>(a.in) + r * a.cols;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      next[j] = c < a.cols ? raw_load<T, VEC>(src + c) : raw_zero<T, VEC>();
    }
  };
  uint64_t row = blockIdx.x;
  if (row < a.rows) load(row);
  for (int b = 0; row < a.rows; row += gridDim.x, b ^= 1) {
#pragma unroll
    for (int j = 0; j < VPT; j++) raw[j] = next[j];
    if (row + gridDim.x < a.rows) load(row + gridDim.x);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      float v[VEC];
      unpack(raw[j], v);
#pragma unroll
      for (int k = 0; k < VEC; k++) s += v[k];
    }
    // buffer b: its last readers have passed the two barriers of the row between
    const float mu = group_sum<NT>(s, sm[b][0]) * inv_n;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      if ((t + j * NT) * VEC < a.cols) {
        float v[VEC];
        unpack(raw[j], v);
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const float d = v[k] - mu;
          ss = fmaf(d, d, ss);
        }
      }
    }
    const float rstd = rsqrtf(group_sum<NT>(ss, sm[b][1]) * inv_n + a.eps);
    if (t == 0) {
      if (a.mean_out) a.mean_out[row] = mu;
      if (a.rstd_out) a.rstd_out[row] = rstd;
    }
    T *dst = static_cast<T *>(a.out) + row * a.cols;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      if (c < a.cols) {
        float v[VEC], gm[VEC], bt[VEC];
        unpack(raw[j], v);
        params_from_smem<VEC, VPT, NT>(gs, j, t, gm);
        params_from_smem<VEC, VPT, NT>(bs, j, t, bt);
#pragma unroll
        for (int k = 0; k < VEC; k++) v[k] = fmaf((v[k] - mu) * rstd, gm[k], bt[k]);
        Raw<T, VEC> o;
        pack(v, o);
        raw_store<T, VEC>(dst + c, o);
      }
    }
  }
}

// Rows beyond kMaxRegCols: a CTA reads its row three times (L2 holds it).
template <typename T>
__global__ void __launch_bounds__(512) ln_forward_long(const LnArgs a) {
  __shared__ float sm[2][16];
  const uint64_t row = blockIdx.x;
  const T *src = static_cast<const T *>(a.in) + row * a.cols;
  T *dst = static_cast<T *>(a.out) + row * a.cols;
  const float inv_n = 1.0f / float(a.cols);
  auto at = [&](uint32_t c) {
    Raw<T, 1> r;
    r.r = *reinterpret_cast<const decltype(r.r) *>(src + c);
    float v[1];
    unpack(r, v);
    return v[0];
  };
  float s = 0.f;
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) s += at(c);
  const float mu = group_sum<512>(s, sm[0]) * inv_n;
  float ss = 0.f;
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) {
    const float d = at(c) - mu;
    ss = fmaf(d, d, ss);
  }
  const float rstd = rsqrtf(group_sum<512>(ss, sm[1]) * inv_n + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean_out) a.mean_out[row] = mu;
    if (a.rstd_out) a.rstd_out[row] = rstd;
  }
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) {
    float v[1] = {fmaf((at(c) - mu) * rstd, a.gamma[c], a.beta[c])};
    Raw<T, 1> o;
    pack(v, o);
    raw_store<T, 1>(dst + c, o);
  }
}

// ----------------------------------------------------------------- backward
// One row of a group: the raw vectors of x, dy and the residual gradient.
template <typename T, int VEC, int VPT, int NT, bool RES>
struct LnRow {
  Raw<T, VEC> x[VPT], dy[VPT], res[RES ? VPT : 1];
  float mean, rstd;
  __device__ __forceinline__ void load(const LnArgs &a, uint64_t row, uint32_t t) {
    const T *px = static_cast<const T *>(a.in) + row * a.cols;
    const T *py = static_cast<const T *>(a.dout) + row * a.cols;
    const T *pr = static_cast<const T *>(a.dres) + row * a.cols;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      const bool in = c < a.cols;
      x[j] = in ? raw_load<T, VEC>(px + c) : raw_zero<T, VEC>();
      dy[j] = in ? raw_load<T, VEC>(py + c) : raw_zero<T, VEC>();
      if (RES) res[j] = in ? raw_load<T, VEC>(pr + c) : raw_zero<T, VEC>();
    }
    mean = a.mean[row];
    rstd = a.rstd[row];
  }
};

// Rows of more than 8192 columns (32 elements a thread) have no registers for
// the sums and the next row: the sums then live in shared memory.  512 threads have 128
// registers each, and rows of 4097 to 8192 columns (16 elements) spill some of theirs: 104
// bytes a thread of fp32 vectors with a residual gradient, up to 306 where elements move one
// by one.
template <int VEC, int VPT, int NT, int GROUPS>
struct BwdCfg {
  static constexpr int E = VEC * VPT;
  static constexpr bool WIDE = E == 32;
  static constexpr bool PARAMS = VEC == 8;  // gamma in shared memory
  static constexpr int PARAM_FLOATS = PARAMS ? E * NT : 0;
  static constexpr bool ACC_S = WIDE || GROUPS > 1;
  static uint32_t smem(uint32_t cols) { return (PARAM_FLOATS + (ACC_S ? 2 * cols : 0)) * sizeof(float); }
};

template <typename T, int VEC, int VPT, int NT, int GROUPS, bool RES>
__global__ void __launch_bounds__(NT *GROUPS) ln_backward(const LnArgs a) {
  using Cfg = BwdCfg<VEC, VPT, NT, GROUPS>;
  constexpr int NW = NT / 32, E = VPT * VEC;
  constexpr bool WARP = NT == 32, ACCREG = !Cfg::WIDE, PF = !Cfg::WIDE;
  extern __shared__ __align__(16) float dyn[];
  float *acc_s = dyn + Cfg::PARAM_FLOATS;  // dgamma[cols], dbeta[cols] of this CTA
  const float4 *gs = reinterpret_cast<const float4 *>(dyn);
  __shared__ float2 sm[2][NW];
  const uint32_t t = threadIdx.x % NT, g = threadIdx.x / NT;
  auto gamma_at = [&](int j, float(&f)[VEC]) {
    if constexpr (Cfg::PARAMS) params_from_smem<VEC, VPT, NT>(gs, j, t, f);
    else load_f32<VEC>(a.gamma + (t + j * NT) * VEC, f);
  };
  let_next_start();
  wait_for_previous();
  if constexpr (Cfg::PARAMS) params_to_smem<VEC, VPT, NT>(reinterpret_cast<float4 *>(dyn), a.gamma, a.cols, t);
  float ag[ACCREG ? E : 1], ab[ACCREG ? E : 1];
  if (ACCREG) {
#pragma unroll
    for (int i = 0; i < E; i++) ag[ACCREG ? i : 0] = ab[ACCREG ? i : 0] = 0.f;
  } else {
    for (uint32_t c = threadIdx.x; c < 2 * a.cols; c += NT * GROUPS) acc_s[c] = 0.f;
    __syncthreads();
  }
  const float inv_n = 1.0f / float(a.cols);
  const uint64_t step = uint64_t(gridDim.x) * GROUPS;
  int buf = 0;
  LnRow<T, VEC, VPT, NT, RES> r, next;
  uint64_t row = uint64_t(blockIdx.x) * GROUPS + g;
  if (PF && row < a.rows) next.load(a, row, t);
  for (; row < a.rows; row += step) {
    if (PF) {
      r = next;
      if (row + step < a.rows) next.load(a, row + step, t);
    } else {
      r.load(a, row, t);
    }
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      if (c < a.cols) {
        float x[VEC], dy[VEC], gm[VEC], sg[VEC], sb[VEC];
        unpack(r.x[j], x);
        unpack(r.dy[j], dy);
        gamma_at(j, gm);
        if (!ACCREG) {
          load_f32<VEC>(acc_s + c, sg);
          load_f32<VEC>(acc_s + a.cols + c, sb);
        }
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const float xh = (x[k] - r.mean) * r.rstd;
          const float w = dy[k] * gm[k];
          c1 += w;
          c2 = fmaf(w, xh, c2);
          if (ACCREG) {
            const int i = ACCREG ? j * VEC + k : 0;
            ag[i] = fmaf(dy[k], xh, ag[i]);
            ab[i] += dy[k];
          } else {
            sg[k] = fmaf(dy[k], xh, sg[k]);
            sb[k] += dy[k];
          }
        }
        if (!ACCREG) {
          store_f32<VEC>(acc_s + c, sg);
          store_f32<VEC>(acc_s + a.cols + c, sb);
        }
      }
    }
    c1 = warp_sum(c1);
    c2 = warp_sum(c2);
    if (!WARP) {
      if ((threadIdx.x & 31) == 0) sm[buf][threadIdx.x >> 5] = make_float2(c1, c2);
      __syncthreads();  // the other buffer's readers are past it once every warp is here
      c1 = c2 = 0.f;
#pragma unroll
      for (int i = 0; i < NW; i++) {
        c1 += sm[buf][i].x;
        c2 += sm[buf][i].y;
      }
      buf ^= 1;
    }
    c1 *= inv_n;
    c2 *= inv_n;
    T *dst = static_cast<T *>(a.out) + row * a.cols;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      if (c < a.cols) {
        float x[VEC], dy[VEC], gm[VEC], res[VEC];
        unpack(r.x[j], x);
        unpack(r.dy[j], dy);
        gamma_at(j, gm);
        if (RES) unpack(r.res[RES ? j : 0], res);
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const float xh = (x[k] - r.mean) * r.rstd;
          const float w = dy[k] * gm[k];
          x[k] = r.rstd * (w - c1 - xh * c2);
          if (RES) x[k] += res[k];
        }
        Raw<T, VEC> o;
        pack(x, o);
        raw_store<T, VEC>(dst + c, o);
      }
    }
  }
  float *part = a.part + uint64_t(blockIdx.x) * 2 * a.cols;
  if (ACCREG && GROUPS == 1) {
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      if (c < a.cols) {
        float sg[VEC], sb[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const int i = ACCREG ? j * VEC + k : 0;
          sg[k] = ag[i];
          sb[k] = ab[i];
        }
        store_f32<VEC>(part + c, sg);
        store_f32<VEC>(part + a.cols + c, sb);
      }
    }
    return;
  }
  if (ACCREG) {  // the CTA's groups add their sums in order
#pragma unroll 1
    for (int w = 0; w < GROUPS; w++) {
      if (int(g) == w) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
          const uint32_t c = (t + j * NT) * VEC;
          if (c < a.cols) {
#pragma unroll
            for (int k = 0; k < VEC; k++) {
              const int i = ACCREG ? j * VEC + k : 0;
              acc_s[c + k] = w ? acc_s[c + k] + ag[i] : ag[i];
              acc_s[a.cols + c + k] = w ? acc_s[a.cols + c + k] + ab[i] : ab[i];
            }
          }
        }
      }
      __syncthreads();
    }
  } else {
    __syncthreads();
  }
  for (uint32_t c = threadIdx.x; c < 2 * a.cols; c += NT * GROUPS) part[c] = acc_s[c];
}

// Rows beyond kMaxRegCols.  The column sums run first (din may be dout or in).
template <typename T>
__global__ void __launch_bounds__(256) ln_backward_cols(const LnArgs a) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.cols) return;
  const T *px = static_cast<const T *>(a.in), *py = static_cast<const T *>(a.dout);
  float g = 0.f, b = 0.f;
  for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    float x[1], dy[1];
    unpack(raw_load<T, 1>(px + row * a.cols + c), x);
    unpack(raw_load<T, 1>(py + row * a.cols + c), dy);
    g = fmaf(dy[0], (x[0] - a.mean[row]) * a.rstd[row], g);
    b += dy[0];
  }
  float *part = a.part + uint64_t(blockIdx.y) * 2 * a.cols;
  part[c] = g;
  part[a.cols + c] = b;
}

template <typename T, bool RES>
__global__ void __launch_bounds__(512) ln_backward_long(const LnArgs a) {
  __shared__ float sm[2][16];
  const uint64_t row = blockIdx.x;
  const T *px = static_cast<const T *>(a.in) + row * a.cols;
  const T *py = static_cast<const T *>(a.dout) + row * a.cols;
  const T *pr = static_cast<const T *>(a.dres) + row * a.cols;
  T *dst = static_cast<T *>(a.out) + row * a.cols;
  const float mean = a.mean[row], rstd = a.rstd[row], inv_n = 1.0f / float(a.cols);
  auto at = [&](const T *p, uint32_t c) {
    Raw<T, 1> r;
    r.r = *reinterpret_cast<const decltype(r.r) *>(p + c);
    float v[1];
    unpack(r, v);
    return v[0];
  };
  float c1 = 0.f, c2 = 0.f;
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) {
    const float w = at(py, c) * a.gamma[c];
    c1 += w;
    c2 = fmaf(w, (at(px, c) - mean) * rstd, c2);
  }
  c1 = group_sum<512>(c1, sm[0]) * inv_n;
  c2 = group_sum<512>(c2, sm[1]) * inv_n;
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) {
    float v[1] = {rstd * (at(py, c) * a.gamma[c] - c1 - (at(px, c) - mean) * rstd * c2)};
    if (RES) v[0] += at(pr, c);
    Raw<T, 1> o;
    pack(v, o);
    raw_store<T, 1>(dst + c, o);
  }
}

// dgamma / dbeta: the partial rows added in an order that only their number
// decides.  COLS columns a CTA, 1024 / COLS threads for the rows of each.  Few columns
// spread over more SMs with 8 of them (768 columns, 888 partial rows: 4.7 us with 32).
template <int COLS>
__global__ void __launch_bounds__(1024) ln_finish(const float *part, uint32_t nparts, uint32_t cols, float *dgamma,
                                                  float *dbeta) {
  constexpr uint32_t SLICES = 1024 / COLS;
  __shared__ float sm[32][33];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * COLS + threadIdx.x % COLS;
  float s = 0.f;
  let_next_start();
  wait_for_previous();
  if (c < 2 * cols) {
#pragma unroll 8
    for (uint32_t i = threadIdx.x / COLS; i < nparts; i += SLICES) s += load_streaming(part + uint64_t(i) * 2 * cols + c);
  }
#pragma unroll
  for (int step = COLS; step < 32; step *= 2) s += __shfl_xor_sync(0xffffffffu, s, step);
  if (lane < COLS) sm[warp][lane] = s;
  __syncthreads();
  if (warp < COLS) {  // the warps' sums of column `warp`
    s = warp_sum(sm[lane][warp]);
    const uint32_t col = blockIdx.x * COLS + warp;
    if (lane == 0 && col < 2 * cols) {
      if (col < cols) dgamma[col] = s;
      else dbeta[col - cols] = s;
    }
  }
}

// --------------------------------------------------------------------- host
// Calls f.run<VEC, VPT, NT, GROUPS>() with NT threads of VEC * VPT elements for
// a row of `cols`.
template <int VEC, typename F>
silcu_status by_cols_forward(uint32_t cols, F &&f) {
  if (cols <= 32 * 8) return f.template run<VEC, 8 / VEC, 32, 8>();
  if (cols <= 64 * 8) return f.template run<VEC, 8 / VEC, 64, 1>();
  if (cols <= 96 * 8) return f.template run<VEC, 8 / VEC, 96, 1>();
  if (cols <= 128 * 8) return f.template run<VEC, 8 / VEC, 128, 1>();
  if (cols <= 128 * 16) return f.template run<VEC, 16 / VEC, 128, 1>();
  if (cols <= 256 * 16) return f.template run<VEC, 16 / VEC, 256, 1>();
  if (cols <= 512 * 16) return f.template run<VEC, 16 / VEC, 512, 1>();
  return f.template run<VEC, 32 / VEC, 512, 1>();
}

// Measured for 16384 x 768: 192 threads of 4 fp32 elements 34 us, 96 of 8 35;
// bf16 96 of 8 21 us, a warp of 24 33.
template <int VEC, typename F>
auto by_cols_backward(uint32_t cols, F &&f) {
  if (cols <= 32 * 8) return f.template run<VEC, 8 / VEC, 32, 8>();
  if constexpr (VEC <= 4) {
    if (cols <= 128 * 4) return f.template run<VEC, 4 / VEC, 128, 1>();
    if (cols <= 192 * 4) return f.template run<VEC, 4 / VEC, 192, 1>();
    if (cols <= 128 * 8) return f.template run<VEC, 8 / VEC, 128, 1>();
    if (cols <= 256 * 8) return f.template run<VEC, 8 / VEC, 256, 1>();
  } else {
    if (cols <= 64 * 8) return f.template run<VEC, 1, 64, 1>();
    if (cols <= 96 * 8) return f.template run<VEC, 1, 96, 1>();
    if (cols <= 64 * 16) return f.template run<VEC, 2, 64, 1>();
    if (cols <= 128 * 16) return f.template run<VEC, 2, 128, 1>();
  }
  if (cols <= 256 * 16) return f.template run<VEC, 16 / VEC, 256, 1>();
  if (cols <= 512 * 16) return f.template run<VEC, 16 / VEC, 512, 1>();
  return f.template run<VEC, 32 / VEC, 512, 1>();
}

template <typename K>
silcu_status allow_smem(K kernel, uint32_t bytes, bool (&configured)[64], const char *what) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && configured[dev]) return SILCU_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  if (e != cudaSuccess) return fail(SILCU_CUDA_ERROR, "%s: smem attribute: %s", what, cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) configured[dev] = true;
  return SILCU_OK;
}

template <typename T>
struct Forward {
  LnArgs a;
  cudaStream_t s;
  template <int VEC, int VPT, int NT, int GROUPS>
  silcu_status run() {
    const uint64_t grid = (a.rows + GROUPS - 1) / GROUPS;
    ln_forward<T, VEC, VPT, NT, GROUPS><<<uint32_t(grid), NT * GROUPS, 0, s>>>(a);
    return check_launch("layer_norm_forward");
  }
  // CTAS per SM fill the registers (64 to 94 a thread).
  template <int VPT, int NT, int CTAS>
  silcu_status stream() {
    constexpr uint32_t smem = VPT * NT * 8 * 2 * sizeof(float);
    static bool configured[64] = {false};
    const silcu_status st =
        allow_smem(ln_forward_stream<T, 8, VPT, NT, CTAS>, smem, configured, "layer_norm_forward");
    if (st != SILCU_OK) return st;
    const uint64_t cap = uint64_t(sm_count()) * CTAS;
    launch_after(ln_forward_stream<T, 8, VPT, NT, CTAS>, uint32_t(a.rows < cap ? a.rows : cap), NT, smem, s, a);
    return check_launch("layer_norm_forward");
  }
};

// CTAs of the persistent backward grid: as many as the registers hold, two
// rows or more for each where that still fills the SMs (every CTA's partial
// row is written and read again).  The workspace holds one for each.
struct BackwardGrid {
  uint64_t rows;
  template <int VEC, int VPT, int NT, int GROUPS>
  uint32_t run() const {
    constexpr int E = VEC * VPT, threads = E == 4 ? 1152 : E == 8 ? 768 : E == 16 ? (NT <= 128 ? 640 : 512) : 512;
    constexpr int per_sm = threads / (NT * GROUPS);
    const uint64_t sms = uint64_t(sm_count()), groups = (rows + GROUPS - 1) / GROUPS;
    uint64_t g = groups / 2 > sms ? groups / 2 : sms;
    if (g > groups) g = groups;
    return uint32_t(g < sms * per_sm ? g : sms * per_sm);
  }
};
uint32_t long_grid(uint64_t rows) {
  const uint64_t sms = uint64_t(sm_count());
  return uint32_t(rows < sms ? rows : sms);
}

template <typename T, bool RES>
struct Backward {
  LnArgs a;
  cudaStream_t s;
  uint32_t *grid;  // its number of partial rows
  template <int VEC, int VPT, int NT, int GROUPS>
  silcu_status run() {
    using Cfg = BwdCfg<VEC, VPT, NT, GROUPS>;
    static bool configured[64] = {false};
    const auto kernel = ln_backward<T, VEC, VPT, NT, GROUPS, RES>;
    const silcu_status st = allow_smem(kernel, Cfg::smem(Cfg::E * NT), configured, "layer_norm_backward");
    if (st != SILCU_OK) return st;
    *grid = BackwardGrid{a.rows}.run<VEC, VPT, NT, GROUPS>();
    launch_after(kernel, *grid, NT * GROUPS, Cfg::smem(a.cols), s, a);
    return check_launch("layer_norm_backward");
  }
};

template <typename T>
silcu_status forward(const LnArgs &a, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (a.cols > kMaxRegCols) {
    ln_forward_long<T><<<uint32_t(a.rows), 512, 0, s>>>(a);
    return check_launch("layer_norm_forward");
  }
  Forward<T> f{a, s};
  const bool vec = a.cols % V == 0 && aligned16(a.in) && aligned16(a.out) && aligned16(a.gamma) && aligned16(a.beta);
  if constexpr (V == 8) {
    if (vec) {
      if (a.cols <= 256) return f.template stream<1, 32, 28>();
      if (a.cols <= 512) return f.template stream<2, 32, 24>();
      if (a.cols <= 768) return f.template stream<3, 32, 20>();
      if (a.cols <= 1024) return f.template stream<4, 32, 16>();
      if (a.cols <= 2048) return f.template stream<4, 64, 10>();
      if (a.cols <= 4096) return f.template stream<4, 128, 5>();
      if (a.cols <= 8192) return f.template stream<4, 256, 3>();
      return f.template stream<4, 512, 1>();
    }
  } else {
    if (vec) return by_cols_forward<V>(a.cols, f);
  }
  return by_cols_forward<1>(a.cols, f);
}

template <typename T, bool RES>
silcu_status backward(const LnArgs &a, cudaStream_t s, uint32_t *grid) {
  constexpr int V = 16 / sizeof(T);
  if (a.cols > kMaxRegCols) {
    *grid = long_grid(a.rows);
    ln_backward_cols<T><<<dim3((a.cols + 255) / 256, *grid), 256, 0, s>>>(a);
    ln_backward_long<T, RES><<<uint32_t(a.rows), 512, 0, s>>>(a);
    return check_launch("layer_norm_backward", 2);
  }
  Backward<T, RES> f{a, s, grid};
  if (a.cols % V == 0 && aligned16(a.in) && aligned16(a.dout) && aligned16(a.out) && aligned16(a.gamma) &&
      aligned16(a.part) && (!RES || aligned16(a.dres)))
    return by_cols_backward<V>(a.cols, f);
  return by_cols_backward<1>(a.cols, f);
}

silcu_status check_extent(const char *what, size_t rows, size_t cols, int dtype) {
  if (!dtype_known(dtype)) return fail(SILCU_INVALID_ARGUMENT, "%s: unknown dtype %d", what, dtype);
  if (cols == 0) return fail(SILCU_INVALID_ARGUMENT, "%s: no columns", what);
  if (rows > 0x7FFFFFFFull || cols > (1u << 24)) return fail(SILCU_UNSUPPORTED, "%s: extent too large", what);
  return SILCU_OK;
}

// Row pointers and float pointers lie on their elements' boundaries (null ones pass).
silcu_status check_aligned(const char *what, int dtype, std::initializer_list<const void *> rows,
                           std::initializer_list<const void *> floats) {
  const uintptr_t mask = dtype_bytes(dtype) - 1;
  for (const void *p : rows)
    if (reinterpret_cast<uintptr_t>(p) & mask) return fail(SILCU_INVALID_ARGUMENT, "%s: misaligned pointer", what);
  for (const void *p : floats)
    if (reinterpret_cast<uintptr_t>(p) & 3) return fail(SILCU_INVALID_ARGUMENT, "%s: misaligned pointer", what);
  return SILCU_OK;
}

}  // namespace
}  // namespace silcu

extern "C" {

silcu_status silcu_layer_norm_forward(const void *in, void *out, float *mean, float *rstd, const float *gamma,
                                      const float *beta, size_t rows, size_t cols, float eps, int dtype,
                                      silcu_stream stream) {
  using namespace silcu;
  if (rows == 0) return SILCU_OK;
  silcu_status st = check_extent("layer_norm_forward", rows, cols, dtype);
  if (st != SILCU_OK) return st;
  if (!in || !out || !gamma || !beta) return fail(SILCU_INVALID_ARGUMENT, "layer_norm_forward: null pointer");
  st = check_aligned("layer_norm_forward", dtype, {in, out}, {mean, rstd, gamma, beta});
  if (st != SILCU_OK) return st;
  const int64_t bytes = int64_t(rows * cols * dtype_bytes(dtype)), row4 = int64_t(4 * rows), col4 = int64_t(4 * cols);
  const Span outs[] = {flat(out, bytes), flat(mean, row4), flat(rstd, row4)};
  const Span ins[] = {flat(gamma, col4), flat(beta, col4), flat(out == in ? nullptr : in, bytes)};
  if (outputs_overlap(outs, 3, ins, 3))
    return fail(SILCU_INVALID_ARGUMENT, "layer_norm_forward: overlapping operands");
  LnArgs a = {};
  a.in = in;
  a.out = out;
  a.mean_out = mean;
  a.rstd_out = rstd;
  a.gamma = gamma;
  a.beta = beta;
  a.rows = rows;
  a.cols = uint32_t(cols);
  a.eps = eps;
  return dtype == SILCU_BF16 ? forward<__nv_bfloat16>(a, as_stream(stream)) : forward<float>(a, as_stream(stream));
}

size_t silcu_layer_norm_backward_workspace_bytes(size_t rows, size_t cols, int dtype) {
  using namespace silcu;
  if (rows == 0 || cols == 0 || rows > 0x7FFFFFFFull || cols > (1u << 24)) return 0;
  const uint32_t c = uint32_t(cols);
  uint32_t grid;
  if (c > kMaxRegCols) {
    grid = long_grid(rows);
  } else {  // the larger of the vector and the element-wise variant: alignment is known at the call
    const BackwardGrid g{rows};
    const uint32_t v = dtype == SILCU_BF16 ? by_cols_backward<8>(c, g) : by_cols_backward<4>(c, g);
    const uint32_t e = by_cols_backward<1>(c, g);
    grid = v > e ? v : e;
  }
  return size_t(grid) * 2 * cols * sizeof(float);
}

silcu_status silcu_layer_norm_backward(const void *dout, const void *in, const float *mean, const float *rstd,
                                       const float *gamma, const void *dresidual, void *din, float *dgamma,
                                       float *dbeta, size_t rows, size_t cols, int dtype, void *workspace,
                                       size_t workspace_bytes, silcu_stream stream) {
  using namespace silcu;
  silcu_status st = check_extent("layer_norm_backward", rows, cols, dtype);
  if (st != SILCU_OK) return st;
  if (!dgamma || !dbeta) return fail(SILCU_INVALID_ARGUMENT, "layer_norm_backward: null pointer");
  st = check_aligned("layer_norm_backward", dtype, {dout, in, dresidual, din}, {mean, rstd, gamma, dgamma, dbeta, workspace});
  if (st != SILCU_OK) return st;
  cudaStream_t s = as_stream(stream);
  uint32_t grid = 0;
  if (rows) {
    if (!dout || !in || !mean || !rstd || !gamma || !din)
      return fail(SILCU_INVALID_ARGUMENT, "layer_norm_backward: null pointer");
    const size_t need = silcu_layer_norm_backward_workspace_bytes(rows, cols, dtype);
    if (!workspace || workspace_bytes < need)
      return fail(SILCU_WORKSPACE_TOO_SMALL, "layer_norm_backward: workspace %zu < %zu", workspace_bytes, need);
    const int64_t bytes = int64_t(rows * cols * dtype_bytes(dtype)), row4 = int64_t(4 * rows), col4 = int64_t(4 * cols);
    auto other = [&](const void *p) { return flat(p == din ? nullptr : p, bytes); };  // din may be one of these
    const Span outs[] = {flat(din, bytes), flat(dgamma, col4), flat(dbeta, col4)};
    const Span ins[] = {other(dout), other(in), other(dresidual), flat(gamma, col4), flat(mean, row4), flat(rstd, row4)};
    if (outputs_overlap(outs, 3, ins, 6))
      return fail(SILCU_INVALID_ARGUMENT, "layer_norm_backward: overlapping operands");
    LnArgs a = {};
    a.in = in;
    a.dout = dout;
    a.dres = dresidual;
    a.out = din;
    a.mean = mean;
    a.rstd = rstd;
    a.gamma = gamma;
    a.part = static_cast<float *>(workspace);
    a.rows = rows;
    a.cols = uint32_t(cols);
    if (dtype == SILCU_BF16)
      st = dresidual ? backward<__nv_bfloat16, true>(a, s, &grid) : backward<__nv_bfloat16, false>(a, s, &grid);
    else
      st = dresidual ? backward<float, true>(a, s, &grid) : backward<float, false>(a, s, &grid);
    if (st != SILCU_OK) return st;
  }
  const bool few = 2 * cols <= 8 * 2 * size_t(sm_count());  // 8 columns a CTA, two CTAs an SM
  launch_after(few ? ln_finish<8> : ln_finish<32>, uint32_t((2 * cols + (few ? 7 : 31)) / (few ? 8 : 32)), 1024, 0, s,
               static_cast<const float *>(workspace), grid, uint32_t(cols), dgamma, dbeta);
  return check_launch("layer_norm_backward finish");
}

}  // extern "C"
