// layer_norm for training: the forward pass that keeps each row's statistics,
// and the backward pass with the reduction of gamma's and beta's gradients.
//
//   mu = avg(x), r = 1 / sqrt(avg((x - mu)^2) + eps), xh = (x - mu) r, y = xh gamma + beta
//   a = dy gamma,  dx = r (a - avg(a) - xh avg(a xh)) (+ residual gradient)
//   dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// Both are bound by HBM: the forward reads x and writes y, the backward reads
// dy, x (and the residual gradient) and writes dx, each once.  A row lives in
// registers: a warp per row up to 1024 columns, a CTA per row up to 16384, a
// re-reading loop beyond.  Elements move as 16-byte vectors where the columns
// and pointers allow (VEC = 4 fp32 / 8 bf16), else one by one (VEC = 1).
//
// Backward: a persistent grid; each group of threads walks its rows and adds
// its columns' dgamma / dbeta terms as it goes (in registers for a warp per
// row, in the thread's own shared-memory slots for a CTA per row), writes one
// partial row per CTA, and ln_finish adds the partials in CTA order.  All sums
// are fp32 in an order fixed by the shape and the SM count.
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
  const float rstd = 1.0f / sqrtf(group_sum<NT>(ss, sm[1]) * inv_n + a.eps);
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
  const float rstd = 1.0f / sqrtf(group_sum<512>(ss, sm[1]) * inv_n + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean_out) a.mean_out[row] = mu;
    if (a.rstd_out) a.rstd_out[row] = rstd;
  }
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) {
    float v[1] = {fmaf((at(c) - mu) * rstd, __ldg(a.gamma + c), __ldg(a.beta + c))};
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
    mean = __ldg(a.mean + row);
    rstd = __ldg(a.rstd + row);
  }
};

template <typename T, int VEC, int VPT, int NT, int GROUPS, bool RES>
__global__ void __launch_bounds__(NT *GROUPS) ln_backward(const LnArgs a) {
  constexpr int NW = NT / 32, E = VPT * VEC;
  constexpr bool WARP = NT == 32;
  extern __shared__ __align__(16) float acc_s[];  // dgamma[cols], dbeta[cols] of this CTA
  __shared__ float2 sm[2][NW];
  const uint32_t t = threadIdx.x % NT, g = threadIdx.x / NT;
  float ag[WARP ? E : 1], ab[WARP ? E : 1];
  if (WARP) {
#pragma unroll
    for (int i = 0; i < E; i++) ag[i] = ab[i] = 0.f;
  } else {
    for (uint32_t c = threadIdx.x; c < 2 * a.cols; c += NT * GROUPS) acc_s[c] = 0.f;
    __syncthreads();
  }
  const float inv_n = 1.0f / float(a.cols);
  const uint64_t step = uint64_t(gridDim.x) * GROUPS;
  int buf = 0;
  for (uint64_t row = uint64_t(blockIdx.x) * GROUPS + g; row < a.rows; row += step) {
    LnRow<T, VEC, VPT, NT, RES> r;
    r.load(a, row, t);
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; j++) {
      const uint32_t c = (t + j * NT) * VEC;
      if (c < a.cols) {
        float x[VEC], dy[VEC], gm[VEC], sg[VEC], sb[VEC];
        unpack(r.x[j], x);
        unpack(r.dy[j], dy);
        load_f32<VEC>(a.gamma + c, gm);
        if (!WARP) {
          load_f32<VEC>(acc_s + c, sg);
          load_f32<VEC>(acc_s + a.cols + c, sb);
        }
#pragma unroll
        for (int k = 0; k < VEC; k++) {
          const float xh = (x[k] - r.mean) * r.rstd;
          const float w = dy[k] * gm[k];
          c1 += w;
          c2 = fmaf(w, xh, c2);
          if (WARP) {
            ag[j * VEC + k] = fmaf(dy[k], xh, ag[j * VEC + k]);
            ab[j * VEC + k] += dy[k];
          } else {
            sg[k] = fmaf(dy[k], xh, sg[k]);
            sb[k] += dy[k];
          }
        }
        if (!WARP) {
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
        load_f32<VEC>(a.gamma + c, gm);
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
  if (WARP) {  // the CTA's warps add their sums in warp order
#pragma unroll 1
    for (int w = 0; w < GROUPS; w++) {
      if (int(g) == w) {
#pragma unroll
        for (int j = 0; j < VPT; j++) {
          const uint32_t c = (t + j * NT) * VEC;
          if (c < a.cols) {
#pragma unroll
            for (int k = 0; k < VEC; k++) {
              const int i = j * VEC + k;
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
  float *part = a.part + uint64_t(blockIdx.x) * 2 * a.cols;
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
    g = fmaf(dy[0], (x[0] - __ldg(a.mean + row)) * __ldg(a.rstd + row), g);
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
    const float w = at(py, c) * __ldg(a.gamma + c);
    c1 += w;
    c2 = fmaf(w, (at(px, c) - mean) * rstd, c2);
  }
  c1 = group_sum<512>(c1, sm[0]) * inv_n;
  c2 = group_sum<512>(c2, sm[1]) * inv_n;
  for (uint32_t c = threadIdx.x; c < a.cols; c += 512) {
    float v[1] = {rstd * (at(py, c) * __ldg(a.gamma + c) - c1 - (at(px, c) - mean) * rstd * c2)};
    if (RES) v[0] += at(pr, c);
    Raw<T, 1> o;
    pack(v, o);
    raw_store<T, 1>(dst + c, o);
  }
}

// dgamma / dbeta: the partial rows added in CTA order, in 8 interleaved
// slices per column that then add in slice order.
__global__ void __launch_bounds__(256) ln_finish(const float *__restrict__ part, uint32_t nparts, uint32_t cols,
                                                 float *__restrict__ dgamma, float *__restrict__ dbeta) {
  __shared__ float sm[8][33];
  const uint32_t lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const uint32_t c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * cols) {
#pragma unroll 8
    for (uint32_t i = slice; i < nparts; i += 8) s += __ldcs(part + uint64_t(i) * 2 * cols + c);
  }
  sm[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < 2 * cols) {
#pragma unroll
    for (int i = 1; i < 8; i++) s += sm[i][lane];
    if (c < cols) dgamma[c] = s;
    else dbeta[c - cols] = s;
  }
}

// --------------------------------------------------------------------- host
// Calls f.run<VEC, VPT, NT, GROUPS>() for a row of `cols`: the fewest
// registers that hold it.  VEC is the vector width, 1 for unaligned rows.
template <int VEC, typename F>
silcu_status by_cols(uint32_t cols, F &&f) {
  constexpr int V = VEC == 1 ? 1 : VEC;
  if (cols <= 32 * 8) return f.template run<V, 8 / V, 32, 8>();
  if (cols <= 32 * 16) return f.template run<V, 16 / V, 32, 8>();
  if (cols <= 32 * 24) return f.template run<V, 24 / V, 32, 8>();
  if (cols <= 32 * 32) return f.template run<V, 32 / V, 32, 8>();
  if (cols <= 128 * 16) return f.template run<V, 16 / V, 128, 1>();
  if (cols <= 256 * 16) return f.template run<V, 16 / V, 256, 1>();
  if (cols <= 512 * 16) return f.template run<V, 16 / V, 512, 1>();
  return f.template run<V, 32 / V, 512, 1>();
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
};

// CTAs of the persistent backward grid: enough to fill the SMs, never more
// than the groups of rows there are.  The workspace holds one partial row pair
// for each.
constexpr int kBwdCtasPerSm = 4;
uint32_t bwd_ctas(uint64_t rows, uint32_t cols) {
  const uint64_t groups = cols <= 1024 ? (rows + 7) / 8 : rows;
  const uint64_t cap = uint64_t(sm_count()) * (cols <= kMaxRegCols ? kBwdCtasPerSm : 1);
  return uint32_t(groups < cap ? groups : cap);
}

template <typename T, bool RES>
struct Backward {
  LnArgs a;
  uint32_t grid;
  cudaStream_t s;
  template <int VEC, int VPT, int NT, int GROUPS>
  silcu_status run() {
    const uint32_t smem = 2 * a.cols * sizeof(float);
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (smem > 48 * 1024 - 1024 && dev >= 0 && dev < 64 && !configured[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(ln_backward<T, VEC, VPT, NT, GROUPS, RES>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 int(2 * kMaxRegCols * sizeof(float)));
      if (e != cudaSuccess)
        return fail(SILCU_CUDA_ERROR, "layer_norm_backward: smem attribute: %s", cudaGetErrorString(e));
      configured[dev] = true;
    }
    ln_backward<T, VEC, VPT, NT, GROUPS, RES><<<grid, NT * GROUPS, smem, s>>>(a);
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
  if (a.cols % V == 0 && aligned16(a.in) && aligned16(a.out) && aligned16(a.gamma) && aligned16(a.beta))
    return by_cols<V>(a.cols, Forward<T>{a, s});
  return by_cols<1>(a.cols, Forward<T>{a, s});
}

template <typename T, bool RES>
silcu_status backward(const LnArgs &a, uint32_t grid, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (a.cols > kMaxRegCols) {
    ln_backward_cols<T><<<dim3((a.cols + 255) / 256, grid), 256, 0, s>>>(a);
    ln_backward_long<T, RES><<<uint32_t(a.rows), 512, 0, s>>>(a);
    return check_launch("layer_norm_backward", 2);
  }
  if (a.cols % V == 0 && aligned16(a.in) && aligned16(a.dout) && aligned16(a.out) && aligned16(a.gamma) &&
      (!RES || aligned16(a.dres)))
    return by_cols<V>(a.cols, Backward<T, RES>{a, grid, s});
  return by_cols<1>(a.cols, Backward<T, RES>{a, grid, s});
}

silcu_status check_extent(const char *what, size_t rows, size_t cols, int dtype) {
  if (!dtype_known(dtype)) return fail(SILCU_INVALID_ARGUMENT, "%s: unknown dtype %d", what, dtype);
  if (cols == 0) return fail(SILCU_INVALID_ARGUMENT, "%s: no columns", what);
  if (rows > 0x7FFFFFFFull || cols > (1u << 24)) return fail(SILCU_UNSUPPORTED, "%s: extent too large", what);
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

size_t silcu_layer_norm_backward_workspace_bytes(size_t rows, size_t cols, int) {
  using namespace silcu;
  if (rows == 0 || cols == 0 || rows > 0x7FFFFFFFull || cols > (1u << 24)) return 0;
  return size_t(bwd_ctas(rows, uint32_t(cols))) * 2 * cols * sizeof(float);
}

silcu_status silcu_layer_norm_backward(const void *dout, const void *in, const float *mean, const float *rstd,
                                       const float *gamma, const void *dresidual, void *din, float *dgamma,
                                       float *dbeta, size_t rows, size_t cols, int dtype, void *workspace,
                                       size_t workspace_bytes, silcu_stream stream) {
  using namespace silcu;
  silcu_status st = check_extent("layer_norm_backward", rows, cols, dtype);
  if (st != SILCU_OK) return st;
  if (!dgamma || !dbeta) return fail(SILCU_INVALID_ARGUMENT, "layer_norm_backward: null pointer");
  cudaStream_t s = as_stream(stream);
  const uint32_t grid = rows ? bwd_ctas(rows, uint32_t(cols)) : 0;
  if (rows) {
    if (!dout || !in || !mean || !rstd || !gamma || !din)
      return fail(SILCU_INVALID_ARGUMENT, "layer_norm_backward: null pointer");
    const size_t need = silcu_layer_norm_backward_workspace_bytes(rows, cols, dtype);
    if (!workspace || workspace_bytes < need)
      return fail(SILCU_WORKSPACE_TOO_SMALL, "layer_norm_backward: workspace %zu < %zu", workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 3)
      return fail(SILCU_INVALID_ARGUMENT, "layer_norm_backward: misaligned workspace");
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
      st = dresidual ? backward<__nv_bfloat16, true>(a, grid, s) : backward<__nv_bfloat16, false>(a, grid, s);
    else
      st = dresidual ? backward<float, true>(a, grid, s) : backward<float, false>(a, grid, s);
    if (st != SILCU_OK) return st;
  }
  ln_finish<<<uint32_t((2 * cols + 31) / 32), 256, 0, s>>>(static_cast<const float *>(workspace), grid,
                                                           uint32_t(cols), dgamma, dbeta);
  return check_launch("layer_norm_backward finish");
}

}  // extern "C"
