// The 2-norm over a list of tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors of x^2),  out = x * min(1, max_norm / (norm + eps))
//
// Bound by HBM: the norm reads every element once; clipping reads it again
// and writes it.  The list travels in the kernel's parameters (up to CAP
// tensors a launch), so nothing is staged in device memory.  The elements of
// all tensors of a launch count as one sequence, cut into equal spans, one per
// warp: large tensors spread over the whole grid and small ones share a warp.
// The clipping pass walks its spans from the last to the first, as the norm
// pass's most recent reads are what the L2 still holds.
//
// Squares add in fp32 over four 16-byte vectors of a thread, and those sums in fp64.
// Vectors whose fp32 sum may have overflowed or lost denormal squares add
// again in fp64.  Every CTA writes one fp64 partial; all of them add in CTA
// order, so results repeat bit for bit.
#include <math.h>

#include "elem.cuh"

namespace silcu {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCtasPerSm = 5;  // what the registers hold; a sixth would run as a tail (700 MB: 120 us, 105 with 5)
constexpr uint64_t kMinSpan = 256;  // elements; a launch of few elements uses few warps

template <int CAP>
struct ListArgs {
  const void *in[CAP];
  void *out[CAP];
  uint64_t start[CAP + 1];  // of each tensor in the sequence; start[count] = all elements
  unsigned char dtype[CAP];
  int count;
  uint64_t span;
  double *part;       // this launch's partials
  const double *all;  // every launch's (clipping)
  int nparts;
  float *norm;
  float max_norm, eps;
};

// Whether a fp32 sum of squares stands: nothing overflowed, and no square
// small enough to have vanished matters in it.
__device__ __forceinline__ bool in_range(float s) { return s > 1e-28f && s < 1e37f; }

template <int N>
__device__ __forceinline__ float squares32(const float (&f)[N]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < N; k++) s = fmaf(f[k], f[k], s);
  return s;
}
template <int N>
__device__ __forceinline__ double squares64(const float (&f)[N]) {
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < N; k++) d = fma(double(f[k]), double(f[k]), d);
  return d;
}

// A warp's part of one tensor: f.vec4 / f.vec for whole 16-byte vectors from a
// 128-byte line on, f.one for the elements before and after them.  `head` =
// elements before the first line, or < 0 where the operands have no common one.
template <typename T, typename F>
__device__ __forceinline__ void walk(uint64_t n, int head, F &&f) {
  constexpr int V = 16 / sizeof(T);
  const uint32_t lane = threadIdx.x & 31;
  if (head < 0) {
    for (uint64_t i = lane; i < n; i += 32) f.one(i);
    return;
  }
  if (uint64_t(head) > n) head = int(n);
  for (int i = lane; i < head; i += 32) f.one(i);
  const uint64_t nv = (n - head) / V;
  uint64_t i = lane;
  for (; i + 96 < nv; i += 128) f.vec4(head + i * V);
  for (; i < nv; i += 32) f.vec(head + i * V);
  const uint64_t done = head + nv * V;
  if (done + lane < n) f.one(done + lane);
}

// Elements of T from p to the next 128-byte line.
template <typename T>
__device__ __forceinline__ int head_of(const void *p) {
  return int(((128 - (reinterpret_cast<uintptr_t>(p) & 127)) & 127) / sizeof(T));
}

template <typename T>
struct SumSquares {
  static constexpr int V = 16 / sizeof(T);
  const T *p;
  double acc;
  __device__ __forceinline__ void one(uint64_t i) {
    float f[1];
    unpack(raw_ld<1>(i), f);
    acc += squares64(f);
  }
  __device__ __forceinline__ void vec(uint64_t i) {
    float f[V];
    unpack(raw_ld<V>(i), f);
    const float s = squares32(f);
    acc += in_range(s) ? double(s) : squares64(f);
  }
  __device__ __forceinline__ void vec4(uint64_t i) {
    Raw<T, V> r[4];
#pragma unroll
    for (int u = 0; u < 4; u++) r[u] = raw_ld<V>(i + u * 32 * V);
    float s[4];
    bool all = true;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      float f[V];
      unpack(r[u], f);
      s[u] = squares32(f);
      all = all && in_range(s[u]);
    }
    if (all) {
      acc += double((s[0] + s[1]) + (s[2] + s[3]));
    } else {
#pragma unroll
      for (int u = 0; u < 4; u++) {
        float f[V];
        unpack(r[u], f);
        acc += squares64(f);
      }
    }
  }
  // plain loads: the clipping pass finds the newest of them in the L2
  template <int N>
  __device__ __forceinline__ Raw<T, N> raw_ld(uint64_t i) {
    Raw<T, N> r;
    r.r = *reinterpret_cast<const decltype(r.r) *>(p + i);
    return r;
  }
};

template <typename T>
struct Scale {
  static constexpr int V = 16 / sizeof(T);
  const T *p;
  T *o;
  float c;
  template <int N>
  __device__ __forceinline__ void scale(Raw<T, N> r, uint64_t i) {
    float f[N];
    unpack(r, f);
#pragma unroll
    for (int k = 0; k < N; k++) f[k] *= c;
    pack(f, r);
    raw_store<T, N>(o + i, r);
  }
  __device__ __forceinline__ void one(uint64_t i) { scale<1>(raw_load<T, 1>(p + i), i); }
  __device__ __forceinline__ void vec(uint64_t i) { scale<V>(raw_load<T, V>(p + i), i); }
  __device__ __forceinline__ void vec4(uint64_t i) {
    Raw<T, V> r[4];
#pragma unroll
    for (int u = 0; u < 4; u++) r[u] = raw_load<T, V>(p + i + u * 32 * V);
#pragma unroll
    for (int u = 0; u < 4; u++) scale<V>(r[u], i + u * 32 * V);
  }
};

// Calls f(tensor, first element, elements) for the tensors of a span.
template <int CAP, typename F>
__device__ __forceinline__ void for_span(const ListArgs<CAP> &a, uint64_t worker, F &&f) {
  uint64_t at = worker * a.span;
  const uint64_t total = a.start[a.count];
  if (at >= total) return;
  const uint64_t end = at + a.span < total ? at + a.span : total;
  int lo = 0, hi = a.count;  // the last tensor that starts at or before `at`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.start[mid] <= at) lo = mid;
    else hi = mid;
  }
  for (int t = lo; at < end; t++) {
    const uint64_t stop = a.start[t + 1] < end ? a.start[t + 1] : end;
    if (stop > at) f(t, at - a.start[t], stop - at);
    at = stop;
  }
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) sum_squares(const __grid_constant__ ListArgs<CAP> a) {
  __shared__ double sm[kWarps];
  let_next_start();
  wait_for_previous();
  double acc = 0.0;
  for_span(a, uint64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5), [&](int t, uint64_t first, uint64_t n) {
    if (a.dtype[t] == SILCU_BF16) {
      SumSquares<__nv_bfloat16> f{static_cast<const __nv_bfloat16 *>(a.in[t]) + first, acc};
      walk<__nv_bfloat16>(n, head_of<__nv_bfloat16>(f.p), f);
      acc = f.acc;
    } else {
      SumSquares<float> f{static_cast<const float *>(a.in[t]) + first, acc};
      walk<float>(n, head_of<float>(f.p), f);
      acc = f.acc;
    }
  });
  acc = warp_sum(acc);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = sm[0];
    for (int i = 1; i < kWarps; i++) s += sm[i];
    a.part[blockIdx.x] = s;
  }
}

// All partials in a fixed order; every thread gets the norm.
__device__ __forceinline__ double total_norm(const double *part, int nparts) {
  __shared__ double sm[kWarps];
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += kThreads) s += part[i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = s;
  __syncthreads();
  s = sm[0];
#pragma unroll
  for (int i = 1; i < kWarps; i++) s += sm[i];
  return sqrt(s);
}

__global__ void __launch_bounds__(kThreads) norm_finish(const double *part, int nparts, float *norm) {
  let_next_start();
  wait_for_previous();
  const double n = total_norm(part, nparts);
  if (threadIdx.x == 0) *norm = float(n);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads) clip_scale(const __grid_constant__ ListArgs<CAP> a) {
  let_next_start();
  wait_for_previous();
  const double norm = total_norm(a.all, a.nparts);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm) *a.norm = float(norm);
  const double below = norm + double(a.eps);
  double c = below > 0.0 || !(below == below) ? double(a.max_norm) / below : 1.0;  // all zeros stay zeros
  if (c > 1.0) c = 1.0;  // a NaN stays one
  const uint64_t worker = uint64_t(gridDim.x - 1 - blockIdx.x) * kWarps + (threadIdx.x >> 5);
  for_span(a, worker, [&](int t, uint64_t first, uint64_t n) {
    if (c == 1.0 && a.in[t] == a.out[t]) return;  // nothing to change in place
    if (a.dtype[t] == SILCU_BF16) {
      using T = __nv_bfloat16;
      Scale<T> f{static_cast<const T *>(a.in[t]) + first, static_cast<T *>(a.out[t]) + first, float(c)};
      walk<T>(n, head_of<T>(f.p) == head_of<T>(f.o) ? head_of<T>(f.p) : -1, f);
    } else {
      using T = float;
      Scale<T> f{static_cast<const T *>(a.in[t]) + first, static_cast<T *>(a.out[t]) + first, float(c)};
      walk<T>(n, head_of<T>(f.p) == head_of<T>(f.o) ? head_of<T>(f.p) : -1, f);
    }
  });
}

// --------------------------------------------------------------------- host
constexpr int kSmallCap = 64, kCap = 1024;  // 1.6 / 25.6 KB of parameters

uint64_t span_of(uint64_t total) {
  const uint64_t workers = uint64_t(sm_count()) * kCtasPerSm * kWarps;
  uint64_t span = (total + workers - 1) / workers;
  span = (span + 127) / 128 * 128;
  return span < kMinSpan ? kMinSpan : span;
}
uint32_t grid_of(uint64_t total) {
  const uint64_t w = (total + span_of(total) - 1) / span_of(total);
  return uint32_t((w + kWarps - 1) / kWarps);
}

struct Piece {
  size_t first, count;
  uint64_t total;
  uint32_t grid, part0;
};

// The launches of a list: kCap tensors each.
template <typename F>
uint32_t for_pieces(const silcu_tensor *t, size_t count, F &&f) {
  uint32_t parts = 0;
  for (size_t first = 0; first < count; first += kCap) {
    Piece p = {first, count - first < size_t(kCap) ? count - first : size_t(kCap), 0, 0, parts};
    for (size_t i = 0; i < p.count; i++) p.total += t[first + i].n;
    p.grid = p.total ? grid_of(p.total) : 0;
    parts += p.grid;
    if (p.grid) f(p);
  }
  return parts;
}

template <int CAP>
void fill(ListArgs<CAP> &a, const silcu_tensor *t, void *const *outs, const Piece &p) {
  uint64_t at = 0;
  for (size_t i = 0; i < p.count; i++) {
    const silcu_tensor &x = t[p.first + i];
    a.in[i] = x.data;
    a.out[i] = outs ? outs[p.first + i] : x.data;
    a.dtype[i] = static_cast<unsigned char>(x.dtype);
    a.start[i] = at;
    at += x.n;
  }
  a.start[p.count] = at;
  a.count = int(p.count);
  a.span = span_of(at);
}

silcu_status check_list(const char *what, const silcu_tensor *t, void *const *outs, size_t count) {
  if (!t && count) return fail(SILCU_INVALID_ARGUMENT, "%s: null list", what);
  for (size_t i = 0; i < count; i++) {
    const uintptr_t mask = dtype_bytes(t[i].dtype) - 1;
    if (!dtype_known(t[i].dtype))
      return fail(SILCU_INVALID_ARGUMENT, "%s: tensor %zu has unknown dtype %d", what, i, t[i].dtype);
    if (t[i].n >> 48) return fail(SILCU_UNSUPPORTED, "%s: tensor %zu is too large", what, i);
    if (t[i].n && (!t[i].data || (reinterpret_cast<uintptr_t>(t[i].data) & mask)))
      return fail(SILCU_INVALID_ARGUMENT, "%s: tensor %zu has a null or misaligned pointer", what, i);
    if (outs && t[i].n && (!outs[i] || (reinterpret_cast<uintptr_t>(outs[i]) & mask)))
      return fail(SILCU_INVALID_ARGUMENT, "%s: output %zu has a null or misaligned pointer", what, i);
  }
  return SILCU_OK;
}

silcu_status check_workspace(const char *what, const silcu_tensor *t, size_t count, void *ws, size_t bytes) {
  const size_t need = silcu_grad_norm_workspace_bytes(t, count);
  if (need && (!ws || bytes < need))
    return fail(SILCU_WORKSPACE_TOO_SMALL, "%s: workspace %zu < %zu", what, bytes, need);
  if (reinterpret_cast<uintptr_t>(ws) & 7) return fail(SILCU_INVALID_ARGUMENT, "%s: misaligned workspace", what);
  return SILCU_OK;
}

template <int CAP>
void launch_sum(const silcu_tensor *t, const Piece &p, double *part, cudaStream_t s) {
  ListArgs<CAP> a = {};
  fill(a, t, nullptr, p);
  a.part = part + p.part0;
  launch_after(sum_squares<CAP>, p.grid, kThreads, 0, s, a);
}

template <int CAP>
void launch_scale(const silcu_tensor *t, void *const *outs, const Piece &p, ListArgs<CAP> a, cudaStream_t s) {
  fill(a, t, outs, p);
  launch_after(clip_scale<CAP>, p.grid, kThreads, 0, s, a);
}

// The partials of the whole list; their number.
uint32_t sum_list(const silcu_tensor *t, size_t count, double *part, cudaStream_t s) {
  return for_pieces(t, count, [&](const Piece &p) {
    if (p.count <= size_t(kSmallCap)) launch_sum<kSmallCap>(t, p, part, s);
    else launch_sum<kCap>(t, p, part, s);
  });
}

int pieces(const silcu_tensor *t, size_t count) {
  int n = 0;
  for_pieces(t, count, [&](const Piece &) { n++; });
  return n;
}

}  // namespace
}  // namespace silcu

extern "C" {

size_t silcu_grad_norm_workspace_bytes(const silcu_tensor *tensors, size_t count) {
  using namespace silcu;
  if (!tensors) return 0;
  return size_t(for_pieces(tensors, count, [](const Piece &) {})) * sizeof(double);
}

silcu_status silcu_grad_norm(const silcu_tensor *tensors, size_t count, float *norm, void *workspace,
                             size_t workspace_bytes, silcu_stream stream) {
  using namespace silcu;
  silcu_status st = check_list("grad_norm", tensors, nullptr, count);
  if (st != SILCU_OK) return st;
  if (!norm || (reinterpret_cast<uintptr_t>(norm) & 3))
    return fail(SILCU_INVALID_ARGUMENT, "grad_norm: null or misaligned pointer");
  st = check_workspace("grad_norm", tensors, count, workspace, workspace_bytes);
  if (st != SILCU_OK) return st;
  cudaStream_t s = as_stream(stream);
  double *part = static_cast<double *>(workspace);
  const uint32_t parts = sum_list(tensors, count, part, s);
  launch_after(norm_finish, 1, kThreads, 0, s, part, int(parts), norm);
  return check_launch("grad_norm", pieces(tensors, count) + 1);
}

silcu_status silcu_clip_grad_norm(const silcu_tensor *tensors, void *const *outputs, size_t count, float max_norm,
                                  float eps, float *norm, void *workspace, size_t workspace_bytes,
                                  silcu_stream stream) {
  using namespace silcu;
  silcu_status st = check_list("clip_grad_norm", tensors, outputs, count);
  if (st != SILCU_OK) return st;
  if (!norm || (reinterpret_cast<uintptr_t>(norm) & 3))
    return fail(SILCU_INVALID_ARGUMENT, "clip_grad_norm: null or misaligned pointer");
  if (!(max_norm >= 0.f) || !(eps >= 0.f))
    return fail(SILCU_INVALID_ARGUMENT, "clip_grad_norm: max_norm and eps must not be negative");
  st = check_workspace("clip_grad_norm", tensors, count, workspace, workspace_bytes);
  if (st != SILCU_OK) return st;
  cudaStream_t s = as_stream(stream);
  double *part = static_cast<double *>(workspace);
  const uint32_t parts = sum_list(tensors, count, part, s);
  if (parts == 0) {
    norm_finish<<<1, kThreads, 0, s>>>(part, 0, norm);
    return check_launch("clip_grad_norm");
  }
  bool first = true;
  for_pieces(tensors, count, [&](const Piece &p) {
    auto go = [&](auto a) {
      a.all = part;
      a.nparts = int(parts);
      a.norm = first ? norm : nullptr;
      a.max_norm = max_norm;
      a.eps = eps;
      first = false;
      launch_scale(tensors, outputs, p, a, s);
    };
    if (p.count <= size_t(kSmallCap)) go(ListArgs<kSmallCap>{});
    else go(ListArgs<kCap>{});
  });
  return check_launch("clip_grad_norm", 2 * pieces(tensors, count));
}

}  // extern "C"
