// Element types of the training operators (silcu_dtype): 16-byte vectors of
// fp32 or bf16 elements, or single ones, read and written as fp32 values.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>
#include <string.h>

#include "common.cuh"

namespace silcu {

inline size_t dtype_bytes(int dtype) { return dtype == SILCU_BF16 ? 2 : 4; }
inline bool dtype_known(int dtype) { return dtype == SILCU_F32 || dtype == SILCU_BF16; }

// Rows in memory: `width` bytes each, `stride` bytes apart.
struct Span {
  const void *p;
  int64_t rows, width, stride;
};
// Whether two of them share a byte.  Rows of one stride that lie side by side
// (column ranges of one matrix) do not; other interleaved rows count as sharing.
inline bool overlap(const Span &a, const Span &b) {
  if (!a.p || !b.p || a.rows * a.width == 0 || b.rows * b.width == 0) return false;
  const int64_t a0 = int64_t(reinterpret_cast<uintptr_t>(a.p)), b0 = int64_t(reinterpret_cast<uintptr_t>(b.p));
  if (a0 + (a.rows - 1) * a.stride + a.width <= b0 || b0 + (b.rows - 1) * b.stride + b.width <= a0) return false;
  const int64_t stride = a.rows > 1 ? a.stride : b.stride;
  if (stride <= 0 || (a.rows > 1 && b.rows > 1 && a.stride != b.stride)) return true;
  const int64_t d = ((b0 - a0) % stride + stride) % stride;  // b's column in a's rows
  return d < a.width || d + b.width > stride;
}
inline Span flat(const void *p, int64_t bytes) { return Span{p, 1, bytes, bytes}; }
// Whether an output shares memory with an input or another output.
inline bool outputs_overlap(const Span *outs, int nouts, const Span *ins, int nins) {
  for (int i = 0; i < nouts; i++) {
    for (int j = 0; j < nins; j++)
      if (overlap(outs[i], ins[j])) return true;
    for (int j = 0; j < i; j++)
      if (overlap(outs[i], outs[j])) return true;
  }
  return false;
}

// VEC elements as they lie in memory: one 16-byte vector, or one element.
template <typename T, int VEC> struct Raw;
template <> struct Raw<float, 4> { float4 r; };
template <> struct Raw<float, 1> { float r; };
template <> struct Raw<__nv_bfloat16, 8> { uint4 r; };
template <> struct Raw<__nv_bfloat16, 1> { unsigned short r; };

// Streaming loads and stores (the data is not read again by this kernel).
// The loads are volatile, so they stay behind wait_for_previous(), and not of the read-only
// path: an earlier kernel that is still running may write what they read (see
// launch_after), and outputs may be one of the inputs.
__device__ __forceinline__ float load_streaming(const float *p) {
  float v;
  asm volatile("ld.global.cs.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned short load_streaming(const unsigned short *p) {
  unsigned short v;
  asm volatile("ld.global.cs.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float2 load_streaming(const float2 *p) {
  float2 v;
  asm volatile("ld.global.cs.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_streaming(const float4 *p) {
  float4 v;
  asm volatile("ld.global.cs.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ uint4 load_streaming(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
// The same from the L2: what other CTAs of this kernel have written.
__device__ __forceinline__ float load_l2(const float *p) {
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> raw_load(const T *p) {
  Raw<T, VEC> v;
  v.r = load_streaming(reinterpret_cast<const decltype(v.r) *>(p));
  return v;
}
template <typename T, int VEC>
__device__ __forceinline__ void raw_store(T *p, const Raw<T, VEC> &v) {
  __stcs(reinterpret_cast<decltype(v.r) *>(p), v.r);
}
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> raw_zero() {
  Raw<T, VEC> v;
  memset(&v, 0, sizeof(v));
  return v;
}

__device__ __forceinline__ void unpack(const Raw<float, 4> &v, float (&f)[4]) {
  f[0] = v.r.x, f[1] = v.r.y, f[2] = v.r.z, f[3] = v.r.w;
}
__device__ __forceinline__ void unpack(const Raw<float, 1> &v, float (&f)[1]) { f[0] = v.r; }
__device__ __forceinline__ void unpack2(uint32_t u, float &a, float &b) {
  a = __uint_as_float(u << 16);
  b = __uint_as_float(u & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16, 8> &v, float (&f)[8]) {
  unpack2(v.r.x, f[0], f[1]);
  unpack2(v.r.y, f[2], f[3]);
  unpack2(v.r.z, f[4], f[5]);
  unpack2(v.r.w, f[6], f[7]);
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16, 1> &v, float (&f)[1]) {
  f[0] = __uint_as_float(uint32_t(v.r) << 16);
}

// VEC fp32 parameters (or shared-memory sums), as 16-byte vectors for VEC >= 4.
template <int VEC>
__device__ __forceinline__ void load_f32(const float *p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = *p;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p + k);
      f[k] = v.x, f[k + 1] = v.y, f[k + 2] = v.z, f[k + 3] = v.w;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void store_f32(float *p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = f[0];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4 *>(p + k) = make_float4(f[k], f[k + 1], f[k + 2], f[k + 3]);
  }
}

// Two values rounded to nearest even bf16, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void pack(const float (&f)[4], Raw<float, 4> &v) {
  v.r = make_float4(f[0], f[1], f[2], f[3]);
}
__device__ __forceinline__ void pack(const float (&f)[1], Raw<float, 1> &v) { v.r = f[0]; }
__device__ __forceinline__ void pack(const float (&f)[8], Raw<__nv_bfloat16, 8> &v) {
  v.r = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ void pack(const float (&f)[1], Raw<__nv_bfloat16, 1> &v) {
  v.r = __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
}

}  // namespace silcu
