// Shared helpers for the sm_100a kernels behind include/silcu.h.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/silcu.h"

namespace silcu {

// 148 SMs on B200; the grid helpers query the real count once per device.
int sm_count();

// Records a message for silcu_last_error() and returns the status.
silcu_status fail(silcu_status st, const char *fmt, ...);

// Device address of the error word that bounded waits set (per device).
int *device_error_ptr();

// Counts `launches` kernel launches and maps cudaGetLastError() into a status.
silcu_status check_launch(const char *what, int launches = 1);

inline cudaStream_t as_stream(silcu_stream s) {
  return reinterpret_cast<cudaStream_t>(s);
}

inline bool aligned16(const void *p) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// Launches a kernel that may start before the one ahead of it in the stream
// has ended (programmatic dependent launch): its start-up overlaps the other's
// tail.  It calls wait_for_previous() before it reads or writes anything that
// others touch; the one ahead calls let_next_start() early on.
// Such a kernel's life overlaps the writes of its predecessors, so nothing it reads is
// constant for that life: no read-only loads, and no const parameters declared free of
// aliases, which let the compiler choose such loads or move them above the wait.
template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

// ---------------------------------------------------------------- device side
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// IEEE round-to-nearest arithmetic without contraction: the reference CPU
// path rounds after every operation, so fused kernels use these to keep the
// same rounding sequence (nvcc would otherwise fuse a*b+c into one FMA).
__device__ __forceinline__ float add_rn(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ float sub_rn(float a, float b) { return __fsub_rn(a, b); }
__device__ __forceinline__ float mul_rn(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float div_rn(float a, float b) { return __fdiv_rn(a, b); }

// sigmoid in the reference's order (include/cpu.h:290-297): negate, exp,
// add one, reciprocal.  expf is CUDA's accurate single-precision exp.
__device__ __forceinline__ float sigmoid_ref(float x) {
  float t = expf(-x);
  t = __fadd_rn(t, 1.0f);
  return __frcp_rn(t);
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float warp_min(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

}  // namespace silcu
