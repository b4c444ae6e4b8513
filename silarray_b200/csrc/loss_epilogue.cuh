// What the vocabulary projections of the cross entropy do with their scores
// in registers: a thread holds up to 128 neighbouring scores of one row.
//
//   forward   maximum m and l = sum exp(s - m) of the row over the thread's
//             columns (a "part"), and the target's score;
//   backward  ds = g (exp(s - lse) - [column = target]).
#pragma once

#include "common.cuh"

namespace silcu {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

struct LossArgs {
  const int32_t *targets;  // [rows]; outside [0, V) = the row is left out
  int32_t v0, V;           // vocabulary index of this launch's column 0; vocabulary size
  float2 *part;            // forward: [parts][rows] (m, l)
  float *target_score;     // forward: [rows], written for rows that count
  const float *lse;        // backward: [rows]
  const float *scale;      // backward: [rows] gradient of each row's loss, or null = 1
};

// Folds 32 scores, of which the first `valid` exist, into (m, l).  The terms
// are 2^(s log2 e - m log2 e): one multiply-add and one ex2 each.  A row of
// -inf alone keeps l = 0; NaN and +inf make l NaN.
__device__ __forceinline__ void softmax_fold(const float (&v)[32], int valid, float &m, float &l) {
  float mx = m;
#pragma unroll
  for (int i = 0; i < 32; i++)
    if (i < valid) mx = fmaxf(mx, v[i]);
  const float neg = mx == -INFINITY ? 0.f : -mx * kLog2e;
  l *= ex2(fmaf(m, kLog2e, neg));  // m = -inf: 0
  float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 32; i++)
    if (i < valid) a[i & 3] += ex2(fmaf(v[i], kLog2e, neg));
  l += (a[0] + a[1]) + (a[2] + a[3]);
  m = mx;
}

// The scores' gradients in place of the scores.  `at` = the target's column
// relative to the first of them, `counts` = the row is not left out (a row that
// is gets exact zeros, whatever its scores are).
__device__ __forceinline__ void score_gradient(float (&v)[32], float lse_log2e, float g, int at, bool counts) {
#pragma unroll
  for (int i = 0; i < 32; i++) {
    float p = ex2(fmaf(v[i], kLog2e, -lse_log2e));
    if (i == at) p -= 1.0f;
    v[i] = counts ? g * p : 0.f;
  }
}

}  // namespace silcu
