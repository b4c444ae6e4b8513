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
  unsigned *done;          // forward: set to 0 for what follows
  const float *lse;        // backward: [rows]
  const float *scale;      // backward: gradient of the rows' loss, one or (per_row) [rows], or null = 1
  int per_row;
};

// (m, l) of 128 scores, of which the first `valid` exist.  The terms are
// 2^(s log2 e - m log2 e): one multiply-add and one ex2 each, in chains short
// enough that two warps per scheduler keep up.  A row of -inf alone has l = 0;
// NaN and +inf make l NaN.
__device__ __forceinline__ void softmax_part(const float (&v)[128], int valid, float &m, float &l) {
  float mx[8], a[8];
#pragma unroll
  for (int i = 0; i < 8; i++) mx[i] = -INFINITY, a[i] = 0.f;
#pragma unroll
  for (int i = 0; i < 128; i++)
    if (i < valid) mx[i & 7] = fmaxf(mx[i & 7], v[i]);
  m = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
  const float neg = m == -INFINITY ? 0.f : -m * kLog2e;
#pragma unroll
  for (int i = 0; i < 128; i++)
    if (i < valid) a[i & 7] += ex2(fmaf(v[i], kLog2e, neg));
  l = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
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
