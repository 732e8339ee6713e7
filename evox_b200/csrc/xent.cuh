// Row-wise softmax statistics shared by the cross-entropy epilogues: a row is cut into slices of 128 columns, each
// reduced to (maximum, sum of exp(z - maximum)) in 32 bits; xent_finish joins them.
#pragma once
#include <math.h>

#include "common.cuh"

namespace evox {

constexpr int kSlice = 128;  // columns that one (maximum, sum) covers
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(z - m) of one row's values. The difference is taken before the factor log2(e), not z log2(e) - m log2(e) in one
// instruction: the maximum's own term is then exactly 1, so that no loss comes out below 0, and a maximum near the end
// of the range (a mask of the type's lowest value that leaves nothing else) does not overflow.
__device__ __forceinline__ void exp_from(float (&z)[32], float m) {
  m = m == -INFINITY ? 0.f : m;  // nothing but -inf: every exponential is 0
#pragma unroll
  for (int j = 0; j < 32; ++j) z[j] = exp2_approx((z[j] - m) * kLog2e);
}
// Weight of a sum taken at maximum `m` when the maximum becomes `top` >= m.
__device__ __forceinline__ float rescale_to(float m, float top) { return exp2_approx((m - (top == -INFINITY ? 0.f : top)) * kLog2e); }

// Takes 32 more values of a row into its running (maximum, sum); `z` is overwritten.
__device__ __forceinline__ void take_into(float (&z)[32], float& m, float& sum) {
  float top = m;
#pragma unroll
  for (int j = 0; j < 32; ++j) top = fmaxf(top, z[j]);
  exp_from(z, top);
  float part = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) part += z[j];
  sum = fmaf(sum, rescale_to(m, top), part);
  m = top;
}

// Where a row's label is column `label - c` of the 32 values at hand, stores that value.
__device__ __forceinline__ void keep_label(const float (&z)[32], long long label, int c, float* at_row) {
  if (label < c || label >= c + 32) return;
  float at = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) at = (label == c + j) ? z[j] : at;
  *at_row = at;
}

// loss[i] (and norm[i] = (maximum, 1 / sum), if not null) of `rows` rows from stats[slice][row] and the labels' logits; row i
// has label labels[i % label_period]. NaN if the status word is set.
int xent_finish(const float2* stats, long long ld_stats, const float* label_logit, const long long* labels, long long label_period,
                long long ignore_index, long long rows, long long vocab, float2* norm, float* loss, const int* status, cudaStream_t stream);

}  // namespace evox
