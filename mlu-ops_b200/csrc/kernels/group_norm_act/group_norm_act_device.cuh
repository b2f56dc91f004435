// Device functions of group norm: samples as rows, arithmetic on pairs of floats.
#ifndef MLUOP_B200_KERNELS_GROUP_NORM_ACT_DEVICE_CUH_
#define MLUOP_B200_KERNELS_GROUP_NORM_ACT_DEVICE_CUH_

#include <cuda_runtime.h>

#include "core/convert.cuh"
#include "core/pair.cuh"
#include "mlu_op.h"

namespace mluop {
namespace group_norm_act {

struct Rows {
  int64_t rows, samples, sample_rows, block_rows;
  const int32_t *ends;  // null: samples of sample_rows rows
  float one;            // 1 (see addRounded)
};

// First row of sample s (s <= samples); within [0, rows] whatever the entries hold.
__device__ __forceinline__ int64_t sampleStart(const Rows &r, int64_t s) {
  if (s <= 0) return 0;
  if (!r.ends) return s * r.sample_rows;
  const int64_t e = r.ends[s - 1];
  return e < 0 ? 0 : (e > r.rows ? r.rows : e);
}

// How many samples end at row `row` or before: the sample that the row belongs to (`samples` behind the last one).
// Called by the whole block.
__device__ __forceinline__ int64_t samplesUpTo(const Rows &r, int64_t row) {
  if (!r.ends) {
    if (r.sample_rows == 0) return r.samples;
    const int64_t s = row / r.sample_rows;
    return s < r.samples ? s : r.samples;
  }
  int64_t before = 0;
  for (int64_t base = 0; base < r.samples; base += blockDim.x) {
    const int64_t i = base + threadIdx.x;
    before += __syncthreads_count(i < r.samples && r.ends[i] <= row);
  }
  return before;
}

// An entry of weight or bias, kept in float or in T.
template <typename T>
__device__ __forceinline__ float loadAffine(const void *p, bool is_float, int c) {
  return is_float ? static_cast<const float *>(p)[c] : toFloat(static_cast<const T *>(p)[c]);
}
template <typename T>
__device__ __forceinline__ void storeAffineGrad(void *p, bool is_float, int c, double v) {
  if (is_float) static_cast<float *>(p)[c] = (float)v;
  else static_cast<T *>(p)[c] = fromFloat<T>((float)v);
}

// 1 / (1 + exp(-u)).  The approximations are good to 2^-22, and flush what is below the float range, where the quotient
// is 0 or 1 in float.
__device__ __forceinline__ Two sigmoid(Two u) {
  float2 e = split(u * two(-1.4426950408889634f, -1.4426950408889634f));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
  float2 d = split(two(e.x, e.y) + two(1.0f, 1.0f));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.y));
  return two(d.x, d.y);
}
template <int ACT>
__device__ __forceinline__ Two activate(Two u) {
  if (ACT == MLUOP_GROUP_NORM_ACT_RELU) {
    const float2 f = split(u);
    return two(f.x < 0.0f ? 0.0f : f.x, f.y < 0.0f ? 0.0f : f.y);  // (NaN stays)
  }
  return ACT == MLUOP_GROUP_NORM_ACT_SILU ? u * sigmoid(u) : u;
}
// dy * act'(u)
template <int ACT>
__device__ __forceinline__ Two activateGrad(Two dy, Two u) {
  if (ACT == MLUOP_GROUP_NORM_ACT_RELU) {
    const float2 g = split(dy), f = split(u);
    return two(f.x > 0.0f ? g.x : 0.0f, f.y > 0.0f ? g.y : 0.0f);
  }
  if (ACT == MLUOP_GROUP_NORM_ACT_SILU) {
    const Two one = two(1.0f, 1.0f), s = sigmoid(u);
    return dy * (s * fma(u, fma(s, two(-1.0f, -1.0f), one), one));
  }
  return dy;
}

// (In pairs an element takes about 7 (relu) to 11 (silu) instructions in a pass over it, against about twice that in
// single floats, where the passes wait for arithmetic instead of memory.)
// What the normalisation of a thread's channels in a sample needs.  UNIFORM: they lie in one group.
template <int VEC, bool UNIFORM>
struct Norm {
  static constexpr int kPairs = (VEC + 1) / 2, kGroups = UNIFORM ? 1 : kPairs;
  Two minus_mean[kGroups], rstd[kGroups], gamma[kPairs], beta[kPairs];
  float one;
  // The activation's argument, rounded after every operation: a value next to the border of relu falls on the same
  // side in the forward pass, in both backward passes and in the formula evaluated step by step.
  __device__ __forceinline__ Two xhat(int j, Two x) const { return (x + minus_mean[UNIFORM ? 0 : j]) * rstd[UNIFORM ? 0 : j]; }
  __device__ __forceinline__ Two affine(int j, Two xh) const { return addRounded(xh * gamma[j], beta[j], one); }
};
// value(c) for the channels of pair j of a thread whose first channel is `first`.
template <int VEC, typename F>
__device__ __forceinline__ Two ofPair(int first, int j, F value) {
  return two(value(first + 2 * j), VEC > 1 ? value(first + 2 * j + 1) : 0.0f);
}
template <typename T, int VEC, bool UNIFORM>
__device__ __forceinline__ void loadNorm(Norm<VEC, UNIFORM> &c, const float *mean, const float *rstd, const void *weight,
                                         const void *bias, bool float_affine, int first, int group_channels, float one) {
  c.one = one;
#pragma unroll
  for (int j = 0; j < Norm<VEC, UNIFORM>::kGroups; ++j) {
    c.minus_mean[j] = ofPair<UNIFORM ? 2 : VEC>(first, j, [&](int ch) { return -mean[(UNIFORM ? first : ch) / group_channels]; });
    c.rstd[j] = ofPair<UNIFORM ? 2 : VEC>(first, j, [&](int ch) { return rstd[(UNIFORM ? first : ch) / group_channels]; });
  }
#pragma unroll
  for (int j = 0; j < Norm<VEC, UNIFORM>::kPairs; ++j) {
    c.gamma[j] = ofPair<VEC>(first, j, [&](int ch) { return weight ? loadAffine<T>(weight, float_affine, ch) : 1.0f; });
    c.beta[j] = ofPair<VEC>(first, j, [&](int ch) { return bias ? loadAffine<T>(bias, float_affine, ch) : 0.0f; });
  }
}

}  // namespace group_norm_act
}  // namespace mluop

#endif  // MLUOP_B200_KERNELS_GROUP_NORM_ACT_DEVICE_CUH_
