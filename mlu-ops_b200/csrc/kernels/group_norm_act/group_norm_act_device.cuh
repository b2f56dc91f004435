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

// 1 / (1 + exp(-u)).  The approximations are good to 2^-22 of their results; the rounding of u log2(e) before them puts
// exp(-u) off by |u| 2^-24 of itself (2^-17 at u = -80, which is 2^-17 of a sigmoid of 10^-35; for positive u it vanishes
// beside the 1).  They flush what is below the float range, where the quotient is 0 or 1 in float.
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
  // gamma du - m1 - xhat m2.  The product is rounded before m1 is taken off it, as it is in m1: in a group of one value
  // nothing is left, where a fused difference would leave the rounding, which rstd makes 316 times larger.
  __device__ __forceinline__ Two inputGrad(int j, Two du, Two xh, Two minus_m1, Two minus_m2) const {
    return fma(xh, minus_m2, addRounded(du * gamma[j], minus_m1, one));
  }
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

// A block's threads: `columns` side by side on a row, `row_threads` rows at a time.
struct Lanes {
  int columns, row_threads;
};

// Bytes of scratch that joinRowThreads needs.
__host__ __device__ constexpr size_t joinBytes(int vec, int threads) { return (size_t)threads * (vec > 2 ? vec : 2) * sizeof(float2); }

// Each thread's two values (a, b) of each of its channels, joined over the block's row threads in double and in a fixed
// order: value(row thread, values, row thread 0's values) is added up, and store(channel, sum, row thread 0's values)
// called once for each of the block's channels.  The values lie side by side in `scratch`, so that lanes read and write
// neighbouring words, and are added in two steps, `parts` threads to a channel first.
template <int VEC, int THREADS, typename V, typename F>
__device__ __forceinline__ void joinRowThreads(const Two (&a)[(VEC + 1) / 2], const Two (&b)[(VEC + 1) / 2], Lanes l,
                                               float2 *scratch, V value, F store) {
  const int tid = threadIdx.x, used = l.columns * l.row_threads;
  __syncthreads();
  if (tid < used) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 x = split(a[j / 2]), y = split(b[j / 2]);
      scratch[j * used + tid] = j % 2 ? make_float2(x.y, y.y) : make_float2(x.x, y.x);
    }
  }
  __syncthreads();
  const int items = VEC * l.columns;  // (j, column), column fastest
  int parts = THREADS / items;
  parts = parts < 1 ? 1 : (parts > l.row_threads ? l.row_threads : parts);
  auto add = [&](double2 &s, int row, float2 v, float2 v0) {
    const double2 t = value(row, v, v0);
    s.x += t.x;
    s.y += t.y;
  };
  if (parts == 1) {
    for (int item = tid; item < items; item += THREADS) {
      const int column = item % l.columns, j = item / l.columns;
      const float2 *from = scratch + j * used + column, v0 = from[0];
      double2 s = make_double2(0.0, 0.0);
      for (int row = 0; row < l.row_threads; ++row) add(s, row, from[row * l.columns], v0);
      store(column * VEC + j, s, v0);
    }
    return;
  }
  double2 *joined = reinterpret_cast<double2 *>(scratch);  // (j, part, column) after the first step
  double2 s = make_double2(0.0, 0.0);
  const int column = tid % l.columns, part = tid / l.columns % parts, j = tid / (l.columns * parts);
  if (j < VEC) {
    const float2 *from = scratch + j * used + column, v0 = from[0];
    for (int row = part; row < l.row_threads; row += parts) add(s, row, from[row * l.columns], v0);
  }
  const bool mine = tid < items;
  const int own_column = tid % l.columns, own_j = tid / l.columns;
  const float2 v0 = mine ? scratch[own_j * used + own_column] : make_float2(0.0f, 0.0f);
  __syncthreads();
  if (j < VEC) joined[tid] = s;
  __syncthreads();
  if (mine) {
    s = make_double2(0.0, 0.0);
    for (int k = 0; k < parts; ++k) {
      const double2 v = joined[(own_j * parts + k) * l.columns + own_column];
      s.x += v.x;
      s.y += v.y;
    }
    store(own_column * VEC + own_j, s, v0);
  }
}
struct PlainSums {
  __device__ __forceinline__ double2 operator()(int, float2 v, float2) const { return make_double2(v.x, v.y); }
};

// (mean, sum of squared deviations) of each of a thread's channels over its `n` rows from sums about k.  Each thread takes
// its own first row as k: the squares then lose no more than a factor of its few rows, wherever an outlier lies.
template <int VEC>
__device__ __forceinline__ void closeMoments(Two (&a)[(VEC + 1) / 2], Two (&b)[(VEC + 1) / 2],
                                             const Two (&minus_k)[(VEC + 1) / 2], int n) {
  const float over = n > 0 ? 1.0f / (float)n : 0.0f;
  const Two inverse = two(over, over), minus = two(-1.0f, -1.0f);
#pragma unroll
  for (int j = 0; j < (VEC + 1) / 2; ++j) {
    const Two off = a[j] * inverse;
    const float2 squares = split(fma(a[j] * minus, off, b[j]));
    b[j] = two(squares.x < 0.0f ? 0.0f : squares.x, squares.y < 0.0f ? 0.0f : squares.y);  // (NaN stays)
    a[j] = off + minus_k[j] * minus;
  }
}
// Joins them over the row threads of `rows` rows: store(channel, mean, sum of squared deviations).
template <int VEC, int THREADS, typename F>
__device__ __forceinline__ void joinMoments(const Two (&a)[(VEC + 1) / 2], const Two (&b)[(VEC + 1) / 2], Lanes l, int rows,
                                            float2 *scratch, F store) {
  const int each = rows / l.row_threads, more = rows % l.row_threads;  // rows of a thread, threads with one more
  joinRowThreads<VEC, THREADS>(
      a, b, l, scratch,
      [&](int row, float2 v, float2 v0) {
        const int own = each + (row < more);
        if (own == 0) return make_double2(0.0, 0.0);
        const double off = (double)v.x - v0.x, part = own * off;
        return make_double2(part, v.y + part * off);
      },
      [&](int c, double2 s, float2 v0) {
        const double off = s.x / (double)rows, squares = s.y - s.x * off;
        store(c, v0.x + off, squares < 0.0 ? 0.0 : squares);
      });
}

}  // namespace group_norm_act
}  // namespace mluop

#endif  // MLUOP_B200_KERNELS_GROUP_NORM_ACT_DEVICE_CUH_
