// Group norm with an activation on channels-last rows, and its gradients.
//
// Forward, for sample n and group q over the sample's rows and the group's channels:
//   rstd = 1 / sqrt(var + eps),  y = act(gamma (x - mean) rstd + beta)
// Backward, with xhat = (x - mean) rstd and du = dy act'(gamma xhat + beta):
//   dbeta = sum du,  dgamma = sum du xhat,
//   dx = rstd (gamma du - mean(gamma du) - xhat mean(gamma du xhat))
//
// Both are bound by memory: x (and dy) read once and one tensor written is the floor.
// Both are two passes over the rows with a small kernel between them:
//   1. sums per block of rows and channel (a block's threads lie side by side on the
//      channels, 16 bytes each, and walk down the rows);
//   2. one block per (sample, group) joins them, in double and in a fixed order;
//   3. the outputs, from the rows again.  The blocks run from the last rows to the
//      first, so that the rows that pass 1 read last are still in L2.
// A block that meets the end of a sample closes its sums and begins new ones: its
// sums for sample s go to slot block + s, which is unique and makes the slots of one
// sample neighbours, whatever the samples' sizes (they are known on the device only).
//
// Variance: pass 1 sums x - k and (x - k)^2 with k the block's first value of that
// channel, which is within a few deviations of the mean; the blocks' (mean, sum of
// squared deviations) pairs are joined without cancellation.
#include "kernels/group_norm_act/group_norm_act_kernels.h"

#include <cuda_runtime.h>

#include <algorithm>

#include "core/convert.cuh"
#include "core/trace.h"
#include "core/type.h"

namespace mluop {
namespace group_norm_act {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows a thread has in flight

struct Rows {
  int64_t rows, samples, sample_rows, block_rows;
  const int32_t *ends;  // null: samples of sample_rows rows
};

// First row of sample s (s <= samples); within [0, rows] whatever the entries hold.
__device__ __forceinline__ int64_t sampleStart(const Rows &r, int64_t s) {
  if (s <= 0) return 0;
  if (!r.ends) return s * r.sample_rows;
  const int64_t e = r.ends[s - 1];
  return e < 0 ? 0 : (e > r.rows ? r.rows : e);
}

// The sample that row `row` belongs to (`samples` behind the last one); called by the whole block.
__device__ __forceinline__ int64_t sampleOf(const Rows &r, int64_t row) {
  if (!r.ends) return r.sample_rows ? row / r.sample_rows : r.samples;
  int64_t before = 0;
  for (int64_t base = 0; base < r.samples; base += kThreads) {
    const int64_t i = base + threadIdx.x;
    before += __syncthreads_count(i < r.samples && r.ends[i] <= row);
  }
  return before;
}

__device__ __forceinline__ float loadAffine(const void *p, bool is_float, const float *, int c) {
  return static_cast<const float *>(p)[c];
}
template <typename T>
__device__ __forceinline__ float loadAffine(const void *p, bool is_float, const T *, int c) {
  return is_float ? static_cast<const float *>(p)[c] : toFloat(static_cast<const T *>(p)[c]);
}

template <int ACT>
__device__ __forceinline__ float activate(float u) {
  if (ACT == MLUOP_GROUP_NORM_ACT_RELU) return u < 0.0f ? 0.0f : u;  // (NaN stays)
  if (ACT == MLUOP_GROUP_NORM_ACT_SILU) return __fdividef(u, 1.0f + __expf(-u));
  return u;
}
// dy * act'(u)
template <int ACT>
__device__ __forceinline__ float activateGrad(float dy, float u) {
  if (ACT == MLUOP_GROUP_NORM_ACT_RELU) return u > 0.0f ? dy : 0.0f;
  if (ACT == MLUOP_GROUP_NORM_ACT_SILU) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-u));
    return dy * (s * (1.0f + u * (1.0f - s)));
  }
  return dy;
}

// Adds (a, b) of each channel over the block's row threads; the sums are returned to row thread 0.
template <int VEC>
__device__ __forceinline__ void addOverRowThreads(float (&a)[VEC], float (&b)[VEC], int column, int row, int columns,
                                                  int row_threads, bool active, float2 *scratch) {
  __syncthreads();
  if (active) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) scratch[(row * VEC + j) * columns + column] = make_float2(a[j], b[j]);
  }
  for (int half = row_threads; half > 1;) {
    const int next = (half + 1) / 2;
    __syncthreads();
    if (active && row + next < half) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 mine = scratch[(row * VEC + j) * columns + column];
        const float2 other = scratch[((row + next) * VEC + j) * columns + column];
        scratch[(row * VEC + j) * columns + column] = make_float2(mine.x + other.x, mine.y + other.y);
      }
    }
    half = next;
  }
  if (active && row == 0) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 sum = scratch[j * columns + column];
      a[j] = sum.x;
      b[j] = sum.y;
    }
  }
}

// Per channel of the thread: what the normalisation needs.
template <int VEC>
struct Channel {
  float mean[VEC], rstd[VEC], gamma[VEC], beta[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void loadChannels(Channel<VEC> &c, const float *mean, const float *rstd, const void *weight,
                                             const void *bias, bool float_affine, int64_t sample, int first, int groups,
                                             int group_channels) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const int64_t q = sample * groups + (first + j) / group_channels;
    c.mean[j] = mean[q];
    c.rstd[j] = rstd[q];
    c.gamma[j] = weight ? loadAffine(weight, float_affine, (const T *)nullptr, first + j) : 1.0f;
    c.beta[j] = bias ? loadAffine(bias, float_affine, (const T *)nullptr, first + j) : 0.0f;
  }
}
// The activation's argument, rounded after every operation: a value next to the border of relu falls on the same
// side in the forward pass, in both backward passes and in the formula evaluated step by step.
template <int VEC>
__device__ __forceinline__ float normalised(const Channel<VEC> &c, int j, float x) {
  return __fmul_rn(__fsub_rn(x, c.mean[j]), c.rstd[j]);
}
template <int VEC>
__device__ __forceinline__ float affine(const Channel<VEC> &c, int j, float xhat) {
  return __fadd_rn(__fmul_rn(xhat, c.gamma[j]), c.beta[j]);
}

// Pass 1 forward: partial[slot][channel] = (mean, sum of squared deviations) of the block's rows of a sample.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
statisticsKernel(const T *x, Rows r, int channels, int columns, int row_threads, float2 *partial) {
  extern __shared__ float2 scratch[];
  const int column = threadIdx.x % columns, row = threadIdx.x / columns;
  const int first = (blockIdx.y * columns + column) * VEC;
  const bool active = row < row_threads && first < channels;
  const int64_t begin = (int64_t)blockIdx.x * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  int64_t sample = sampleOf(r, begin);
  for (int64_t at = begin; at < end && sample < r.samples; ++sample) {
    int64_t stop = sampleStart(r, sample + 1);
    stop = stop < end ? stop : end;
    if (stop <= at) continue;
    float k[VEC], s[VEC], q[VEC];
    if (active) {
      const Pack<VEC, T> p = loadPack<VEC>(x + at * channels + first);
#pragma unroll
      for (int j = 0; j < VEC; ++j) k[j] = toFloat(p.v[j]);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = q[j] = 0.0f;
    if (active) {
      int64_t i = at + row;
      for (; i + (kUnroll - 1) * row_threads < stop; i += kUnroll * row_threads) {
        Pack<VEC, T> p[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) p[u] = loadPack<VEC>(x + (i + u * row_threads) * channels + first);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float d = toFloat(p[u].v[j]) - k[j];
            s[j] += d;
            q[j] += d * d;
          }
        }
      }
      for (; i < stop; i += row_threads) {
        const Pack<VEC, T> p = loadPack<VEC>(x + i * channels + first);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = toFloat(p.v[j]) - k[j];
          s[j] += d;
          q[j] += d * d;
        }
      }
    }
    addOverRowThreads<VEC>(s, q, column, row, columns, row_threads, active, scratch);
    if (active && row == 0) {
      const float n = (float)(stop - at);
      float2 *out = partial + (blockIdx.x + sample) * channels + first;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float off = s[j] / n;
        const float squares = q[j] - s[j] * off;
        out[j] = make_float2(k[j] + off, squares < 0.0f ? 0.0f : squares);  // (NaN stays)
      }
    }
    at = stop;
  }
}

// Sum over the block in a fixed order, returned to every thread.
__device__ __forceinline__ double blockSum(double v, double *scratch) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < kThreads / 32; ++w) v += scratch[w];
  return v;
}

// Pass 2 forward: one block per (sample, group).
__global__ void __launch_bounds__(kThreads)
joinStatisticsKernel(const float2 *partial, Rows r, int channels, int groups, float epsilon, float *mean, float *rstd) {
  __shared__ double scratch[kThreads / 32];
  const int64_t sample = blockIdx.x / groups;
  const int group = blockIdx.x % groups, group_channels = channels / groups;
  const int64_t begin = sampleStart(r, sample), end = sampleStart(r, sample + 1);
  double m = 0.0, sq = 0.0;
  if (end > begin) {
    const int64_t b0 = begin / r.block_rows, b1 = (end - 1) / r.block_rows;
    const int64_t items = (b1 - b0 + 1) * group_channels;
    const double total = (double)(end - begin) * group_channels;
    for (int64_t i = threadIdx.x; i < items; i += kThreads) {
      const int64_t b = b0 + i / group_channels;
      const int64_t from = b * r.block_rows > begin ? b * r.block_rows : begin;
      const int64_t to = (b + 1) * r.block_rows < end ? (b + 1) * r.block_rows : end;
      m += (double)(to - from) * partial[(b + sample) * channels + group * group_channels + i % group_channels].x;
    }
    m = blockSum(m, scratch) / total;
    for (int64_t i = threadIdx.x; i < items; i += kThreads) {
      const int64_t b = b0 + i / group_channels;
      const int64_t from = b * r.block_rows > begin ? b * r.block_rows : begin;
      const int64_t to = (b + 1) * r.block_rows < end ? (b + 1) * r.block_rows : end;
      const float2 v = partial[(b + sample) * channels + group * group_channels + i % group_channels];
      const double d = (double)v.x - m;
      sq += (double)v.y + (double)(to - from) * d * d;
    }
    sq = blockSum(sq, scratch) / total;
  }
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = (float)m;
    rstd[blockIdx.x] = (float)(1.0 / sqrt(sq + (double)epsilon));
  }
}

// Pass 3 forward.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kThreads)
normaliseKernel(const T *x, const void *weight, const void *bias, bool float_affine, const float *mean,
                const float *rstd, Rows r, int channels, int groups, int columns, int row_threads, T *y) {
  const int column = threadIdx.x % columns, row = threadIdx.x / columns;
  const int first = (blockIdx.y * columns + column) * VEC;
  const bool active = row < row_threads && first < channels;
  const int64_t begin = (int64_t)(gridDim.x - 1 - blockIdx.x) * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  int64_t sample = sampleOf(r, begin);
  if (!active) return;
  for (int64_t at = begin; at < end; ++sample) {
    if (sample >= r.samples) {  // rows of no sample
      Pack<VEC, T> zero;
#pragma unroll
      for (int j = 0; j < VEC; ++j) zero.v[j] = fromFloat<T>(0.0f);
      for (int64_t i = at + row; i < end; i += row_threads) storePack<VEC>(y + i * channels + first, zero);
      return;
    }
    int64_t stop = sampleStart(r, sample + 1);
    stop = stop < end ? stop : end;
    if (stop <= at) continue;
    Channel<VEC> c;
    loadChannels<T, VEC>(c, mean, rstd, weight, bias, float_affine, sample, first, groups, channels / groups);
    int64_t i = at + row;
    for (; i + (kUnroll - 1) * row_threads < stop; i += kUnroll * row_threads) {
      Pack<VEC, T> p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = loadPack<VEC>(x + (i + u * row_threads) * channels + first);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          p[u].v[j] = fromFloat<T>(activate<ACT>(affine(c, j, normalised(c, j, toFloat(p[u].v[j])))));
        storePack<VEC>(y + (i + u * row_threads) * channels + first, p[u]);
      }
    }
    for (; i < stop; i += row_threads) {
      Pack<VEC, T> p = loadPack<VEC>(x + i * channels + first);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        p.v[j] = fromFloat<T>(activate<ACT>(affine(c, j, normalised(c, j, toFloat(p.v[j])))));
      storePack<VEC>(y + i * channels + first, p);
    }
    at = stop;
  }
}

// Pass 1 backward: partial[slot][channel] = (sum du, sum du xhat) of the block's rows of a sample.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kThreads)
gradSumsKernel(const T *dy, const T *x, const void *weight, const void *bias, bool float_affine, const float *mean,
               const float *rstd, Rows r, int channels, int groups, int columns, int row_threads, float2 *partial) {
  extern __shared__ float2 scratch[];
  const int column = threadIdx.x % columns, row = threadIdx.x / columns;
  const int first = (blockIdx.y * columns + column) * VEC;
  const bool active = row < row_threads && first < channels;
  const int64_t begin = (int64_t)blockIdx.x * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  int64_t sample = sampleOf(r, begin);
  for (int64_t at = begin; at < end && sample < r.samples; ++sample) {
    int64_t stop = sampleStart(r, sample + 1);
    stop = stop < end ? stop : end;
    if (stop <= at) continue;
    float a[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = b[j] = 0.0f;
    if (active) {
      Channel<VEC> c;
      loadChannels<T, VEC>(c, mean, rstd, weight, bias, float_affine, sample, first, groups, channels / groups);
      int64_t i = at + row;
      for (; i + (kUnroll - 1) * row_threads < stop; i += kUnroll * row_threads) {
        Pack<VEC, T> p[kUnroll], g[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          p[u] = loadPack<VEC>(x + (i + u * row_threads) * channels + first);
          g[u] = loadPack<VEC>(dy + (i + u * row_threads) * channels + first);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float xhat = normalised(c, j, toFloat(p[u].v[j]));
            const float du = activateGrad<ACT>(toFloat(g[u].v[j]), affine(c, j, xhat));
            a[j] += du;
            b[j] += du * xhat;
          }
        }
      }
      for (; i < stop; i += row_threads) {
        const Pack<VEC, T> p = loadPack<VEC>(x + i * channels + first);
        const Pack<VEC, T> g = loadPack<VEC>(dy + i * channels + first);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xhat = normalised(c, j, toFloat(p.v[j]));
          const float du = activateGrad<ACT>(toFloat(g.v[j]), affine(c, j, xhat));
          a[j] += du;
          b[j] += du * xhat;
        }
      }
    }
    addOverRowThreads<VEC>(a, b, column, row, columns, row_threads, active, scratch);
    if (active && row == 0) {
      float2 *out = partial + (blockIdx.x + sample) * channels + first;
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[j] = make_float2(a[j], b[j]);
    }
    at = stop;
  }
}

// Pass 2 backward: one block per (sample, group): the sample's sums per channel, and the group's two means.
template <typename T>
__global__ void __launch_bounds__(kThreads)
joinGradSumsKernel(const float2 *partial, const void *weight, bool float_affine, Rows r, int channels, int groups,
                   float2 *sample_sums, float2 *group_means) {
  __shared__ double scratch[kThreads / 32];
  __shared__ double2 lanes[kThreads];
  const int64_t sample = blockIdx.x / groups;
  const int group = blockIdx.x % groups, group_channels = channels / groups;
  const int64_t begin = sampleStart(r, sample), end = sampleStart(r, sample + 1);
  // a tile of up to 32 channels side by side, the other threads along the slots
  const int width = group_channels < 32 ? group_channels : 32, depth = kThreads / width;
  const int c = threadIdx.x % width, d = threadIdx.x / width;
  double m1 = 0.0, m2 = 0.0;
  for (int base = 0; base < group_channels; base += width) {
    const int channel = group * group_channels + base + c;
    const bool active = d < depth && base + c < group_channels;
    double a = 0.0, b = 0.0;
    if (active && end > begin) {
      const int64_t last = (end - 1) / r.block_rows;
      for (int64_t k = begin / r.block_rows + d; k <= last; k += depth) {
        const float2 v = partial[(k + sample) * channels + channel];
        a += v.x;
        b += v.y;
      }
    }
    __syncthreads();
    lanes[threadIdx.x] = make_double2(a, b);
    __syncthreads();
    if (active && d == 0) {
      for (int i = 1; i < depth; ++i) {
        a += lanes[i * width + c].x;
        b += lanes[i * width + c].y;
      }
      sample_sums[sample * channels + channel] = make_float2((float)a, (float)b);
      const double gamma = weight ? (double)loadAffine(weight, float_affine, (const T *)nullptr, channel) : 1.0;
      m1 += gamma * a;
      m2 += gamma * b;
    }
  }
  m1 = blockSum(m1, scratch);
  m2 = blockSum(m2, scratch);
  if (threadIdx.x == 0) {
    const double n = end > begin ? (double)(end - begin) * group_channels : 1.0;
    group_means[blockIdx.x] = make_float2((float)(m1 / n), (float)(m2 / n));
  }
}

template <typename T>
__device__ __forceinline__ void storeAffineGrad(void *p, bool is_float, int c, double v) {
  if (is_float) static_cast<float *>(p)[c] = (float)v;
  else static_cast<T *>(p)[c] = fromFloat<T>((float)v);
}

// Pass 3 backward: the input gradient; the first blocks also add the samples' sums to the affine gradients.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kThreads)
inputGradKernel(const T *dy, const T *x, const void *weight, const void *bias, bool float_affine, const float *mean,
                const float *rstd, const float2 *sample_sums, const float2 *group_means, Rows r, int channels,
                int groups, int columns, int row_threads, T *dx, void *weight_grad, void *bias_grad,
                bool float_affine_grad) {
  const int column = threadIdx.x % columns, row = threadIdx.x / columns;
  const int first = (blockIdx.y * columns + column) * VEC;
  const bool active = row < row_threads && first < channels;
  if (weight_grad) {
    const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int64_t all = (int64_t)gridDim.x * gridDim.y * kThreads;
    for (int64_t ch = block * kThreads + threadIdx.x; ch < channels; ch += all) {
      double a = 0.0, b = 0.0;
      for (int64_t s = 0; s < r.samples; ++s) {
        const float2 v = sample_sums[s * channels + ch];
        a += v.x;
        b += v.y;
      }
      storeAffineGrad<T>(bias_grad, float_affine_grad, (int)ch, a);
      storeAffineGrad<T>(weight_grad, float_affine_grad, (int)ch, b);
    }
  }
  const int64_t begin = (int64_t)(gridDim.x - 1 - blockIdx.x) * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  int64_t sample = sampleOf(r, begin);
  if (!active) return;
  const int group_channels = channels / groups;
  for (int64_t at = begin; at < end; ++sample) {
    if (sample >= r.samples) {  // rows of no sample
      Pack<VEC, T> zero;
#pragma unroll
      for (int j = 0; j < VEC; ++j) zero.v[j] = fromFloat<T>(0.0f);
      for (int64_t i = at + row; i < end; i += row_threads) storePack<VEC>(dx + i * channels + first, zero);
      return;
    }
    int64_t stop = sampleStart(r, sample + 1);
    stop = stop < end ? stop : end;
    if (stop <= at) continue;
    Channel<VEC> c;
    loadChannels<T, VEC>(c, mean, rstd, weight, bias, float_affine, sample, first, groups, group_channels);
    float m1[VEC], m2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 v = group_means[sample * groups + (first + j) / group_channels];
      m1[j] = v.x;
      m2[j] = v.y;
    }
    for (int64_t i = at + row; i < stop; i += 2 * row_threads) {
      const bool two = i + row_threads < stop;
      Pack<VEC, T> p[2], g[2];
      p[0] = loadPack<VEC>(x + i * channels + first);
      g[0] = loadPack<VEC>(dy + i * channels + first);
      if (two) {
        p[1] = loadPack<VEC>(x + (i + row_threads) * channels + first);
        g[1] = loadPack<VEC>(dy + (i + row_threads) * channels + first);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (u == 1 && !two) break;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xhat = normalised(c, j, toFloat(p[u].v[j]));
          const float du = activateGrad<ACT>(toFloat(g[u].v[j]), affine(c, j, xhat));
          g[u].v[j] = fromFloat<T>((du * c.gamma[j] - m1[j] - xhat * m2[j]) * c.rstd[j]);
        }
        storePack<VEC>(dx + (i + u * row_threads) * channels + first, g[u]);
      }
    }
    at = stop;
  }
}

size_t roundUp(size_t v) { return (v + 255) / 256 * 256; }

Rows rowsOf(const NormProblem &p, const NormPlan &plan) {
  return Rows{p.rows, p.samples, p.sample_rows, plan.block_rows, p.sample_ends};
}

char *scratchBase(void *workspace) {
  return reinterpret_cast<char *>((reinterpret_cast<size_t>(workspace) + 255) / 256 * 256);
}

double rowBytes(const NormProblem &p) {
  return (double)p.rows * p.channels * mluop::getSizeOfDataType(p.dtype);
}

template <typename T, int VEC>
cudaError_t forward(const NormProblem &p, const NormPlan &plan, const void *input, const void *weight,
                    const void *bias, void *workspace, void *output, float *mean, float *rstd, cudaStream_t stream) {
  char *base = scratchBase(workspace);
  float2 *partial = reinterpret_cast<float2 *>(base + plan.partial);
  const T *x = static_cast<const T *>(input);
  T *y = static_cast<T *>(output);
  const Rows r = rowsOf(p, plan);
  const dim3 grid((unsigned)plan.blocks, (unsigned)plan.column_tiles);
  const size_t smem = (size_t)plan.column_threads * plan.row_threads * VEC * sizeof(float2);
  {
    trace::Scope scope("groupNormStatisticsKernel", stream, rowBytes(p));
    statisticsKernel<T, VEC><<<grid, kThreads, smem, stream>>>(x, r, p.channels, plan.column_threads,
                                                               plan.row_threads, partial);
  }
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  if (p.samples > 0) {
    trace::Scope scope("groupNormJoinKernel", stream);
    joinStatisticsKernel<<<(unsigned)(p.samples * p.groups), kThreads, 0, stream>>>(partial, r, p.channels, p.groups,
                                                                                    p.epsilon, mean, rstd);
  }
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  trace::Scope scope("groupNormNormaliseKernel", stream, 2 * rowBytes(p));
  auto kernel = p.activation == MLUOP_GROUP_NORM_ACT_RELU   ? normaliseKernel<T, VEC, MLUOP_GROUP_NORM_ACT_RELU>
                : p.activation == MLUOP_GROUP_NORM_ACT_SILU ? normaliseKernel<T, VEC, MLUOP_GROUP_NORM_ACT_SILU>
                                                            : normaliseKernel<T, VEC, MLUOP_GROUP_NORM_ACT_NONE>;
  kernel<<<grid, kThreads, 0, stream>>>(x, weight, bias, p.float_affine, mean, rstd, r, p.channels, p.groups,
                                        plan.column_threads, plan.row_threads, y);
  return cudaGetLastError();
}

template <typename T, int VEC, int ACT>
cudaError_t backward(const NormProblem &p, const NormPlan &plan, const void *output_grad, const void *input,
                     const void *weight, const void *bias, const float *mean, const float *rstd, void *workspace,
                     void *input_grad, void *weight_grad, void *bias_grad, cudaStream_t stream) {
  char *base = scratchBase(workspace);
  float2 *partial = reinterpret_cast<float2 *>(base + plan.partial);
  float2 *sample_sums = reinterpret_cast<float2 *>(base + plan.sample_sums);
  float2 *group_means = reinterpret_cast<float2 *>(base + plan.group_means);
  const T *dy = static_cast<const T *>(output_grad), *x = static_cast<const T *>(input);
  const Rows r = rowsOf(p, plan);
  const dim3 grid((unsigned)plan.blocks, (unsigned)plan.column_tiles);
  const size_t smem = (size_t)plan.column_threads * plan.row_threads * VEC * sizeof(float2);
  {
    trace::Scope scope("groupNormGradSumsKernel", stream, 2 * rowBytes(p));
    gradSumsKernel<T, VEC, ACT><<<grid, kThreads, smem, stream>>>(dy, x, weight, bias, p.float_affine, mean, rstd, r,
                                                                  p.channels, p.groups, plan.column_threads,
                                                                  plan.row_threads, partial);
  }
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  if (p.samples > 0) {
    trace::Scope scope("groupNormGradJoinKernel", stream);
    joinGradSumsKernel<T><<<(unsigned)(p.samples * p.groups), kThreads, 0, stream>>>(
        partial, weight, p.float_affine, r, p.channels, p.groups, sample_sums, group_means);
  }
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  trace::Scope scope("groupNormInputGradKernel", stream, 3 * rowBytes(p));
  inputGradKernel<T, VEC, ACT><<<grid, kThreads, 0, stream>>>(
      dy, x, weight, bias, p.float_affine, mean, rstd, sample_sums, group_means, r, p.channels, p.groups,
      plan.column_threads, plan.row_threads, static_cast<T *>(input_grad), weight_grad, bias_grad,
      p.float_affine_grad);
  return cudaGetLastError();
}

template <typename T, int VEC, typename... Args>
cudaError_t backwardAct(const NormProblem &p, Args... args) {
  switch (p.activation) {
    case MLUOP_GROUP_NORM_ACT_RELU: return backward<T, VEC, MLUOP_GROUP_NORM_ACT_RELU>(p, args...);
    case MLUOP_GROUP_NORM_ACT_SILU: return backward<T, VEC, MLUOP_GROUP_NORM_ACT_SILU>(p, args...);
    default: return backward<T, VEC, MLUOP_GROUP_NORM_ACT_NONE>(p, args...);
  }
}

bool aligned16(const void *p) { return reinterpret_cast<size_t>(p) % 16 == 0; }

}  // namespace

NormPlan planNorm(const NormProblem &p, bool backward, bool vectors) {
  NormPlan plan{};
  const int wide = 16 / (int)mluop::getSizeOfDataType(p.dtype);
  plan.vec = vectors && p.channels % wide == 0 ? wide : 1;
  const int columns = (p.channels + plan.vec - 1) / plan.vec;
  plan.column_threads = std::min(columns, kThreads);
  plan.column_tiles = (columns + plan.column_threads - 1) / plan.column_threads;
  plan.row_threads = kThreads / plan.column_threads;
  // six blocks per SM over all column tiles, and at least one unrolled turn for each block
  const int64_t wanted = std::max<int64_t>(1, (int64_t)6 * p.sm_count / plan.column_tiles);
  const int64_t turn = (int64_t)kUnroll * plan.row_threads;
  plan.block_rows = std::max<int64_t>(1, (p.rows + wanted - 1) / wanted);
  plan.block_rows = (plan.block_rows + turn - 1) / turn * turn;
  plan.blocks = std::max<int64_t>(1, (p.rows + plan.block_rows - 1) / plan.block_rows);
  plan.partial = 0;
  plan.sample_sums = roundUp((size_t)(plan.blocks + p.samples) * p.channels * sizeof(float2));
  plan.group_means = plan.sample_sums + (backward ? roundUp((size_t)p.samples * p.channels * sizeof(float2)) : 0);
  plan.total = plan.group_means + (backward ? roundUp((size_t)p.samples * p.groups * sizeof(float2)) : 0) + 256;
  return plan;
}

size_t normWorkspaceBytes(const NormProblem &p, bool backward) {
  return std::max(planNorm(p, backward, true).total, planNorm(p, backward, false).total);
}

cudaError_t launchNormForward(const NormProblem &p, const void *input, const void *weight, const void *bias,
                              void *workspace, void *output, float *mean, float *rstd, cudaStream_t stream) {
  const NormPlan plan = planNorm(p, false, aligned16(input) && aligned16(output));
#define MLUOP_FORWARD(T, VEC) forward<T, VEC>(p, plan, input, weight, bias, workspace, output, mean, rstd, stream)
  switch (p.dtype) {
    case MLUOP_DTYPE_FLOAT: return plan.vec == 4 ? MLUOP_FORWARD(float, 4) : MLUOP_FORWARD(float, 1);
    case MLUOP_DTYPE_HALF: return plan.vec == 8 ? MLUOP_FORWARD(__half, 8) : MLUOP_FORWARD(__half, 1);
    default: return plan.vec == 8 ? MLUOP_FORWARD(__nv_bfloat16, 8) : MLUOP_FORWARD(__nv_bfloat16, 1);
  }
#undef MLUOP_FORWARD
}

cudaError_t launchNormBackward(const NormProblem &p, const void *output_grad, const void *input, const void *weight,
                               const void *bias, const float *mean, const float *rstd, void *workspace,
                               void *input_grad, void *weight_grad, void *bias_grad, cudaStream_t stream) {
  const NormPlan plan = planNorm(p, true, aligned16(output_grad) && aligned16(input) && aligned16(input_grad));
#define MLUOP_BACKWARD(T, VEC)                                                                                    \
  backwardAct<T, VEC>(p, plan, output_grad, input, weight, bias, mean, rstd, workspace, input_grad, weight_grad, \
                      bias_grad, stream)
  switch (p.dtype) {
    case MLUOP_DTYPE_FLOAT: return plan.vec == 4 ? MLUOP_BACKWARD(float, 4) : MLUOP_BACKWARD(float, 1);
    case MLUOP_DTYPE_HALF: return plan.vec == 8 ? MLUOP_BACKWARD(__half, 8) : MLUOP_BACKWARD(__half, 1);
    default: return plan.vec == 8 ? MLUOP_BACKWARD(__nv_bfloat16, 8) : MLUOP_BACKWARD(__nv_bfloat16, 1);
  }
#undef MLUOP_BACKWARD
}

}  // namespace group_norm_act
}  // namespace mluop
