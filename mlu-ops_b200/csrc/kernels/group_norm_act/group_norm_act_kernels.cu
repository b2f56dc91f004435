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
// Few rows in a sample: the three launches would take longer than their work, and many samples
// would close a block's sums again and again.  There one block takes a slice of channels that
// holds whole groups, of one sample (backward: of some samples one after the other) and does
// all three steps; the second reading comes from L1 or L2.  Very few rows: a few lanes take a
// (sample, group) (shortSamplesKernel).
//
// Variance: pass 1 sums x - k and (x - k)^2 with k the thread's first value of that
// channel; the threads' and the blocks' (mean, sum of squared deviations) pairs are
// joined without cancellation.
#include "kernels/group_norm_act/group_norm_act_kernels.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <numeric>

#include "core/launch.cuh"
#include "core/trace.h"
#include "core/type.h"
#include "kernels/group_norm_act/group_norm_act_device.cuh"

namespace mluop {
namespace group_norm_act {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows a thread has in flight
constexpr int kSmallThreads = 512;
constexpr int kSmallTurns = 4;   // rows a thread of the one-launch form takes, at most

// Calls body(first row, last row + 1, sample) for the parts of rows begin .. end-1 that belong to one sample each, and
// rest(first row) for the rows of no sample; by the whole block.
template <typename F, typename G>
__device__ __forceinline__ void forSamples(const Rows &r, int64_t begin, int64_t end, F body, G rest) {
  int64_t sample = samplesUpTo(r, begin);
  for (int64_t at = begin; at < end; ++sample) {
    if (sample >= r.samples) {
      rest(at);
      return;
    }
    int64_t stop = sampleStart(r, sample + 1);
    stop = stop < end ? stop : end;
    if (stop <= at) continue;
    body(at, stop, sample);
    at = stop;
  }
}

// Pass 1 forward: partial[slot][channel] = (mean, sum of squared deviations) of the block's rows of a sample.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 4)
statisticsKernel(const T *x, Rows r, int channels, Lanes l, float2 *partial) {
  letNextKernelStart();
  extern __shared__ __align__(16) float2 scratch[];
  constexpr int kPairs = (VEC + 1) / 2;
  const int column = threadIdx.x % l.columns, row = threadIdx.x / l.columns;
  const int first0 = blockIdx.y * l.columns * VEC, first = first0 + column * VEC;
  const bool active = row < l.row_threads && first < channels;
  const int64_t begin = (int64_t)blockIdx.x * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  const int64_t step = (int64_t)l.row_threads * channels;
  forSamples(r, begin, end, [&](int64_t at, int64_t stop, int64_t sample) {
    Two a[kPairs], b[kPairs], minus_k[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) a[j] = b[j] = minus_k[j] = two(0.0f, 0.0f);
    const int own = active && stop - at > row ? ((int)(stop - at) - row + l.row_threads - 1) / l.row_threads : 0;
    if (own > 0) {
      Values<T, VEC> k;
      k.load(x + (at + row) * channels + first);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) minus_k[j] = k.pair(j) * two(-1.0f, -1.0f);
      auto add = [&](const Values<T, VEC> &v) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const Two d = v.pair(j) + minus_k[j];
          a[j] = a[j] + d;
          b[j] = fma(d, d, b[j]);
        }
      };
      int left = (int)(stop - at) - row;  // rows from the thread's next one on
      const T *from = x + (at + row) * channels + first;
      for (; left > (kUnroll - 1) * l.row_threads; left -= kUnroll * l.row_threads, from += kUnroll * step) {
        Values<T, VEC> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u].load(from + u * step);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) add(v[u]);
      }
      for (; left > 0; left -= l.row_threads, from += step) {
        Values<T, VEC> v;
        v.load(from);
        add(v);
      }
    }
    closeMoments<VEC>(a, b, minus_k, own);
    float2 *out = partial + (blockIdx.x + sample) * channels + first0;
    joinMoments<VEC, kThreads>(a, b, l, (int)(stop - at), scratch, [&](int c, double m, double squares) {
      if (first0 + c < channels) out[c] = make_float2((float)m, (float)squares);
    });
  }, [](int64_t) {});
}

// Sums over the block in a fixed order, returned to every thread.
__device__ __forceinline__ double2 blockSum(double a, double b, double2 *scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_double2(a, b);
  __syncthreads();
  a = b = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    a += scratch[w].x;
    b += scratch[w].y;
  }
  return make_double2(a, b);
}

// The slots of a sample: those of blocks first .. last.
struct SampleSlots {
  int64_t begin, end;
  int first, last;
  __device__ __forceinline__ SampleSlots(const Rows &r, int64_t sample) {
    begin = sampleStart(r, sample);
    end = sampleStart(r, sample + 1);
    const unsigned rows = (unsigned)r.block_rows;  // (fewer than 2^31 rows)
    first = (int)((unsigned)begin / rows);
    last = end > begin ? (int)((unsigned)(end - 1) / rows) : first - 1;
  }
};

// Pass 2 forward: one block per (sample, group).  The blocks' means are joined as distances from the first one.
__global__ void __launch_bounds__(kThreads)
joinStatisticsKernel(const float2 *partial, Rows r, int channels, int groups, float epsilon, float *mean, float *rstd) {
  letNextKernelStart();
  __shared__ double2 scratch[kThreads / 32];
  const int64_t sample = blockIdx.x / groups;
  const int group = blockIdx.x % groups, group_channels = channels / groups;
  const SampleSlots s(r, sample);
  const int width = group_channels < kThreads ? group_channels : kThreads, depth = kThreads / width;
  const int c0 = threadIdx.x % width, d = threadIdx.x / width;
  double a = 0.0, b = 0.0, ref = 0.0;
  waitForKernelBefore();
  if (s.last >= s.first && d < depth) {
    const float2 *from = partial + sample * channels + (int64_t)group * group_channels;
    ref = from[(int64_t)s.first * channels].x;
    for (int c = c0; c < group_channels; c += width) {
      for (int64_t k = s.first + d; k <= s.last; k += depth) {
        const int64_t lo = k * r.block_rows > s.begin ? k * r.block_rows : s.begin;
        const int64_t hi = (k + 1) * r.block_rows < s.end ? (k + 1) * r.block_rows : s.end;
        const float2 v = from[k * channels + c];
        const double n = (double)(hi - lo), off = (double)v.x - ref;
        a += n * off;
        b += (double)v.y + n * off * off;
      }
    }
  }
  const double2 sum = blockSum(a, b, scratch);
  if (threadIdx.x == 0) {
    float m = 0.0f;
    double var = 0.0;
    if (s.last >= s.first) {
      const double n = (double)(s.end - s.begin) * group_channels, off = sum.x / n;
      m = (float)(ref + off);
      var = sum.y / n - off * off;
      var = var < 0.0 ? 0.0 : var;  // (NaN stays)
    }
    mean[blockIdx.x] = m;
    rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)epsilon));
  }
}

// Pass 3 forward.
template <typename T, int VEC, int ACT, bool UNIFORM>
__global__ void __launch_bounds__(kThreads, 4)
normaliseKernel(const T *x, const void *weight, const void *bias, bool float_affine, const float *mean,
                const float *rstd, Rows r, int channels, int groups, Lanes l, T *y) {
  constexpr int kPairs = (VEC + 1) / 2;
  const int column = threadIdx.x % l.columns, row = threadIdx.x / l.columns;
  const int first = (blockIdx.y * l.columns + column) * VEC;
  const bool active = row < l.row_threads && first < channels;
  const int64_t begin = (int64_t)(gridDim.x - 1 - blockIdx.x) * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  const int64_t step = (int64_t)l.row_threads * channels;
  waitForKernelBefore();
  forSamples(r, begin, end, [&](int64_t at, int64_t stop, int64_t sample) {
    if (!active) return;
    Norm<VEC, UNIFORM> c;
    loadNorm<T>(c, mean + sample * groups, rstd + sample * groups, weight, bias, float_affine, first, channels / groups, r.one);
    auto put = [&](T *to, const Values<T, VEC> &v) {
      Two o[kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j) o[j] = activate<ACT>(c.affine(j, c.xhat(j, v.pair(j))));
      Values<T, VEC>::store(to, o);
    };
    int left = (int)(stop - at) - row;
    const T *from = x + (at + row) * channels + first;
    T *to = y + (at + row) * channels + first;
    for (; left > (kUnroll - 1) * l.row_threads; left -= kUnroll * l.row_threads, from += kUnroll * step, to += kUnroll * step) {
      Values<T, VEC> v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u].load(from + u * step);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) put(to + u * step, v[u]);
    }
    for (; left > 0; left -= l.row_threads, from += step, to += step) {
      Values<T, VEC> v;
      v.load(from);
      put(to, v);
    }
  }, [&](int64_t at) {
    if (!active) return;
    for (int64_t i = at + row; i < end; i += l.row_threads) Values<T, VEC>::storeZero(y + i * channels + first);
  });
}

// Pass 1 backward: partial[slot][channel] = (sum du, sum du xhat) of the block's rows of a sample.
template <typename T, int VEC, int ACT, bool UNIFORM>
__global__ void __launch_bounds__(kThreads, 2)
gradSumsKernel(const T *dy, const T *x, const void *weight, const void *bias, bool float_affine, const float *mean,
               const float *rstd, Rows r, int channels, int groups, Lanes l, float2 *partial) {
  letNextKernelStart();
  extern __shared__ __align__(16) float2 scratch[];
  constexpr int kPairs = (VEC + 1) / 2;
  const int column = threadIdx.x % l.columns, row = threadIdx.x / l.columns;
  const int first0 = blockIdx.y * l.columns * VEC, first = first0 + column * VEC;
  const bool active = row < l.row_threads && first < channels;
  const int64_t begin = (int64_t)blockIdx.x * r.block_rows;
  const int64_t end = begin + r.block_rows < r.rows ? begin + r.block_rows : r.rows;
  const int64_t step = (int64_t)l.row_threads * channels;
  forSamples(r, begin, end, [&](int64_t at, int64_t stop, int64_t sample) {
    Two a[kPairs], b[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) a[j] = b[j] = two(0.0f, 0.0f);
    if (active) {
      Norm<VEC, UNIFORM> c;
      loadNorm<T>(c, mean + sample * groups, rstd + sample * groups, weight, bias, float_affine, first, channels / groups, r.one);
      auto add = [&](const Values<T, VEC> &v, const Values<T, VEC> &g) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const Two xh = c.xhat(j, v.pair(j));
          const Two du = activateGrad<ACT>(g.pair(j), c.affine(j, xh));
          a[j] = a[j] + du;
          b[j] = fma(du, xh, b[j]);
        }
      };
      int left = (int)(stop - at) - row;
      const int64_t offset = (at + row) * channels + first;
      const T *from = x + offset, *from_g = dy + offset;
      constexpr int kRows = kUnroll;
      for (; left > (kRows - 1) * l.row_threads; left -= kRows * l.row_threads, from += kRows * step, from_g += kRows * step) {
        Values<T, VEC> v[kRows], g[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          v[u].load(from + u * step);
          g[u].load(from_g + u * step);
        }
#pragma unroll
        for (int u = 0; u < kRows; ++u) add(v[u], g[u]);
      }
      for (; left > 0; left -= l.row_threads, from += step, from_g += step) {
        Values<T, VEC> v, g;
        v.load(from);
        g.load(from_g);
        add(v, g);
      }
    }
    float2 *out = partial + (blockIdx.x + sample) * channels + first0;
    joinRowThreads<VEC, kThreads>(a, b, l, scratch, PlainSums{}, [&](int c, double2 s, float2) {
      if (first0 + c < channels) out[c] = make_float2((float)s.x, (float)s.y);
    });
  }, [](int64_t) {});
}

// Pass 2 backward: one block per (sample, group): the sample's sums per channel, and the group's two means.
template <typename T>
__global__ void __launch_bounds__(kThreads)
joinGradSumsKernel(const float2 *partial, const void *weight, bool float_affine, Rows r, int channels, int groups,
                   float2 *sample_sums, float2 *group_means) {
  letNextKernelStart();
  __shared__ double2 scratch[kThreads / 32], lanes[kThreads];
  const int64_t sample = blockIdx.x / groups;
  const int group = blockIdx.x % groups, group_channels = channels / groups;
  const SampleSlots s(r, sample);
  // a tile of up to 32 channels side by side, the other threads along the slots
  const int width = group_channels < 32 ? group_channels : 32, depth = kThreads / width;
  const int c = threadIdx.x % width, d = threadIdx.x / width;
  double m1 = 0.0, m2 = 0.0;
  waitForKernelBefore();
  for (int base = 0; base < group_channels; base += width) {
    const int channel = group * group_channels + base + c;
    const bool active = d < depth && base + c < group_channels;
    double a = 0.0, b = 0.0;
    if (active) {
#pragma unroll 4
      for (int64_t k = s.first + d; k <= s.last; k += depth) {
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
      const double gamma = weight ? (double)loadAffine<T>(weight, float_affine, channel) : 1.0;
      m1 += gamma * a;
      m2 += gamma * b;
    }
  }
  const double2 sum = blockSum(m1, m2, scratch);
  if (threadIdx.x == 0) {
    const double n = s.end > s.begin ? (double)(s.end - s.begin) * group_channels : 1.0;
    group_means[blockIdx.x] = make_float2((float)(sum.x / n), (float)(sum.y / n));
  }
}

// Pass 3 backward: the input gradient; the first blocks also add the samples' sums to the affine gradients.
template <typename T, int VEC, int ACT, bool UNIFORM>
__global__ void __launch_bounds__(kThreads, 2)
inputGradKernel(const T *dy, const T *x, const void *weight, const void *bias, bool float_affine, const float *mean,
                const float *rstd, const float2 *sample_sums, const float2 *group_means, Rows r, int channels,
                int groups, Lanes l, T *dx, void *weight_grad, void *bias_grad, bool float_affine_grad) {
  constexpr int kPairs = (VEC + 1) / 2;
  const int column = threadIdx.x % l.columns, row = threadIdx.x / l.columns;
  const int first = (blockIdx.y * l.columns + column) * VEC, group_channels = channels / groups;
  const bool active = row < l.row_threads && first < channels;
  waitForKernelBefore();
  if (weight_grad) {
    const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int64_t all = (int64_t)gridDim.x * gridDim.y * kThreads;
    for (int64_t ch = block * kThreads + threadIdx.x; ch < channels; ch += all) {
      double a = 0.0, b = 0.0;
#pragma unroll 4
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
  const int64_t step = (int64_t)l.row_threads * channels;
  forSamples(r, begin, end, [&](int64_t at, int64_t stop, int64_t sample) {
    if (!active) return;
    Norm<VEC, UNIFORM> c;
    loadNorm<T>(c, mean + sample * groups, rstd + sample * groups, weight, bias, float_affine, first, group_channels, r.one);
    constexpr int kGroups = Norm<VEC, UNIFORM>::kGroups;
    Two minus_m1[kGroups], minus_m2[kGroups];
    const float2 *means = group_means + sample * groups;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
      minus_m1[j] = ofPair<UNIFORM ? 2 : VEC>(first, j, [&](int ch) { return -means[(UNIFORM ? first : ch) / group_channels].x; });
      minus_m2[j] = ofPair<UNIFORM ? 2 : VEC>(first, j, [&](int ch) { return -means[(UNIFORM ? first : ch) / group_channels].y; });
    }
    auto put = [&](T *to, const Values<T, VEC> &v, const Values<T, VEC> &g) {
      Two o[kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int q = UNIFORM ? 0 : j;
        const Two xh = c.xhat(j, v.pair(j));
        const Two du = activateGrad<ACT>(g.pair(j), c.affine(j, xh));
        o[j] = c.inputGrad(j, du, xh, minus_m1[q], minus_m2[q]) * c.rstd[q];
      }
      Values<T, VEC>::store(to, o);
    };
    int left = (int)(stop - at) - row;
    const int64_t offset = (at + row) * channels + first;
    const T *from = x + offset, *from_g = dy + offset;
    T *to = dx + offset;
    constexpr int kRows = kUnroll;
    for (; left > (kRows - 1) * l.row_threads; left -= kRows * l.row_threads, from += kRows * step, from_g += kRows * step, to += kRows * step) {
      Values<T, VEC> v[kRows], g[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        v[u].load(from + u * step);
        g[u].load(from_g + u * step);
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) put(to + u * step, v[u], g[u]);
    }
    for (; left > 0; left -= l.row_threads, from += step, from_g += step, to += step) {
      Values<T, VEC> v, g;
      v.load(from);
      g.load(from_g);
      put(to, v, g);
    }
  }, [&](int64_t at) {
    if (!active) return;
    for (int64_t i = at + row; i < end; i += l.row_threads) Values<T, VEC>::storeZero(dx + i * channels + first);
  });
}

// All three steps in one block: the slice of l.columns vectors from column blockIdx.y * l.columns on, of `chunk` samples
// one after the other.  Backward, `partial` (more chunks than one): a line of the affine gradients' sums for each chunk.
template <typename T, int VEC, int ACT, bool UNIFORM, bool BACKWARD>
__global__ void __launch_bounds__(kSmallThreads, 1)
sliceKernel(const T *dy, const T *x, const void *weight, const void *bias, bool float_affine, float *mean, float *rstd,
            Rows r, int channels, int groups, Lanes l, int64_t chunk, float epsilon, T *out, float2 *partial,
            void *weight_grad, void *bias_grad, bool float_affine_grad) {
  if (BACKWARD) letNextKernelStart();
  constexpr int kPairs = (VEC + 1) / 2, kGroups = UNIFORM ? 1 : kPairs;
  // joinRowThreads' scratch | the slice's channels (two doubles each) | its groups (two floats)
  extern __shared__ __align__(16) float2 scratch[];
  const int slice = l.columns * VEC, group_channels = channels / groups, slice_groups = slice / group_channels;
  double2 *sums = reinterpret_cast<double2 *>(scratch + joinBytes(VEC, kSmallThreads) / sizeof(float2));
  float2 *stats = reinterpret_cast<float2 *>(sums + slice);
  const int tid = threadIdx.x, row = tid / l.columns;
  const int first0 = blockIdx.y * slice, own = tid % l.columns * VEC, first = first0 + own;
  const int group0 = first0 / group_channels;
  const bool active = row < l.row_threads;
  const int64_t step = (int64_t)l.row_threads * channels;
  double total_a = 0.0, total_b = 0.0;  // backward: thread c < slice adds up channel c over the samples
  const int64_t s0 = blockIdx.x * chunk, s1 = s0 + chunk < r.samples ? s0 + chunk : r.samples;
  for (int64_t sample = s0; sample < s1; ++sample) {
    const int64_t begin = sampleStart(r, sample), end = sampleStart(r, sample + 1);
    const int rows = end > begin ? (int)(end - begin) : 0;
    const T *from0 = x + (begin + row) * channels + first;
    const T *grad0 = BACKWARD ? dy + (begin + row) * channels + first : from0;
    Two a[kPairs], b[kPairs], minus_k[kPairs];
    Norm<VEC, UNIFORM> c;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) a[j] = b[j] = minus_k[j] = two(0.0f, 0.0f);
    if (active && rows > 0) {
      if (BACKWARD) {
        loadNorm<T>(c, mean + sample * groups, rstd + sample * groups, weight, bias, float_affine, first, group_channels, r.one);
      } else if (row < rows) {
        Values<T, VEC> k;
        k.load(from0);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) minus_k[j] = k.pair(j) * two(-1.0f, -1.0f);
      }
      const T *from = from0, *grad = grad0;
#pragma unroll 2
      for (int i = row; i < rows; i += l.row_threads, from += step, grad += step) {
        Values<T, VEC> v, g;
        v.load(from);
        if (BACKWARD) g.load(grad);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          if (BACKWARD) {
            const Two xh = c.xhat(j, v.pair(j));
            const Two du = activateGrad<ACT>(g.pair(j), c.affine(j, xh));
            a[j] = a[j] + du;
            b[j] = fma(du, xh, b[j]);
          } else {
            const Two d = v.pair(j) + minus_k[j];
            a[j] = a[j] + d;
            b[j] = fma(d, d, b[j]);
          }
        }
      }
    }
    if (BACKWARD) {
      joinRowThreads<VEC, kSmallThreads>(a, b, l, scratch, PlainSums{}, [&](int ch, double2 v, float2) { sums[ch] = v; });
    } else if (rows > 0) {
      closeMoments<VEC>(a, b, minus_k, row < rows ? (rows - row + l.row_threads - 1) / l.row_threads : 0);
      joinMoments<VEC, kSmallThreads>(a, b, l, rows, scratch, [&](int ch, double m, double squares) { sums[ch] = make_double2(m, squares); });
    }
    __syncthreads();
    if (BACKWARD) {
      if (tid < slice) {  // (slice <= kSmallThreads)
        total_a += sums[tid].x;
        total_b += sums[tid].y;
      }
    }
    for (int q = tid; q < slice_groups; q += kSmallThreads) {
      double u = 0.0, w = 0.0, ref = 0.0;
      for (int i = 0; i < group_channels; ++i) {
        const int ch = q * group_channels + i;
        const double2 v = sums[ch];
        if (BACKWARD) {
          const double gamma = weight ? (double)loadAffine<T>(weight, float_affine, first0 + ch) : 1.0;
          u += gamma * v.x;
          w += gamma * v.y;
        } else if (rows > 0) {
          if (i == 0) ref = v.x;
          u += v.x - ref;
          w += v.y + rows * (v.x - ref) * (v.x - ref);
        }
      }
      const double n = (double)(rows > 0 ? rows : 1) * group_channels;
      if (BACKWARD) {
        stats[q] = make_float2((float)(u / n), (float)(w / n));
      } else {
        const double off = u / group_channels;
        double var = w / n - off * off;
        var = var < 0.0 ? 0.0 : var;
        const float m = (float)(ref + off), s = (float)(1.0 / sqrt(var + (double)epsilon));
        stats[q] = make_float2(m, s);
        mean[sample * groups + group0 + q] = m;
        rstd[sample * groups + group0 + q] = s;
      }
    }
    __syncthreads();
    if (active && rows > 0) {
      Two minus_m1[kGroups], minus_m2[kGroups];
      auto group = [&](int j, auto value) {
        return ofPair<UNIFORM ? 2 : VEC>(own, j, [&](int ch) { return value(stats[(UNIFORM ? own : ch) / group_channels]); });
      };
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        const Two first_stat = group(j, [](float2 v) { return -v.x; });
        if (BACKWARD) {
          minus_m1[j] = first_stat;
          minus_m2[j] = group(j, [](float2 v) { return -v.y; });
        } else {
          c.minus_mean[j] = first_stat;
          c.rstd[j] = group(j, [](float2 v) { return v.y; });
        }
      }
      if (!BACKWARD) {
        c.one = r.one;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          c.gamma[j] = ofPair<VEC>(first, j, [&](int ch) { return weight ? loadAffine<T>(weight, float_affine, ch) : 1.0f; });
          c.beta[j] = ofPair<VEC>(first, j, [&](int ch) { return bias ? loadAffine<T>(bias, float_affine, ch) : 0.0f; });
        }
      }
      const T *from = from0, *grad = grad0;
      T *to = out + (begin + row) * channels + first;
#pragma unroll 2
      for (int i = row; i < rows; i += l.row_threads, from += step, grad += step, to += step) {
        Values<T, VEC> v, g;
        v.load(from);
        if (BACKWARD) g.load(grad);
        Two o[kPairs];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const int q = UNIFORM ? 0 : j;
          const Two xh = c.xhat(j, v.pair(j));
          if (BACKWARD) {
            const Two du = activateGrad<ACT>(g.pair(j), c.affine(j, xh));
            o[j] = c.inputGrad(j, du, xh, minus_m1[q], minus_m2[q]) * c.rstd[q];
          } else {
            o[j] = activate<ACT>(c.affine(j, xh));
          }
        }
        Values<T, VEC>::store(to, o);
      }
    }
  }
  if (BACKWARD && weight_grad && tid < slice) {
    if (partial) {
      partial[(int64_t)blockIdx.x * channels + first0 + tid] = make_float2((float)total_a, (float)total_b);
    } else {
      storeAffineGrad<T>(bias_grad, float_affine_grad, first0 + tid, total_a);
      storeAffineGrad<T>(weight_grad, float_affine_grad, first0 + tid, total_b);
    }
  }
  if (active && blockIdx.x == 0) {  // rows of no sample
    const int64_t covered = sampleStart(r, r.samples);
    for (int64_t i = covered + row; i < r.rows; i += l.row_threads) Values<T, VEC>::storeZero(out + i * channels + first);
  }
}

// The affine gradients as sums over `lines` lines of (sum du, sum du xhat) per channel, in a fixed order: 32 channels
// side by side in a block, 32 threads along the lines.
template <typename T>
__global__ void __launch_bounds__(1024)
affineGradKernel(const float2 *sums, int64_t lines, int channels, void *weight_grad, void *bias_grad, bool float_affine_grad) {
  __shared__ double2 part[32][33];
  const int c = threadIdx.x % 32, d = threadIdx.x / 32, channel = blockIdx.x * 32 + c;
  double a = 0.0, b = 0.0;
  waitForKernelBefore();
  if (channel < channels) {
#pragma unroll 4
    for (int64_t k = d; k < lines; k += 32) {
      const float2 v = sums[k * channels + channel];
      a += v.x;
      b += v.y;
    }
  }
  part[d][c] = make_double2(a, b);
  __syncthreads();
  if (d == 0 && channel < channels) {
    for (int i = 1; i < 32; ++i) {
      a += part[i][c].x;
      b += part[i][c].y;
    }
    storeAffineGrad<T>(bias_grad, float_affine_grad, channel, a);
    storeAffineGrad<T>(weight_grad, float_affine_grad, channel, b);
  }
}

size_t roundUp(size_t v) { return (v + 255) / 256 * 256; }

Rows rowsOf(const NormProblem &p, const NormPlan &plan) {
  return Rows{p.rows, p.samples, p.sample_rows, plan.block_rows, p.sample_ends, 1.0f};
}

char *scratchBase(void *workspace) {
  return reinterpret_cast<char *>((reinterpret_cast<size_t>(workspace) + 255) / 256 * 256);
}

double rowBytes(const NormProblem &p) {
  return (double)p.rows * p.channels * mluop::getSizeOfDataType(p.dtype);
}

}  // namespace

namespace {

// More samples: their sums are added up by a kernel of its own.  Ragged samples of 64 half channels, gradients: 1,024 of 600
// rows 143 us with it and 244 us in the input gradient kernel, whose first blocks walk down the samples; 128 of 5,000 rows
// 101 and 98 us.
constexpr int kAffineSamples = 256;

// The one-launch form for samples of few rows: slices of `columns` vectors, `chunk` samples a block.  columns 0: it does
// not apply.  Its blocks read 32 bytes or so of a row, and the chained launches of the other form cost about 9 us together.
// Measured, half, forward and gradients: 2 samples of 128 rows of 128 channels 6.5 and 9.4 us against 9.5 and 9.9 us, 8 of
// 1,024 rows of 256 channels 9.5 and 11 us against 13.5 and 14 us, 2 of 2,048 rows of 128 channels 12 and 24 us against 10
// and 10 us.
struct SlicePlan {
  int columns;
  int64_t chunk, chunks;
};
SlicePlan planSlices(const NormProblem &p, int vec, bool backward) {
  SlicePlan plan{};
  if (p.samples == 0) return plan;
  const int group_channels = p.channels / p.groups;
  const int columns = std::lcm(group_channels, vec) / vec;
  if (columns * vec > kSmallThreads || p.channels % (columns * vec) != 0 || p.channels / (columns * vec) > 65535) return plan;
  // rows of one sample: where they are known on the device only, their average, and few in all, since one sample may have
  // them all
  const int64_t rows = p.ragged ? (p.rows + p.samples - 1) / p.samples : p.sample_rows;
  const int64_t turns = kSmallThreads / columns * (int64_t)kSmallTurns;
  if (rows > turns || (p.ragged && p.rows > 4 * turns)) return plan;
  // one round of blocks: 2,048 blocks for 256 samples of 64 rows of 128 channels took 74 us against 19 us for the three
  const int64_t slices = p.channels / (columns * vec), most = std::max<int64_t>(1, 2 * p.sm_count / slices);
  if (p.samples > most || (!p.ragged && rows <= kShortRows)) return plan;
  plan.columns = columns;
  // backward, two rows a thread in all: one block for all samples, which then writes the affine gradients
  plan.chunk = backward && p.samples <= 4 && p.rows <= turns / 2 ? p.samples : 1;
  plan.chunks = (p.samples + plan.chunk - 1) / plan.chunk;
  return plan;
}

template <typename T>
cudaError_t launchAffineGrad(const NormProblem &p, const float2 *sums, int64_t lines, void *weight_grad, void *bias_grad,
                             cudaStream_t stream) {
  trace::Scope scope("groupNormAffineGradKernel", stream);
  return launchAfterKernel(affineGradKernel<T>, dim3((unsigned)((p.channels + 31) / 32)), dim3(1024), 0, stream, sums, lines,
                           p.channels, weight_grad, bias_grad, p.float_affine_grad);
}

template <typename T, int VEC, bool UNIFORM, bool BACKWARD>
cudaError_t launchSlices(const NormProblem &p, const SlicePlan &plan, const void *output_grad, const void *input,
                         const void *weight, const void *bias, void *workspace, float *mean, float *rstd, void *out,
                         void *weight_grad, void *bias_grad, cudaStream_t stream) {
  const Lanes l{plan.columns, kSmallThreads / plan.columns};
  const int slice = plan.columns * VEC;
  const size_t smem = joinBytes(VEC, kSmallThreads) + slice * sizeof(double2) + slice / (p.channels / p.groups) * sizeof(float2);
  const dim3 grid((unsigned)plan.chunks, (unsigned)(p.channels / slice));
  float2 *partial = BACKWARD && weight_grad && plan.chunks > 1 ? reinterpret_cast<float2 *>(scratchBase(workspace)) : nullptr;
  auto kernel = p.activation == MLUOP_GROUP_NORM_ACT_RELU   ? sliceKernel<T, VEC, MLUOP_GROUP_NORM_ACT_RELU, UNIFORM, BACKWARD>
                : p.activation == MLUOP_GROUP_NORM_ACT_SILU ? sliceKernel<T, VEC, MLUOP_GROUP_NORM_ACT_SILU, UNIFORM, BACKWARD>
                                                            : sliceKernel<T, VEC, MLUOP_GROUP_NORM_ACT_NONE, UNIFORM, BACKWARD>;
  const Rows r{p.rows, p.samples, p.sample_rows, 0, p.sample_ends, 1.0f};
  {
    trace::Scope scope(BACKWARD ? "groupNormSliceKernel:backward" : "groupNormSliceKernel:forward", stream,
                       (BACKWARD ? 3 : 2) * rowBytes(p));
    kernel<<<grid, kSmallThreads, smem, stream>>>(static_cast<const T *>(output_grad), static_cast<const T *>(input), weight,
                                                  bias, p.float_affine, mean, rstd, r, p.channels, p.groups, l, plan.chunk,
                                                  p.epsilon, static_cast<T *>(out), partial, weight_grad, bias_grad,
                                                  p.float_affine_grad);
  }
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess || !partial) return err;
  return launchAffineGrad<T>(p, partial, plan.chunks, weight_grad, bias_grad, stream);
}

template <typename T, int VEC, bool UNIFORM>
cudaError_t forward(const NormProblem &p, const NormPlan &plan, const void *input, const void *weight,
                    const void *bias, void *workspace, void *output, float *mean, float *rstd, cudaStream_t stream) {
  char *base = scratchBase(workspace);
  float2 *partial = reinterpret_cast<float2 *>(base + plan.partial);
  const T *x = static_cast<const T *>(input);
  T *y = static_cast<T *>(output);
  const Rows r = rowsOf(p, plan);
  const Lanes l{plan.column_threads, plan.row_threads};
  const dim3 grid((unsigned)plan.blocks, (unsigned)plan.column_tiles);
  const size_t smem = joinBytes(VEC, kThreads);
  {
    trace::Scope scope("groupNormStatisticsKernel", stream, rowBytes(p));
    statisticsKernel<T, VEC><<<grid, kThreads, smem, stream>>>(x, r, p.channels, l, partial);
  }
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  if (p.samples > 0) {
    trace::Scope scope("groupNormJoinKernel", stream);
    err = launchAfterKernel(joinStatisticsKernel, dim3((unsigned)(p.samples * p.groups)), dim3(kThreads), 0, stream, partial,
                            r, p.channels, p.groups, p.epsilon, mean, rstd);
  }
  if (err != cudaSuccess) return err;
  trace::Scope scope("groupNormNormaliseKernel", stream, 2 * rowBytes(p));
  auto kernel = p.activation == MLUOP_GROUP_NORM_ACT_RELU   ? normaliseKernel<T, VEC, MLUOP_GROUP_NORM_ACT_RELU, UNIFORM>
                : p.activation == MLUOP_GROUP_NORM_ACT_SILU ? normaliseKernel<T, VEC, MLUOP_GROUP_NORM_ACT_SILU, UNIFORM>
                                                            : normaliseKernel<T, VEC, MLUOP_GROUP_NORM_ACT_NONE, UNIFORM>;
  return launchAfterKernel(kernel, grid, dim3(kThreads), 0, stream, x, weight, bias, p.float_affine, mean, rstd, r,
                           p.channels, p.groups, l, y);
}

template <typename T, int VEC, bool UNIFORM, int ACT>
cudaError_t backward(const NormProblem &p, const NormPlan &plan, const void *output_grad, const void *input,
                     const void *weight, const void *bias, const float *mean, const float *rstd, void *workspace,
                     void *input_grad, void *weight_grad, void *bias_grad, cudaStream_t stream) {
  char *base = scratchBase(workspace);
  float2 *partial = reinterpret_cast<float2 *>(base + plan.partial);
  float2 *sample_sums = reinterpret_cast<float2 *>(base + plan.sample_sums);
  float2 *group_means = reinterpret_cast<float2 *>(base + plan.group_means);
  const T *dy = static_cast<const T *>(output_grad), *x = static_cast<const T *>(input);
  const Rows r = rowsOf(p, plan);
  const Lanes l{plan.column_threads, plan.row_threads};
  const dim3 grid((unsigned)plan.blocks, (unsigned)plan.column_tiles);
  const size_t smem = joinBytes(VEC, kThreads);
  {
    trace::Scope scope("groupNormGradSumsKernel", stream, 2 * rowBytes(p));
    gradSumsKernel<T, VEC, ACT, UNIFORM><<<grid, kThreads, smem, stream>>>(dy, x, weight, bias, p.float_affine, mean, rstd,
                                                                           r, p.channels, p.groups, l, partial);
  }
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  if (p.samples > 0) {
    trace::Scope scope("groupNormGradJoinKernel", stream);
    err = launchAfterKernel(joinGradSumsKernel<T>, dim3((unsigned)(p.samples * p.groups)), dim3(kThreads), 0, stream, partial,
                            weight, p.float_affine, r, p.channels, p.groups, sample_sums, group_means);
  }
  if (err != cudaSuccess) return err;
  const bool many = weight_grad && p.samples > kAffineSamples;
  {
    trace::Scope scope("groupNormInputGradKernel", stream, 3 * rowBytes(p));
    void *none = nullptr;
    err = launchAfterKernel(inputGradKernel<T, VEC, ACT, UNIFORM>, grid, dim3(kThreads), 0, stream, dy, x, weight, bias,
                            p.float_affine, mean, rstd, sample_sums, group_means, r, p.channels, p.groups, l,
                            static_cast<T *>(input_grad), many ? none : weight_grad, many ? none : bias_grad,
                            p.float_affine_grad);
  }
  if (err != cudaSuccess || !many) return err;
  return launchAffineGrad<T>(p, sample_sums, p.samples, weight_grad, bias_grad, stream);
}

template <typename T, int VEC, bool UNIFORM, typename... Args>
cudaError_t backwardAct(const NormProblem &p, Args... args) {
  switch (p.activation) {
    case MLUOP_GROUP_NORM_ACT_RELU: return backward<T, VEC, UNIFORM, MLUOP_GROUP_NORM_ACT_RELU>(p, args...);
    case MLUOP_GROUP_NORM_ACT_SILU: return backward<T, VEC, UNIFORM, MLUOP_GROUP_NORM_ACT_SILU>(p, args...);
    default: return backward<T, VEC, UNIFORM, MLUOP_GROUP_NORM_ACT_NONE>(p, args...);
  }
}

// Vectors of 16 bytes whose channels lie in one group, such vectors across groups, or single values.
template <typename T, int VEC, typename... Args>
cudaError_t forwardType(const NormProblem &p, const NormPlan &plan, Args... args) {
  if (plan.vec == 1) return forward<T, 1, true>(p, plan, args...);
  return p.channels / p.groups % VEC == 0 ? forward<T, VEC, true>(p, plan, args...) : forward<T, VEC, false>(p, plan, args...);
}
template <typename T, int VEC, typename... Args>
cudaError_t backwardType(const NormProblem &p, const NormPlan &plan, Args... args) {
  if (plan.vec == 1) return backwardAct<T, 1, true>(p, plan, args...);
  return p.channels / p.groups % VEC == 0 ? backwardAct<T, VEC, true>(p, plan, args...)
                                          : backwardAct<T, VEC, false>(p, plan, args...);
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
  // as many blocks as run at a time (four to an SM forward, two backward), so that each has long runs of rows, and at
  // least one unrolled turn for each block
  const int64_t wanted = std::max<int64_t>(1, (int64_t)(backward ? 2 : 4) * p.sm_count / plan.column_tiles);
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
  // whichever way the tensors are aligned
  auto bytes = [&](int vec) -> size_t {
    if (const SlicePlan plan = planSlices(p, vec, backward); plan.columns)
      return backward && plan.chunks > 1 ? (size_t)plan.chunks * p.channels * sizeof(float2) + 256 : 0;
    if (const ShortPlan plan = planShort(p, vec); plan.lanes)
      return backward ? (size_t)plan.blocks * p.channels * sizeof(float2) + 256 : 0;
    return planNorm(p, backward, vec > 1).total;
  };
  const int wide = 16 / (int)mluop::getSizeOfDataType(p.dtype);
  return p.channels % wide != 0 ? bytes(1) : std::max(bytes(1), bytes(wide));
}

namespace {

template <typename T, int VEC>
cudaError_t runForward(const NormProblem &p, const void *input, const void *weight, const void *bias, void *workspace,
                       void *output, float *mean, float *rstd, cudaStream_t stream) {
  const NormPlan plan = planNorm(p, false, aligned16(input) && aligned16(output));
  if (const SlicePlan slices = planSlices(p, plan.vec, false); slices.columns) {
    auto launch = plan.vec == 1                        ? launchSlices<T, 1, true, false>
                  : p.channels / p.groups % VEC == 0 ? launchSlices<T, VEC, true, false>
                                                     : launchSlices<T, VEC, false, false>;
    return launch(p, slices, nullptr, input, weight, bias, workspace, mean, rstd, output, nullptr, nullptr, stream);
  }
  if (const ShortPlan few = planShort(p, plan.vec); few.lanes)
    return launchShortForward(p, few, input, weight, bias, output, mean, rstd, stream);
  return forwardType<T, VEC>(p, plan, input, weight, bias, workspace, output, mean, rstd, stream);
}

template <typename T, int VEC>
cudaError_t runBackward(const NormProblem &p, const void *output_grad, const void *input, const void *weight,
                        const void *bias, const float *mean, const float *rstd, void *workspace, void *input_grad,
                        void *weight_grad, void *bias_grad, cudaStream_t stream) {
  const NormPlan plan = planNorm(p, true, aligned16(output_grad) && aligned16(input) && aligned16(input_grad));
  if (const SlicePlan slices = planSlices(p, plan.vec, true); slices.columns) {
    auto launch = plan.vec == 1                        ? launchSlices<T, 1, true, true>
                  : p.channels / p.groups % VEC == 0 ? launchSlices<T, VEC, true, true>
                                                     : launchSlices<T, VEC, false, true>;
    return launch(p, slices, output_grad, input, weight, bias, workspace, const_cast<float *>(mean), const_cast<float *>(rstd),
                  input_grad, weight_grad, bias_grad, stream);
  }
  if (const ShortPlan few = planShort(p, plan.vec); few.lanes) {
    float2 *partial = weight_grad ? reinterpret_cast<float2 *>(scratchBase(workspace)) : nullptr;
    const cudaError_t err = launchShortBackward(p, few, output_grad, input, weight, bias, mean, rstd, partial, input_grad, stream);
    return err != cudaSuccess || !partial ? err
                                          : launchAffineGrad<T>(p, partial, few.blocks, weight_grad, bias_grad, stream);
  }
  return backwardType<T, VEC>(p, plan, output_grad, input, weight, bias, mean, rstd, workspace, input_grad, weight_grad,
                              bias_grad, stream);
}

}  // namespace

cudaError_t launchNormForward(const NormProblem &p, const void *input, const void *weight, const void *bias,
                              void *workspace, void *output, float *mean, float *rstd, cudaStream_t stream) {
  auto run = p.dtype == MLUOP_DTYPE_FLOAT ? runForward<float, 4>
             : p.dtype == MLUOP_DTYPE_HALF ? runForward<__half, 8>
                                           : runForward<__nv_bfloat16, 8>;
  return run(p, input, weight, bias, workspace, output, mean, rstd, stream);
}

cudaError_t launchNormBackward(const NormProblem &p, const void *output_grad, const void *input, const void *weight,
                               const void *bias, const float *mean, const float *rstd, void *workspace,
                               void *input_grad, void *weight_grad, void *bias_grad, cudaStream_t stream) {
  auto run = p.dtype == MLUOP_DTYPE_FLOAT ? runBackward<float, 4>
             : p.dtype == MLUOP_DTYPE_HALF ? runBackward<__half, 8>
                                           : runBackward<__nv_bfloat16, 8>;
  return run(p, output_grad, input, weight, bias, mean, rstd, workspace, input_grad, weight_grad, bias_grad, stream);
}

}  // namespace group_norm_act
}  // namespace mluop
