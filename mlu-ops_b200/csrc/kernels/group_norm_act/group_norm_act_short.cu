// Group norm of samples of very few rows, all of one size (rows that are samples of their own, say): a few lanes of a
// warp take a (sample, group), a vector of VEC channels each (K of them where a group is wider than a warp), and walk
// down its rows once for each sum and once for the outputs; all but the first walk hit L1.  A thread keeps its group and
// its channels from sample to sample, so that the affine gradients gather in registers.
//
// Bound by latency: the walks follow one another, with a join over the lanes, in double, between them.  Samples of one row
// of 128 half channels in 8 groups, forward and gradients: 16,384 of them 6 and 12 us (the three launches 741 and 676 us),
// 100,000 of them 23 and 35 us, 2.3 and 2.2 TB/s.  100,000 rows of 64 channels in 32 groups, single values: 54 and 52 us.
#include <cuda_runtime.h>

#include <algorithm>

#include "core/launch.cuh"
#include "core/trace.h"
#include "core/type.h"
#include "kernels/group_norm_act/group_norm_act_device.cuh"
#include "kernels/group_norm_act/group_norm_act_kernels.h"

namespace mluop {
namespace group_norm_act {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double2 laneSum(double a, double b, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_double2(a, b);
}
// The values of a pair as one: VEC 1 has no second one.
template <int VEC>
__device__ __forceinline__ double both(Two t) {
  const float2 f = split(t);
  return VEC > 1 ? (double)f.x + f.y : (double)f.x;
}

template <typename T, int VEC, int K, int ACT, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, K > 1 ? 1 : 3)
shortSamplesKernel(const T *dy, const T *x, const void *weight, const void *bias, bool float_affine, float *mean, float *rstd,
                   int64_t samples, int rows, int channels, int groups, ShortPlan l, float epsilon, float one, T *out,
                   float2 *partial) {
  if (BACKWARD) letNextKernelStart();
  constexpr int kPairs = (VEC + 1) / 2;
  extern __shared__ __align__(16) float2 scratch[];
  const int unit = threadIdx.x / l.lanes, lane = threadIdx.x % l.lanes, local_sample = unit / l.groups_block;
  const int group = blockIdx.y * l.groups_block + unit % l.groups_block, group_channels = channels / groups;
  const bool mine = local_sample < l.samples_block && group < groups;
  const int pitch = l.lanes * VEC;  // between a lane's vectors
  const int first = mine ? group * group_channels + lane * VEC : 0;
  const double inverse_n = 1.0 / ((double)rows * group_channels);
  const Two zero = two(0.0f, 0.0f);
  Norm<VEC, true> c[K];  // gamma and beta of each vector; mean and rstd in the first one
  Two a[K][kPairs], b[K][kPairs];
  bool has[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    has[k] = mine && lane * VEC + k * pitch < group_channels;
    const int at = has[k] ? first + k * pitch : 0;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      c[k].gamma[j] = ofPair<VEC>(at, j, [&](int ch) { return weight ? loadAffine<T>(weight, float_affine, ch) : 1.0f; });
      c[k].beta[j] = ofPair<VEC>(at, j, [&](int ch) { return bias ? loadAffine<T>(bias, float_affine, ch) : 0.0f; });
      a[k][j] = b[k][j] = zero;
    }
    c[k].one = one;
  }
  for (int64_t s0 = (int64_t)blockIdx.x * l.samples_block; s0 < samples; s0 += (int64_t)gridDim.x * l.samples_block) {
    const int64_t sample = s0 + local_sample, pair = sample * groups + group;
    const int count = mine && sample < samples ? rows : 0;
    const int64_t offset = count ? sample * rows * channels + first : 0;
    const T *from = x + offset, *grad = BACKWARD ? dy + offset : from;
    T *to = out + offset;
    float m = 0.0f, r = 0.0f;
    Two u = zero, w = zero, minus_m1 = zero, minus_m2 = zero;
    auto setNorm = [&] {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        c[k].minus_mean[0] = two(-m, -m);
        c[k].rstd[0] = two(r, r);
      }
    };
    // body(vector, row's offset) for what the lane has of the rows
    auto walk = [&](auto body) {
#pragma unroll 2
      for (int i = 0; i < count; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (has[k]) body(k, (int64_t)i * channels + k * pitch);
      }
    };
    if (BACKWARD) {
      if (count) {
        m = mean[pair];
        r = rstd[pair];
      }
      setNorm();
      walk([&](int k, int64_t at) {
        Values<T, VEC> v, g;
        v.load(from + at);
        g.load(grad + at);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const Two xh = c[k].xhat(0, v.pair(j)), du = activateGrad<ACT>(g.pair(j), c[k].affine(j, xh)), dx = du * c[k].gamma[j];
          a[k][j] = a[k][j] + du;
          b[k][j] = fma(du, xh, b[k][j]);
          u = u + dx;
          w = fma(dx, xh, w);
        }
      });
      const double2 sum = laneSum(both<VEC>(u), both<VEC>(w), l.lanes);
      const float m1 = (float)(sum.x * inverse_n), m2 = (float)(sum.y * inverse_n);
      minus_m1 = two(-m1, -m1);
      minus_m2 = two(-m2, -m2);
    } else {
      walk([&](int, int64_t at) {
        Values<T, VEC> v;
        v.load(from + at);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) u = u + v.pair(j);
      });
      // squares about the mean as the first walk gives it; their sum corrects both
      const float near = (float)(laneSum(both<VEC>(u), 0.0, l.lanes).x * inverse_n);
      const Two minus_near = two(-near, -near);
      u = zero;
      walk([&](int, int64_t at) {
        Values<T, VEC> v;
        v.load(from + at);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const Two d = v.pair(j) + minus_near;
          u = u + d;
          w = fma(d, d, w);
        }
      });
      const double2 sum = laneSum(both<VEC>(u), both<VEC>(w), l.lanes);
      const double off = sum.x * inverse_n;
      double var = sum.y * inverse_n - off * off;
      var = var < 0.0 ? 0.0 : var;  // (NaN stays)
      m = (float)(near + off);
      r = __frcp_rn(__fsqrt_rn((float)(var + (double)epsilon)));  // (three roundings; the same in double takes a quarter of the time)
      setNorm();
      if (count && lane == 0) {
        mean[pair] = m;
        rstd[pair] = r;
      }
    }
    walk([&](int k, int64_t at) {
      Values<T, VEC> v, g;
      v.load(from + at);
      if (BACKWARD) g.load(grad + at);
      Two o[kPairs];
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const Two xh = c[k].xhat(0, v.pair(j));
        if (BACKWARD) {
          const Two du = activateGrad<ACT>(g.pair(j), c[k].affine(j, xh));
          o[j] = c[k].inputGrad(j, du, xh, minus_m1, minus_m2) * c[k].rstd[0];
        } else {
          o[j] = activate<ACT>(c[k].affine(j, xh));
        }
      }
      Values<T, VEC>::store(to + at, o);
    });
  }
  if (BACKWARD && partial) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      joinRowThreads<VEC, kThreads>(a[k], b[k], Lanes{l.groups_block * l.lanes, l.samples_block}, scratch, PlainSums{},
                                    [&](int at, double2 s, float2) {
        const int own = at % pitch + k * pitch, g = blockIdx.y * l.groups_block + at / pitch;
        if (own < group_channels && g < groups)
          partial[(int64_t)blockIdx.x * channels + g * group_channels + own] = make_float2((float)s.x, (float)s.y);
      });
  }
}

template <typename T, int VEC, int K, bool BACKWARD>
cudaError_t launch(const NormProblem &p, const ShortPlan &plan, const void *output_grad, const void *input, const void *weight,
                   const void *bias, float *mean, float *rstd, float2 *partial, void *out, cudaStream_t stream) {
  auto kernel = p.activation == MLUOP_GROUP_NORM_ACT_RELU   ? shortSamplesKernel<T, VEC, K, MLUOP_GROUP_NORM_ACT_RELU, BACKWARD>
                : p.activation == MLUOP_GROUP_NORM_ACT_SILU ? shortSamplesKernel<T, VEC, K, MLUOP_GROUP_NORM_ACT_SILU, BACKWARD>
                                                            : shortSamplesKernel<T, VEC, K, MLUOP_GROUP_NORM_ACT_NONE, BACKWARD>;
  trace::Scope scope(BACKWARD ? "groupNormShortSamplesKernel:backward" : "groupNormShortSamplesKernel:forward", stream,
                     (BACKWARD ? 3.0 : 2.0) * p.rows * p.channels * sizeof(T));
  kernel<<<dim3((unsigned)plan.blocks, (unsigned)plan.tiles), kThreads, BACKWARD ? joinBytes(VEC, kThreads) : 0, stream>>>(
      static_cast<const T *>(output_grad), static_cast<const T *>(input), weight, bias, p.float_affine, mean, rstd, p.samples,
      (int)p.sample_rows, p.channels, p.groups, plan, p.epsilon, 1.0f, static_cast<T *>(out), partial);
  return cudaGetLastError();
}

template <typename T, int VEC, bool BACKWARD, typename... Args>
cudaError_t launchType(const NormProblem &p, const ShortPlan &plan, Args... args) {
  if (plan.vec == 1) return plan.vectors == 1 ? launch<T, 1, 1, BACKWARD>(p, plan, args...) : launch<T, 1, 4, BACKWARD>(p, plan, args...);
  return plan.vectors == 1 ? launch<T, VEC, 1, BACKWARD>(p, plan, args...) : launch<T, VEC, 4, BACKWARD>(p, plan, args...);
}
template <bool BACKWARD, typename... Args>
cudaError_t dispatch(const NormProblem &p, Args... args) {
  switch (p.dtype) {
    case MLUOP_DTYPE_FLOAT: return launchType<float, 4, BACKWARD>(p, args...);
    case MLUOP_DTYPE_HALF: return launchType<__half, 8, BACKWARD>(p, args...);
    default: return launchType<__nv_bfloat16, 8, BACKWARD>(p, args...);
  }
}

}  // namespace

// A lane walks down its rows one after the other, which takes about 0.6 us a row forward and 0.9 us backward until the
// samples fill the SMs; the three launches take about 15 us and 1 us for each sample that a block has.  Measured, forward
// and gradients: 512 samples of 24 rows of 64 channels 12 and 26 us against 41 and 40 us, 1,024 of 64 rows of 128 channels
// 43 and 62 us against 55 and 60 us, 256 of those 42 and 60 us against 19 and 21 us; 4 samples of 8 rows 4 and 9 us
// against 17 and 17 us.
ShortPlan planShort(const NormProblem &p, int vec) {
  ShortPlan plan{};
  const int group_channels = p.channels / p.groups;
  if (p.ragged || p.samples == 0 || p.sample_rows < 1 || p.sample_rows > kMostShortRows) return plan;
  if (p.sample_rows > kShortRows && p.samples < p.sample_rows * p.sample_rows / 4) return plan;
  plan.vec = group_channels % vec == 0 ? vec : 1;
  int lanes = 1;
  while (lanes < 32 && lanes * plan.vec < group_channels) lanes *= 2;
  plan.vectors = (group_channels + lanes * plan.vec - 1) / (lanes * plan.vec);
  if (plan.vectors > 4) return plan;
  plan.groups_block = std::min(p.groups, kThreads / lanes);
  plan.samples_block = kThreads / lanes / plan.groups_block;
  plan.tiles = (p.groups + plan.groups_block - 1) / plan.groups_block;
  const int64_t wanted = std::max<int64_t>(1, (int64_t)(plan.vectors > 1 ? 1 : 3) * p.sm_count / plan.tiles);
  plan.blocks = std::min<int64_t>(wanted, (p.samples + plan.samples_block - 1) / plan.samples_block);
  plan.lanes = lanes;
  return plan;
}

cudaError_t launchShortForward(const NormProblem &p, const ShortPlan &plan, const void *input, const void *weight,
                               const void *bias, void *output, float *mean, float *rstd, cudaStream_t stream) {
  return dispatch<false>(p, plan, nullptr, input, weight, bias, mean, rstd, nullptr, output, stream);
}
cudaError_t launchShortBackward(const NormProblem &p, const ShortPlan &plan, const void *output_grad, const void *input,
                                const void *weight, const void *bias, const float *mean, const float *rstd, float2 *partial,
                                void *input_grad, cudaStream_t stream) {
  return dispatch<true>(p, plan, output_grad, input, weight, bias, const_cast<float *>(mean), const_cast<float *>(rstd), partial,
                        input_grad, stream);
}

}  // namespace group_norm_act
}  // namespace mluop
