// Launch interface of the AdamW step over many tensors.
#ifndef MLUOP_B200_KERNELS_MULTI_TENSOR_ADAMW_KERNELS_H_
#define MLUOP_B200_KERNELS_MULTI_TENSOR_ADAMW_KERNELS_H_

#include <cuda_runtime_api.h>

#include <cstdint>

#include "mlu_op.h"

namespace mluop {
namespace multi_tensor_adamw {

constexpr int64_t kScaleBlock = 256;  // consecutive elements that share a scale in an 8-bit state

struct AdamWProblem {
  mluOpDataType_t param_dtype, grad_dtype;
  bool state_8bit;
  int64_t tensor_num;
  const int64_t *element_num;
  void *const *param;
  const void *const *grad;
  void *const *exp_avg, *const *exp_avg_sq;
  float *const *exp_avg_scale, *const *exp_avg_sq_scale;
  double lr, beta1, beta2, epsilon, weight_decay;
  int64_t step;
  const float *grad_scale, *schedule;
  int sm_count;
  bool stochastic;  // rounding of 8-bit states
  const int64_t *step_count;
};

cudaError_t launchMultiTensorAdamW(const AdamWProblem &p, cudaStream_t stream);

}  // namespace multi_tensor_adamw
}  // namespace mluop

#endif  // MLUOP_B200_KERNELS_MULTI_TENSOR_ADAMW_KERNELS_H_
