// mluOpMultiTensorAdamW and mluOpMultiTensorAdamW_v2: argument checks and dispatch.  No counterpart in the
// reference with this shape (its kernels/adamw updates one tensor with float states).
#include <cuda_runtime_api.h>

#include <cmath>
#include <string>

#include "core/context.h"
#include "core/logging.h"
#include "core/type.h"
#include "kernels/multi_tensor_adamw/multi_tensor_adamw_kernels.h"

namespace {

bool isParamType(mluOpDataType_t t) {
  return t == MLUOP_DTYPE_HALF || t == MLUOP_DTYPE_BFLOAT16 || t == MLUOP_DTYPE_FLOAT;
}

bool aligned(const void *p, size_t to) { return reinterpret_cast<size_t>(p) % to == 0; }

mluOpStatus_t runStep(const std::string &api, mluOpHandle_t handle, const mluOpDataType_t param_dtype,
                      const mluOpDataType_t grad_dtype, const mluOpDataType_t state_dtype, const int64_t tensor_num,
                      const int64_t element_num[], void *const param[], const void *const grad[],
                      void *const exp_avg[], void *const exp_avg_sq[], float *const exp_avg_scale[],
                      float *const exp_avg_sq_scale[], const double lr, const double beta1, const double beta2,
                      const double epsilon, const double weight_decay, const int64_t step, const float *grad_scale,
                      const float *schedule, const mluOpAdamWRounding_t rounding, const int64_t *step_count) {
  PARAM_CHECK(api, handle != nullptr);
  if (handle->arch < MLUOP_MLU370) {
    LOG(ERROR) << api << " needs a compute-capability 10.x device; this handle's device is not one.";
    return MLUOP_STATUS_ARCH_MISMATCH;
  }
  PARAM_CHECK(api, isParamType(param_dtype));
  PARAM_CHECK(api, grad_dtype == param_dtype || grad_dtype == MLUOP_DTYPE_FLOAT);
  PARAM_CHECK(api, state_dtype == MLUOP_DTYPE_FLOAT || state_dtype == MLUOP_DTYPE_UINT8);
  PARAM_CHECK(api, tensor_num >= 0);
  PARAM_CHECK(api, std::isfinite(lr) && lr >= 0.0);
  PARAM_CHECK(api, beta1 >= 0.0 && beta1 < 1.0);
  PARAM_CHECK(api, beta2 >= 0.0 && beta2 < 1.0);
  PARAM_CHECK(api, std::isfinite(epsilon) && epsilon >= 0.0);
  PARAM_CHECK(api, std::isfinite(weight_decay) && weight_decay >= 0.0);
  PARAM_CHECK(api, step >= 1);
  PARAM_CHECK(api, aligned(grad_scale, 4));
  PARAM_CHECK(api, aligned(schedule, 4));
  PARAM_CHECK(api, aligned(step_count, 8));
  PARAM_CHECK(api, rounding == MLUOP_ADAMW_ROUND_NEAREST || rounding == MLUOP_ADAMW_ROUND_STOCHASTIC);
  const bool stochastic = rounding == MLUOP_ADAMW_ROUND_STOCHASTIC && state_dtype == MLUOP_DTYPE_UINT8;
  PARAM_CHECK(api, !stochastic || schedule == nullptr || step_count != nullptr);
  if (tensor_num == 0) {
    VLOG(5) << api << " no tensors.";
    return MLUOP_STATUS_SUCCESS;
  }
  PARAM_CHECK(api, element_num != nullptr);
  PARAM_CHECK(api, param != nullptr);
  PARAM_CHECK(api, grad != nullptr);
  PARAM_CHECK(api, exp_avg != nullptr);
  PARAM_CHECK(api, exp_avg_sq != nullptr);
  const bool state_8bit = state_dtype == MLUOP_DTYPE_UINT8;
  PARAM_CHECK(api, (exp_avg_scale != nullptr) == state_8bit);
  PARAM_CHECK(api, (exp_avg_sq_scale != nullptr) == state_8bit);
  const size_t param_size = mluop::getSizeOfDataType(param_dtype), grad_size = mluop::getSizeOfDataType(grad_dtype);
  const size_t state_size = state_8bit ? 1 : 4;
  bool any = false;
  for (int64_t i = 0; i < tensor_num; ++i) {
    PARAM_CHECK(api, element_num[i] >= 0 && element_num[i] <= (int64_t(1) << 40));
    if (element_num[i] == 0) continue;
    any = true;
    PARAM_CHECK(api, param[i] != nullptr && aligned(param[i], param_size));
    PARAM_CHECK(api, grad[i] != nullptr && aligned(grad[i], grad_size));
    PARAM_CHECK(api, exp_avg[i] != nullptr && aligned(exp_avg[i], state_size));
    PARAM_CHECK(api, exp_avg_sq[i] != nullptr && aligned(exp_avg_sq[i], state_size));
    if (state_8bit) {
      PARAM_CHECK(api, exp_avg_scale[i] != nullptr && aligned(exp_avg_scale[i], 4));
      PARAM_CHECK(api, exp_avg_sq_scale[i] != nullptr && aligned(exp_avg_sq_scale[i], 4));
    }
  }
  if (!any) {
    VLOG(5) << api << " Skip zero element tensors.";
    return MLUOP_STATUS_SUCCESS;
  }
  if (handle->host_only) {
    LOG(ERROR) << api << " this handle was created without a CUDA device; nothing can be launched.";
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  mluop::DeviceGuard guard(handle);
  mluop::multi_tensor_adamw::AdamWProblem p{param_dtype, grad_dtype,    state_8bit,       tensor_num, element_num,
                                            param,       grad,          exp_avg,          exp_avg_sq, exp_avg_scale,
                                            exp_avg_sq_scale, lr,       beta1,            beta2,      epsilon,
                                            weight_decay, step,         grad_scale,       schedule, handle->sm_count,
                                            stochastic,   step_count};
  const cudaError_t err = mluop::multi_tensor_adamw::launchMultiTensorAdamW(p, handle->queue);
  if (err != cudaSuccess) {
    LOG(ERROR) << api << " launch failed: " << cudaGetErrorString(err);
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  return MLUOP_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

mluOpStatus_t MLUOP_WIN_API mluOpMultiTensorAdamW(
    mluOpHandle_t handle, const mluOpDataType_t param_dtype, const mluOpDataType_t grad_dtype,
    const mluOpDataType_t state_dtype, const int64_t tensor_num, const int64_t element_num[], void *const param[],
    const void *const grad[], void *const exp_avg[], void *const exp_avg_sq[], float *const exp_avg_scale[],
    float *const exp_avg_sq_scale[], const double lr, const double beta1, const double beta2, const double epsilon,
    const double weight_decay, const int64_t step, const float *grad_scale, const float *schedule) {
  return runStep("[mluOpMultiTensorAdamW]", handle, param_dtype, grad_dtype, state_dtype, tensor_num, element_num,
                 param, grad, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, lr, beta1, beta2, epsilon,
                 weight_decay, step, grad_scale, schedule, MLUOP_ADAMW_ROUND_NEAREST, nullptr);
}

mluOpStatus_t MLUOP_WIN_API mluOpMultiTensorAdamW_v2(
    mluOpHandle_t handle, const mluOpDataType_t param_dtype, const mluOpDataType_t grad_dtype,
    const mluOpDataType_t state_dtype, const int64_t tensor_num, const int64_t element_num[], void *const param[],
    const void *const grad[], void *const exp_avg[], void *const exp_avg_sq[], float *const exp_avg_scale[],
    float *const exp_avg_sq_scale[], const double lr, const double beta1, const double beta2, const double epsilon,
    const double weight_decay, const int64_t step, const float *grad_scale, const float *schedule,
    const mluOpAdamWRounding_t rounding, const int64_t *step_count) {
  return runStep("[mluOpMultiTensorAdamW_v2]", handle, param_dtype, grad_dtype, state_dtype, tensor_num, element_num,
                 param, grad, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, lr, beta1, beta2, epsilon,
                 weight_decay, step, grad_scale, schedule, rounding, step_count);
}

}  // extern "C"
