// mluOpGroupNormActForward / mluOpGroupNormActBackward and their workspace queries:
// argument checks and dispatch.  No counterpart in the reference.
#include <cuda_runtime_api.h>

#include <cmath>
#include <string>

#include "core/context.h"
#include "core/logging.h"
#include "core/overlap.h"
#include "core/tensor.h"
#include "kernels/group_norm_act/group_norm_act_kernels.h"

using mluop::Span;
using mluop::group_norm_act::NormProblem;

namespace {

constexpr int64_t kMaxChannels = 65536;

bool isRowType(mluOpDataType_t t) {
  return t == MLUOP_DTYPE_HALF || t == MLUOP_DTYPE_BFLOAT16 || t == MLUOP_DTYPE_FLOAT;
}

bool aligned(const void *p, size_t to) { return reinterpret_cast<size_t>(p) % to == 0; }

// In place, or nowhere on the other tensor.
bool sameOrApart(const void *a, const void *b, size_t bytes) { return a == b || !mluop::overlap(a, bytes, b, bytes); }

bool sameDims(const mluOpTensorDescriptor_t a, const mluOpTensorDescriptor_t b) {
  if (a->getDim() != b->getDim()) return false;
  for (int i = 0; i < a->getDim(); ++i)
    if (a->getDimIndex(i) != b->getDimIndex(i)) return false;
  return true;
}

// The rows, samples and channels that the descriptors describe.
mluOpStatus_t makeProblem(const std::string &api, mluOpHandle_t handle, const mluOpTensorDescriptor_t input_desc,
                          const mluOpTensorDescriptor_t sample_ends_desc, int64_t num_groups, NormProblem *p) {
  if (handle->arch < MLUOP_MLU370) {
    LOG(ERROR) << api << " needs a compute-capability 10.x device; this handle's device is not one.";
    return MLUOP_STATUS_ARCH_MISMATCH;
  }
  PARAM_CHECK(api, isRowType(input_desc->getDtype()));
  const int dim = input_desc->getDim();
  PARAM_CHECK(api, dim >= 2);
  STRIDE_TENSOR_CHECK(api + ":", input_desc, "input_desc must be contiguous");
  const int64_t channels = input_desc->getDimIndex(dim - 1);
  PARAM_CHECK(api, channels >= 1);
  PARAM_CHECK(api, num_groups >= 1 && num_groups <= channels);
  PARAM_CHECK(api, channels % num_groups == 0);
  int64_t rows = 1, inner = 1;
  bool too_many = false;
  for (int i = 0; i < dim - 1; ++i) {
    PARAM_CHECK(api, input_desc->getDimIndex(i) >= 0);
    rows *= input_desc->getDimIndex(i);
    if (i > 0) inner *= input_desc->getDimIndex(i);
    too_many |= rows >= (int64_t)LARGE_TENSOR_NUM || inner >= (int64_t)LARGE_TENSOR_NUM;
    if (too_many) break;
  }
  p->samples = input_desc->getDimIndex(0);
  p->sample_rows = inner;
  p->ragged = sample_ends_desc != nullptr;
  if (p->ragged) {
    PARAM_CHECK_EQ(api, dim, 2);
    PARAM_CHECK_EQ(api, sample_ends_desc->getDim(), 1);
    PARAM_CHECK(api, sample_ends_desc->getDtype() == MLUOP_DTYPE_INT32);
    STRIDE_TENSOR_CHECK(api + ":", sample_ends_desc, "sample_ends_desc must be contiguous");
    p->samples = sample_ends_desc->getDimIndex(0);
    p->sample_rows = 0;
  }
  if (too_many || channels > kMaxChannels || p->samples * num_groups >= (int64_t)LARGE_TENSOR_NUM) {
    LOG(ERROR) << api << " Overflow max tensor num. Fewer than 2^31 rows and (sample, group) pairs and at most "
               << kMaxChannels << " channels are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  p->dtype = input_desc->getDtype();
  p->rows = rows;
  p->channels = (int)channels;
  p->groups = (int)num_groups;
  p->sm_count = handle->sm_count > 0 ? handle->sm_count : 148;
  return MLUOP_STATUS_SUCCESS;
}

// weight and bias, or their gradients: [C] of float or the input's type, both the same.
mluOpStatus_t affineCheck(const std::string &api, const NormProblem &p, const mluOpTensorDescriptor_t weight_desc,
                          const mluOpTensorDescriptor_t bias_desc, bool *is_float) {
  PARAM_CHECK(api, (weight_desc == nullptr) == (bias_desc == nullptr));
  *is_float = true;
  if (weight_desc == nullptr) return MLUOP_STATUS_SUCCESS;
  for (const mluOpTensorDescriptor_t d : {weight_desc, bias_desc}) {
    PARAM_CHECK_EQ(api, d->getDim(), 1);
    PARAM_CHECK_EQ(api, d->getDimIndex(0), p.channels);
    STRIDE_TENSOR_CHECK(api + ":", d, "weight and bias must be contiguous");
  }
  PARAM_CHECK_EQ(api, weight_desc->getDtype(), bias_desc->getDtype());
  PARAM_CHECK(api, weight_desc->getDtype() == MLUOP_DTYPE_FLOAT || weight_desc->getDtype() == p.dtype);
  *is_float = weight_desc->getDtype() == MLUOP_DTYPE_FLOAT;
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t statisticsCheck(const std::string &api, const NormProblem &p, const mluOpTensorDescriptor_t mean_desc,
                              const mluOpTensorDescriptor_t rstd_desc) {
  for (const mluOpTensorDescriptor_t d : {mean_desc, rstd_desc}) {
    PARAM_CHECK_EQ(api, d->getDim(), 2);
    PARAM_CHECK_EQ(api, d->getDimIndex(0), p.samples);
    PARAM_CHECK_EQ(api, d->getDimIndex(1), p.groups);
    PARAM_CHECK(api, d->getDtype() == MLUOP_DTYPE_FLOAT);
    STRIDE_TENSOR_CHECK(api + ":", d, "mean and rstd must be contiguous");
  }
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t rowTensorCheck(const std::string &api, const mluOpTensorDescriptor_t input_desc,
                             const mluOpTensorDescriptor_t desc) {
  PARAM_CHECK(api, sameDims(input_desc, desc));
  PARAM_CHECK_EQ(api, desc->getDtype(), input_desc->getDtype());
  STRIDE_TENSOR_CHECK(api + ":", desc, "tensors must be contiguous");
  return MLUOP_STATUS_SUCCESS;
}

bool isActivation(mluOpGroupNormAct_t a) {
  return a == MLUOP_GROUP_NORM_ACT_NONE || a == MLUOP_GROUP_NORM_ACT_RELU || a == MLUOP_GROUP_NORM_ACT_SILU;
}

mluOpStatus_t workspaceSize(const std::string &api, mluOpHandle_t handle, const mluOpTensorDescriptor_t input_desc,
                            const mluOpTensorDescriptor_t sample_ends_desc, int64_t num_groups, bool backward,
                            size_t *workspace_size) {
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, input_desc != nullptr);
  PARAM_CHECK(api, workspace_size != nullptr);
  NormProblem p{};
  const mluOpStatus_t st = makeProblem(api, handle, input_desc, sample_ends_desc, num_groups, &p);
  if (st != MLUOP_STATUS_SUCCESS) return st;
  *workspace_size = mluop::group_norm_act::normWorkspaceBytes(p, backward);
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t workspaceCheck(const std::string &api, const NormProblem &p, bool backward, const void *workspace,
                             size_t workspace_size) {
  const size_t need = mluop::group_norm_act::normWorkspaceBytes(p, backward);
  if ((workspace == nullptr && need > 0) || workspace_size < need) {
    LOG(ERROR) << api << " workspace of " << workspace_size << " bytes is smaller than the " << need
               << " bytes that the query reports.";
    return MLUOP_STATUS_BAD_PARAM;
  }
  return MLUOP_STATUS_SUCCESS;
}

}  // namespace

#define RETURN_UNLESS_OK(call)                        \
  {                                                   \
    const mluOpStatus_t st__ = (call);                \
    if (st__ != MLUOP_STATUS_SUCCESS) return st__;    \
  }

extern "C" {

mluOpStatus_t MLUOP_WIN_API mluOpGetGroupNormActForwardWorkspaceSize(mluOpHandle_t handle,
                                                                     const mluOpTensorDescriptor_t input_desc,
                                                                     const mluOpTensorDescriptor_t sample_ends_desc,
                                                                     const int64_t num_groups,
                                                                     size_t *workspace_size) {
  return workspaceSize("[mluOpGetGroupNormActForwardWorkspaceSize]", handle, input_desc, sample_ends_desc, num_groups,
                       false, workspace_size);
}

mluOpStatus_t MLUOP_WIN_API mluOpGetGroupNormActBackwardWorkspaceSize(mluOpHandle_t handle,
                                                                      const mluOpTensorDescriptor_t input_desc,
                                                                      const mluOpTensorDescriptor_t sample_ends_desc,
                                                                      const int64_t num_groups,
                                                                      size_t *workspace_size) {
  return workspaceSize("[mluOpGetGroupNormActBackwardWorkspaceSize]", handle, input_desc, sample_ends_desc, num_groups,
                       true, workspace_size);
}

mluOpStatus_t MLUOP_WIN_API mluOpGroupNormActForward(
    mluOpHandle_t handle, const mluOpTensorDescriptor_t input_desc, const void *input,
    const mluOpTensorDescriptor_t weight_desc, const void *weight, const mluOpTensorDescriptor_t bias_desc,
    const void *bias, const mluOpTensorDescriptor_t sample_ends_desc, const void *sample_ends,
    const int64_t num_groups, const double epsilon, const mluOpGroupNormAct_t activation, void *workspace,
    const size_t workspace_size, const mluOpTensorDescriptor_t output_desc, void *output,
    const mluOpTensorDescriptor_t mean_desc, void *mean, const mluOpTensorDescriptor_t rstd_desc, void *rstd) {
  const std::string api = "[mluOpGroupNormActForward]";
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, input_desc != nullptr);
  PARAM_CHECK(api, output_desc != nullptr);
  PARAM_CHECK(api, mean_desc != nullptr);
  PARAM_CHECK(api, rstd_desc != nullptr);
  NormProblem p{};
  RETURN_UNLESS_OK(makeProblem(api, handle, input_desc, sample_ends_desc, num_groups, &p));
  RETURN_UNLESS_OK(affineCheck(api, p, weight_desc, bias_desc, &p.float_affine));
  RETURN_UNLESS_OK(rowTensorCheck(api, input_desc, output_desc));
  RETURN_UNLESS_OK(statisticsCheck(api, p, mean_desc, rstd_desc));
  PARAM_CHECK(api, std::isfinite((float)epsilon) && (float)epsilon > 0.0f);
  PARAM_CHECK(api, isActivation(activation));
  if (p.rows == 0 && p.samples == 0) {
    VLOG(5) << api << " Skip zero element tensor.";
    return MLUOP_STATUS_SUCCESS;
  }
  const size_t size = mluop::getSizeOfDataType(p.dtype), affine_size = p.float_affine ? 4 : size;
  if (p.rows > 0) {
    PARAM_CHECK(api, input != nullptr && aligned(input, size));
    PARAM_CHECK(api, output != nullptr && aligned(output, size));
    PARAM_CHECK(api, sameOrApart(output, input, mluop::denseBytes(input_desc)));
    if (weight_desc != nullptr) {
      PARAM_CHECK(api, weight != nullptr && aligned(weight, affine_size));
      PARAM_CHECK(api, bias != nullptr && aligned(bias, affine_size));
    }
  }
  if (p.samples > 0) {
    PARAM_CHECK(api, mean != nullptr && aligned(mean, 4));
    PARAM_CHECK(api, rstd != nullptr && aligned(rstd, 4));
    if (sample_ends_desc != nullptr) PARAM_CHECK(api, sample_ends != nullptr && aligned(sample_ends, 4));
  }
  RETURN_UNLESS_OK(workspaceCheck(api, p, false, workspace, workspace_size));
  const Span ws(workspace, workspace_size), w(weight_desc, weight), b(bias_desc, bias), ends(sample_ends_desc, sample_ends);
  // (output on input: checked above)
  PARAM_CHECK(api, mluop::writtenApart({{output_desc, output}, {mean_desc, mean}, {rstd_desc, rstd}, ws}, {w, b, ends}));
  PARAM_CHECK(api, mluop::writtenApart({{mean_desc, mean}, {rstd_desc, rstd}, ws}, {{input_desc, input}}));
  if (handle->host_only) {
    LOG(ERROR) << api << " this handle was created without a CUDA device; nothing can be launched.";
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  p.sample_ends = sample_ends_desc != nullptr ? static_cast<const int32_t *>(sample_ends) : nullptr;
  p.epsilon = (float)epsilon;
  p.activation = activation;
  mluop::DeviceGuard guard(handle);
  const cudaError_t err = mluop::group_norm_act::launchNormForward(
      p, input, weight_desc ? weight : nullptr, weight_desc ? bias : nullptr, workspace, output,
      static_cast<float *>(mean), static_cast<float *>(rstd), handle->queue);
  if (err != cudaSuccess) {
    LOG(ERROR) << api << " launch failed: " << cudaGetErrorString(err);
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpGroupNormActBackward(
    mluOpHandle_t handle, const mluOpTensorDescriptor_t output_grad_desc, const void *output_grad,
    const mluOpTensorDescriptor_t input_desc, const void *input, const mluOpTensorDescriptor_t weight_desc,
    const void *weight, const mluOpTensorDescriptor_t bias_desc, const void *bias,
    const mluOpTensorDescriptor_t sample_ends_desc, const void *sample_ends,
    const mluOpTensorDescriptor_t mean_desc, const void *mean, const mluOpTensorDescriptor_t rstd_desc,
    const void *rstd, const int64_t num_groups, const mluOpGroupNormAct_t activation, void *workspace,
    const size_t workspace_size, const mluOpTensorDescriptor_t input_grad_desc, void *input_grad,
    const mluOpTensorDescriptor_t weight_grad_desc, void *weight_grad,
    const mluOpTensorDescriptor_t bias_grad_desc, void *bias_grad) {
  const std::string api = "[mluOpGroupNormActBackward]";
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, output_grad_desc != nullptr);
  PARAM_CHECK(api, input_desc != nullptr);
  PARAM_CHECK(api, mean_desc != nullptr);
  PARAM_CHECK(api, rstd_desc != nullptr);
  PARAM_CHECK(api, input_grad_desc != nullptr);
  NormProblem p{};
  RETURN_UNLESS_OK(makeProblem(api, handle, input_desc, sample_ends_desc, num_groups, &p));
  RETURN_UNLESS_OK(affineCheck(api, p, weight_desc, bias_desc, &p.float_affine));
  RETURN_UNLESS_OK(affineCheck(api, p, weight_grad_desc, bias_grad_desc, &p.float_affine_grad));
  RETURN_UNLESS_OK(rowTensorCheck(api, input_desc, output_grad_desc));
  RETURN_UNLESS_OK(rowTensorCheck(api, input_desc, input_grad_desc));
  RETURN_UNLESS_OK(statisticsCheck(api, p, mean_desc, rstd_desc));
  PARAM_CHECK(api, isActivation(activation));
  const size_t size = mluop::getSizeOfDataType(p.dtype), affine_size = p.float_affine ? 4 : size;
  if (weight_grad_desc != nullptr) {
    const size_t grad_size = p.float_affine_grad ? 4 : size;
    PARAM_CHECK(api, weight_grad != nullptr && aligned(weight_grad, grad_size));
    PARAM_CHECK(api, bias_grad != nullptr && aligned(bias_grad, grad_size));
  } else if (p.rows == 0 && p.samples == 0) {
    VLOG(5) << api << " Skip zero element tensor.";
    return MLUOP_STATUS_SUCCESS;
  }
  if (p.rows > 0) {
    PARAM_CHECK(api, output_grad != nullptr && aligned(output_grad, size));
    PARAM_CHECK(api, input != nullptr && aligned(input, size));
    PARAM_CHECK(api, input_grad != nullptr && aligned(input_grad, size));
    PARAM_CHECK(api, sameOrApart(input_grad, output_grad, mluop::denseBytes(input_desc)));
    PARAM_CHECK(api, sameOrApart(input_grad, input, mluop::denseBytes(input_desc)));
    if (weight_desc != nullptr) {
      PARAM_CHECK(api, weight != nullptr && aligned(weight, affine_size));
      PARAM_CHECK(api, bias != nullptr && aligned(bias, affine_size));
    }
  }
  if (p.samples > 0) {
    PARAM_CHECK(api, mean != nullptr && aligned(mean, 4));
    PARAM_CHECK(api, rstd != nullptr && aligned(rstd, 4));
    if (sample_ends_desc != nullptr) PARAM_CHECK(api, sample_ends != nullptr && aligned(sample_ends, 4));
  }
  RETURN_UNLESS_OK(workspaceCheck(api, p, true, workspace, workspace_size));
  const Span ws(workspace, workspace_size), w(weight_desc, weight), b(bias_desc, bias), ends(sample_ends_desc, sample_ends);
  const Span dw(weight_grad_desc, weight_grad), db(bias_grad_desc, bias_grad);
  // (input_grad on output_grad or input: checked above)
  PARAM_CHECK(api, mluop::writtenApart({{input_grad_desc, input_grad}, dw, db, ws},
                                       {w, b, ends, {mean_desc, mean}, {rstd_desc, rstd}}));
  PARAM_CHECK(api, mluop::writtenApart({dw, db, ws}, {{output_grad_desc, output_grad}, {input_desc, input}}));
  if (handle->host_only) {
    LOG(ERROR) << api << " this handle was created without a CUDA device; nothing can be launched.";
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  p.sample_ends = sample_ends_desc != nullptr ? static_cast<const int32_t *>(sample_ends) : nullptr;
  p.activation = activation;
  mluop::DeviceGuard guard(handle);
  const cudaError_t err = mluop::group_norm_act::launchNormBackward(
      p, output_grad, input, weight_desc ? weight : nullptr, weight_desc ? bias : nullptr,
      static_cast<const float *>(mean), static_cast<const float *>(rstd), workspace, input_grad,
      weight_grad_desc ? weight_grad : nullptr, weight_grad_desc ? bias_grad : nullptr, handle->queue);
  if (err != cudaSuccess) {
    LOG(ERROR) << api << " launch failed: " << cudaGetErrorString(err);
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  return MLUOP_STATUS_SUCCESS;
}

}  // extern "C"
