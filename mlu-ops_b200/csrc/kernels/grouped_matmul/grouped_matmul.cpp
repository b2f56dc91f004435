// mluOpGroupedMatMulForward / BackwardInput / BackwardWeight and the workspace query:
// argument checks and dispatch.  No counterpart in the reference.
#include <cuda_runtime_api.h>

#include <string>

#include "core/context.h"
#include "core/logging.h"
#include "core/overlap.h"
#include "core/tensor.h"
#include "kernels/grouped_matmul/grouped_matmul_kernels.h"

using mluop::grouped_matmul::Problem;

namespace {

constexpr int64_t kMaxChannels = 65536;

bool isRowType(mluOpDataType_t t) {
  return t == MLUOP_DTYPE_HALF || t == MLUOP_DTYPE_BFLOAT16 || t == MLUOP_DTYPE_FLOAT;
}

bool aligned(const void *p, mluOpDataType_t t) {
  return reinterpret_cast<size_t>(p) % mluop::getSizeOfDataType(t) == 0;
}

// wide [rows, Ci] and narrow [rows, Co] are the two row matrices, stack [G, Ci, Co] the groups' matrices.
mluOpStatus_t makeProblem(const std::string &api, mluOpHandle_t handle, mluop::grouped_matmul::Mode mode,
                          const mluOpTensorDescriptor_t input_desc, const mluOpTensorDescriptor_t output_desc,
                          const mluOpTensorDescriptor_t weight_desc, Problem *p) {
  if (handle->arch < MLUOP_MLU370) {
    LOG(ERROR) << api << " needs a compute-capability 10.x device; this handle's device is not one.";
    return MLUOP_STATUS_ARCH_MISMATCH;
  }
  PARAM_CHECK_EQ(api, input_desc->getDim(), 2);
  PARAM_CHECK_EQ(api, output_desc->getDim(), 2);
  PARAM_CHECK_EQ(api, weight_desc->getDim(), 3);
  PARAM_CHECK(api, isRowType(input_desc->getDtype()));
  PARAM_CHECK_EQ(api, output_desc->getDtype(), input_desc->getDtype());
  p->mode = mode;
  p->dtype = input_desc->getDtype();
  p->float_weight_grad = false;
  if (mode == mluop::grouped_matmul::kBackwardWeight) {
    PARAM_CHECK(api, weight_desc->getDtype() == p->dtype || weight_desc->getDtype() == MLUOP_DTYPE_FLOAT);
    p->float_weight_grad = weight_desc->getDtype() == MLUOP_DTYPE_FLOAT;
  } else {
    PARAM_CHECK_EQ(api, weight_desc->getDtype(), p->dtype);
  }
  STRIDE_TENSOR_CHECK(api + ":", input_desc, "tensors must be contiguous");
  STRIDE_TENSOR_CHECK(api + ":", output_desc, "tensors must be contiguous");
  STRIDE_TENSOR_CHECK(api + ":", weight_desc, "tensors must be contiguous");
  const int64_t rows = input_desc->getDimIndex(0), ci = input_desc->getDimIndex(1);
  const int64_t groups = weight_desc->getDimIndex(0), co = output_desc->getDimIndex(1);
  PARAM_CHECK(api, rows >= 0);
  PARAM_CHECK_EQ(api, output_desc->getDimIndex(0), rows);
  PARAM_CHECK_EQ(api, weight_desc->getDimIndex(1), ci);
  PARAM_CHECK_EQ(api, weight_desc->getDimIndex(2), co);
  PARAM_CHECK(api, groups >= 1 && ci >= 1 && co >= 1);
  const int64_t columns = ci > co ? ci : co;
  const bool large = rows >= (int64_t)LARGE_TENSOR_NUM || groups > mluop::grouped_matmul::kMaxGroups ||
                     columns > kMaxChannels ||
                     (rows / 128 + groups + 1) * ((columns + 63) / 64) >= (int64_t)1 << 30 ||
                     (mode == mluop::grouped_matmul::kBackwardWeight &&
                      (rows / 512 + groups) * ((ci + 127) / 128) * ((co + 63) / 64) >= (int64_t)1 << 30);
  if (large) {
    LOG(ERROR) << api << " at most " << mluop::grouped_matmul::kMaxGroups << " groups, " << kMaxChannels
               << " channels, 2^31 - 1 rows and 2^30 tiles are supported.";
    return MLUOP_STATUS_NOT_SUPPORTED;
  }
  p->rows = rows;
  p->groups = (int)groups;
  p->ci = (int)ci;
  p->co = (int)co;
  p->sm_count = handle->sm_count > 0 ? handle->sm_count : 148;
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t endsCheck(const std::string &api, const Problem &p, const mluOpTensorDescriptor_t ends_desc) {
  PARAM_CHECK_EQ(api, ends_desc->getDim(), 1);
  PARAM_CHECK_EQ(api, ends_desc->getDimIndex(0), p.groups);
  PARAM_CHECK(api, ends_desc->getDtype() == MLUOP_DTYPE_INT32);
  STRIDE_TENSOR_CHECK(api + ":", ends_desc, "group_ends_desc must be contiguous");
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t run(const std::string &api, mluOpHandle_t handle, Problem &p, const void *a, const void *b,
                  const void *ends, void *c, void *workspace) {
  if (handle->host_only) {
    LOG(ERROR) << api << " this handle was created without a CUDA device; nothing can be launched.";
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  if (mluop::takeStickyDeviceError(handle, api.c_str())) return MLUOP_STATUS_EXECUTION_FAILED;
  mluop::DeviceGuard guard(handle);
  p.sticky = mluop::stickyDeviceWord(handle);
  const int32_t *group_ends = static_cast<const int32_t *>(ends);
  const cudaError_t err =
      mluop::grouped_matmul::tensorCoresEligible(p, a, b, c)
          ? mluop::grouped_matmul::launchTensorCores(p, a, b, group_ends, c, workspace, handle->queue)
          : mluop::grouped_matmul::launchGeneral(p, a, b, group_ends, c, workspace, handle->queue);
  if (err != cudaSuccess) {
    LOG(ERROR) << api << " launch failed: " << cudaGetErrorString(err);
    return MLUOP_STATUS_EXECUTION_FAILED;
  }
  return mluop::reportIfRequested(handle, api.c_str());
}

}  // namespace

#define RETURN_UNLESS_OK(call)                     \
  {                                                \
    const mluOpStatus_t st__ = (call);             \
    if (st__ != MLUOP_STATUS_SUCCESS) return st__; \
  }

extern "C" {

mluOpStatus_t MLUOP_WIN_API mluOpGroupedMatMulForward(mluOpHandle_t handle, const mluOpTensorDescriptor_t input_desc,
                                                      const void *input, const mluOpTensorDescriptor_t weight_desc,
                                                      const void *weight,
                                                      const mluOpTensorDescriptor_t group_ends_desc,
                                                      const void *group_ends,
                                                      const mluOpTensorDescriptor_t output_desc, void *output) {
  const std::string api = "[mluOpGroupedMatMulForward]";
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, input_desc != nullptr);
  PARAM_CHECK(api, weight_desc != nullptr);
  PARAM_CHECK(api, group_ends_desc != nullptr);
  PARAM_CHECK(api, output_desc != nullptr);
  Problem p{};
  RETURN_UNLESS_OK(makeProblem(api, handle, mluop::grouped_matmul::kForward, input_desc, output_desc, weight_desc, &p));
  RETURN_UNLESS_OK(endsCheck(api, p, group_ends_desc));
  if (p.rows == 0) {
    VLOG(5) << api << " Skip zero element tensor.";
    return MLUOP_STATUS_SUCCESS;
  }
  PARAM_CHECK(api, input != nullptr && aligned(input, p.dtype));
  PARAM_CHECK(api, weight != nullptr && aligned(weight, p.dtype));
  PARAM_CHECK(api, group_ends != nullptr && aligned(group_ends, MLUOP_DTYPE_INT32));
  PARAM_CHECK(api, output != nullptr && aligned(output, p.dtype));
  PARAM_CHECK(api, mluop::writtenApart({{output_desc, output}},
                                       {{input_desc, input}, {weight_desc, weight}, {group_ends_desc, group_ends}}));
  return run(api, handle, p, input, weight, group_ends, output, nullptr);
}

mluOpStatus_t MLUOP_WIN_API mluOpGroupedMatMulBackwardInput(
    mluOpHandle_t handle, const mluOpTensorDescriptor_t output_grad_desc, const void *output_grad,
    const mluOpTensorDescriptor_t weight_desc, const void *weight, const mluOpTensorDescriptor_t group_ends_desc,
    const void *group_ends, const mluOpTensorDescriptor_t input_grad_desc, void *input_grad) {
  const std::string api = "[mluOpGroupedMatMulBackwardInput]";
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, output_grad_desc != nullptr);
  PARAM_CHECK(api, weight_desc != nullptr);
  PARAM_CHECK(api, group_ends_desc != nullptr);
  PARAM_CHECK(api, input_grad_desc != nullptr);
  Problem p{};
  RETURN_UNLESS_OK(makeProblem(api, handle, mluop::grouped_matmul::kBackwardInput, input_grad_desc, output_grad_desc,
                               weight_desc, &p));
  RETURN_UNLESS_OK(endsCheck(api, p, group_ends_desc));
  if (p.rows == 0) {
    VLOG(5) << api << " Skip zero element tensor.";
    return MLUOP_STATUS_SUCCESS;
  }
  PARAM_CHECK(api, output_grad != nullptr && aligned(output_grad, p.dtype));
  PARAM_CHECK(api, weight != nullptr && aligned(weight, p.dtype));
  PARAM_CHECK(api, group_ends != nullptr && aligned(group_ends, MLUOP_DTYPE_INT32));
  PARAM_CHECK(api, input_grad != nullptr && aligned(input_grad, p.dtype));
  PARAM_CHECK(api, mluop::writtenApart({{input_grad_desc, input_grad}}, {{output_grad_desc, output_grad},
                                                                         {weight_desc, weight},
                                                                         {group_ends_desc, group_ends}}));
  return run(api, handle, p, output_grad, weight, group_ends, input_grad, nullptr);
}

mluOpStatus_t MLUOP_WIN_API mluOpGetGroupedMatMulBackwardWeightWorkspaceSize(
    mluOpHandle_t handle, const mluOpTensorDescriptor_t input_desc, const mluOpTensorDescriptor_t output_grad_desc,
    const mluOpTensorDescriptor_t weight_grad_desc, size_t *workspace_size) {
  const std::string api = "[mluOpGetGroupedMatMulBackwardWeightWorkspaceSize]";
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, input_desc != nullptr);
  PARAM_CHECK(api, output_grad_desc != nullptr);
  PARAM_CHECK(api, weight_grad_desc != nullptr);
  PARAM_CHECK(api, workspace_size != nullptr);
  Problem p{};
  RETURN_UNLESS_OK(makeProblem(api, handle, mluop::grouped_matmul::kBackwardWeight, input_desc, output_grad_desc,
                               weight_grad_desc, &p));
  *workspace_size = mluop::grouped_matmul::weightGradWorkspaceBytes(p);
  return MLUOP_STATUS_SUCCESS;
}

mluOpStatus_t MLUOP_WIN_API mluOpGroupedMatMulBackwardWeight(
    mluOpHandle_t handle, const mluOpTensorDescriptor_t input_desc, const void *input,
    const mluOpTensorDescriptor_t output_grad_desc, const void *output_grad,
    const mluOpTensorDescriptor_t group_ends_desc, const void *group_ends, void *workspace,
    const size_t workspace_size, const mluOpTensorDescriptor_t weight_grad_desc, void *weight_grad) {
  const std::string api = "[mluOpGroupedMatMulBackwardWeight]";
  PARAM_CHECK(api, handle != nullptr);
  PARAM_CHECK(api, input_desc != nullptr);
  PARAM_CHECK(api, output_grad_desc != nullptr);
  PARAM_CHECK(api, group_ends_desc != nullptr);
  PARAM_CHECK(api, weight_grad_desc != nullptr);
  Problem p{};
  RETURN_UNLESS_OK(makeProblem(api, handle, mluop::grouped_matmul::kBackwardWeight, input_desc, output_grad_desc,
                               weight_grad_desc, &p));
  RETURN_UNLESS_OK(endsCheck(api, p, group_ends_desc));
  PARAM_CHECK(api, weight_grad != nullptr && aligned(weight_grad, weight_grad_desc->getDtype()));
  if (p.rows > 0) {
    PARAM_CHECK(api, input != nullptr && aligned(input, p.dtype));
    PARAM_CHECK(api, output_grad != nullptr && aligned(output_grad, p.dtype));
    PARAM_CHECK(api, group_ends != nullptr && aligned(group_ends, MLUOP_DTYPE_INT32));
  }
  const size_t need = mluop::grouped_matmul::weightGradWorkspaceBytes(p);
  if (workspace == nullptr || workspace_size < need) {
    LOG(ERROR) << api << " workspace of " << workspace_size << " bytes is smaller than the " << need
               << " bytes mluOpGetGroupedMatMulBackwardWeightWorkspaceSize reports.";
    return MLUOP_STATUS_BAD_PARAM;
  }
  PARAM_CHECK(api, mluop::writtenApart({{weight_grad_desc, weight_grad}, {workspace, workspace_size}},
                                       {{input_desc, input}, {output_grad_desc, output_grad}, {group_ends_desc, group_ends}}));
  if (p.rows == 0 && !handle->host_only) {  // every group is empty
    mluop::DeviceGuard guard(handle);
    const size_t bytes = (size_t)mluOpGetTensorElementNum(weight_grad_desc) *
                         mluop::getSizeOfDataType(weight_grad_desc->getDtype());
    if (cudaMemsetAsync(weight_grad, 0, bytes, handle->queue) != cudaSuccess) {
      LOG(ERROR) << api << " launch failed: " << cudaGetErrorString(cudaGetLastError());
      return MLUOP_STATUS_EXECUTION_FAILED;
    }
    return MLUOP_STATUS_SUCCESS;
  }
  return run(api, handle, p, input, output_grad, group_ends, weight_grad, workspace);
}

}  // extern "C"
