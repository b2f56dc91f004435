// Launch interface of the matrix products grouped by row blocks.
#ifndef MLUOP_B200_KERNELS_GROUPED_MATMUL_KERNELS_H_
#define MLUOP_B200_KERNELS_GROUPED_MATMUL_KERNELS_H_

#include <cuda_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "mlu_op.h"

namespace mluop {
namespace grouped_matmul {

constexpr int kMaxGroups = 1024;

enum Mode {
  kForward = 0,         // output[r,:] = input[r,:] * weight[g]
  kBackwardInput = 1,   // input_grad[r,:] = output_grad[r,:] * weight[g]^T
  kBackwardWeight = 2,  // weight_grad[g] = input[rows of g]^T * output_grad[rows of g]
};

struct Problem {
  Mode mode;
  mluOpDataType_t dtype;
  bool float_weight_grad;  // the weight gradient in float, else in `dtype`
  int64_t rows;
  int groups;
  int ci, co;
  int sm_count;
  int32_t *sticky;  // device-visible host word that a bounded wait's error is recorded in, or null
};

// Weight gradient: how many rows of a group one block takes, and the scratch that follows from it.  A group of
// more rows is split into chunks whose float sums lie in `partial` and are added by a second kernel.
struct WeightGradPlan {
  bool tensor_cores;
  int tile_m, tile_n;
  int64_t chunk_rows;
  int64_t slots;  // chunks of split groups there can be
  size_t maps, partial, total;  // byte offsets (from a 256-byte boundary in the workspace) and size
};
WeightGradPlan planWeightGrad(const Problem &p, bool tensor_cores);
// The tensor-core kernel's tile of a weight gradient of these sizes.
void weightGradTile(const Problem &p, int *tile_m, int *tile_n);
// Large enough for either kernel.
size_t weightGradWorkspaceBytes(const Problem &p);

// Whether the tensor-core kernel can take operands of these types, sizes and addresses.
bool tensorCoresEligible(const Problem &p, const void *a, const void *b, const void *c);

// `a` is input (forward, weight gradient) or output_grad (input gradient); `b` is weight or output_grad; `c` the result.
cudaError_t launchGeneral(const Problem &p, const void *a, const void *b, const int32_t *ends, void *c, void *workspace,
                          cudaStream_t stream);
cudaError_t launchTensorCores(const Problem &p, const void *a, const void *b, const int32_t *ends, void *c,
                              void *workspace, cudaStream_t stream);
// Adds the chunks of the split groups (weight gradient, either kernel).
cudaError_t launchAddChunks(const Problem &p, const WeightGradPlan &plan, const int32_t *ends, const float *partial,
                            void *c, cudaStream_t stream);

}  // namespace grouped_matmul
}  // namespace mluop

#endif  // MLUOP_B200_KERNELS_GROUPED_MATMUL_KERNELS_H_
