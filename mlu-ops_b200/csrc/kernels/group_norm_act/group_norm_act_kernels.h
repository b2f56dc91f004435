// Launch interface of group norm with an activation on channels-last rows.
#ifndef MLUOP_B200_KERNELS_GROUP_NORM_ACT_KERNELS_H_
#define MLUOP_B200_KERNELS_GROUP_NORM_ACT_KERNELS_H_

#include <cuda_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "mlu_op.h"

namespace mluop {
namespace group_norm_act {

struct NormProblem {
  mluOpDataType_t dtype;
  bool float_affine, float_affine_grad;  // weight and bias (and their gradients) in float, else in `dtype`
  int64_t rows;         // all rows
  int64_t samples;
  int64_t sample_rows;  // rows of each sample where sample_ends is null
  int channels, groups;
  const int32_t *sample_ends;
  float epsilon;
  mluOpGroupNormAct_t activation;
  int sm_count;
};

// How the rows are split over blocks, and where the scratch of the two passes lies (bytes; it starts on
// a 256-byte boundary inside the workspace).
struct NormPlan {
  int vec;             // channels a thread moves at once
  int column_threads;  // threads side by side on a row
  int row_threads;     // rows a block takes at once
  int column_tiles;
  int64_t block_rows;
  int64_t blocks;  // row blocks
  size_t partial, sample_sums, group_means, total;
};

// The one-launch form for few rows: the width of its slices in vectors of `vec` channels, or 0 where it does not apply.
int sliceColumns(const NormProblem &p, int vec, bool backward);
NormPlan planNorm(const NormProblem &p, bool backward, bool vectors);
size_t normWorkspaceBytes(const NormProblem &p, bool backward);

cudaError_t launchNormForward(const NormProblem &p, const void *input, const void *weight, const void *bias,
                              void *workspace, void *output, float *mean, float *rstd, cudaStream_t stream);
cudaError_t launchNormBackward(const NormProblem &p, const void *output_grad, const void *input, const void *weight,
                               const void *bias, const float *mean, const float *rstd, void *workspace,
                               void *input_grad, void *weight_grad, void *bias_grad, cudaStream_t stream);

}  // namespace group_norm_act
}  // namespace mluop

#endif  // MLUOP_B200_KERNELS_GROUP_NORM_ACT_KERNELS_H_
