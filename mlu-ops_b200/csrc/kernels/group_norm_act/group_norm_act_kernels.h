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
  bool ragged;          // sample_ends is given
  int64_t sample_rows;  // rows of each sample where it is not
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

// The form for samples of very few rows (group_norm_act_short.cu).
constexpr int kShortRows = 8;       // it takes samples of up to as many rows always,
constexpr int kMostShortRows = 64;  // and of up to as many where there are enough samples
struct ShortPlan {
  int vec;            // channels of a vector
  int lanes;          // of one (sample, group): a power of two, at most a warp; 0: the form does not apply
  int vectors;        // of a lane, at most
  int groups_block;   // groups side by side in a block
  int samples_block;  // samples of a block at a time
  int tiles;          // blocks along the groups
  int64_t blocks;     // and along the samples
};
ShortPlan planShort(const NormProblem &p, int vec);
cudaError_t launchShortForward(const NormProblem &p, const ShortPlan &plan, const void *input, const void *weight,
                               const void *bias, void *output, float *mean, float *rstd, cudaStream_t stream);
// partial: null, or the sums of du and du xhat, a line of `channels` for each of plan.blocks
cudaError_t launchShortBackward(const NormProblem &p, const ShortPlan &plan, const void *output_grad, const void *input,
                                const void *weight, const void *bias, const float *mean, const float *rstd, float2 *partial,
                                void *input_grad, cudaStream_t stream);

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
