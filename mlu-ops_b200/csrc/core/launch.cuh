// Launches of kernels that follow one another in a stream.
//
// A kernel that begins with letNextKernelStart() allows the next one of its chain to be
// set up while it runs: the next one's blocks start where there is room and stop in
// waitForKernelBefore() until the kernel before has finished and its writes are visible.
// What they do before that call may touch nothing that the chain writes.  It hides about
// two microseconds of launch latency between two kernels.
#ifndef MLUOP_B200_CORE_LAUNCH_CUH_
#define MLUOP_B200_CORE_LAUNCH_CUH_

#include <cuda_runtime.h>

namespace mluop {

__device__ __forceinline__ void letNextKernelStart() { cudaTriggerProgrammaticLaunchCompletion(); }
__device__ __forceinline__ void waitForKernelBefore() { cudaGridDependencySynchronize(); }

// kernel<<<grid, block, smem, stream>>>(args...) for a kernel that calls waitForKernelBefore().
template <typename... Params, typename... Args>
cudaError_t launchAfterKernel(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                              Args... args) {
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

}  // namespace mluop

#endif  // MLUOP_B200_CORE_LAUNCH_CUH_
