// dependent_launch.cuh - launches that may begin while the one before them ends.
#pragma once
#include <cuda_runtime.h>

namespace vcb {

// The kernel, which takes its parameters as one structure, waits for the results
// of the launch before it itself (grid_dependency_wait), before it reads or
// writes global memory.
template <class P>
cudaError_t launch_dependent(void (*kernel)(P), dim3 grid, int threads, int smem, const P &p,
                             cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace vcb
