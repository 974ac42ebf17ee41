// cq_launch.cuh -- launches that overlap with the end of the kernel before them.
#pragma once

#include <string>

#include "cq_common.cuh"

namespace cq {

// A launch that may start while the kernel before it in the stream drains: the
// kernel waits for that one's results itself (ptx::grid_dependency_wait, in every
// thread before its first access to memory).
template <class... P, class... X>
inline int launch_after(void (*fn)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, const char *what,
                        X... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the next call
    return set_error(CQ_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  return check_launch(what);
}

}  // namespace cq
