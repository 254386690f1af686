// Programmatic dependent launch of short kernels: a kernel launched with launch_early may be scheduled while
// the one before it on the stream still runs, so that its launch overlaps that one's end.
#pragma once
#include <cuda_runtime.h>

#include "common.cuh"

namespace astrai {

// What such a kernel begins with: everything that ran before it on the stream is complete and visible (so
// completion stays transitive along the stream), and the kernel after it may be scheduled.
__device__ __forceinline__ void begin_early() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... A>
void launch_early(void (*kernel)(A...), dim3 grid, dim3 block, int smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  note_launch();
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace astrai
