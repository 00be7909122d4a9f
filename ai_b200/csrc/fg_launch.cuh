// Launching a kernel so that it overlaps the end of the one before it in its
// stream (programmatic dependent launch): its blocks may be set up while the
// last blocks of that one still run. They call wait_for_previous() before
// anything that it wrote, or reads, is touched; and what it wrote is not read
// through the read-only path (__ldg), for it changes in the kernel's lifetime.
#pragma once

#include <cuda_runtime.h>

#include "fg_internal.h"

namespace fg {

__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The next kernel in the stream, where it was launched with launch_after, may
// be set up once all blocks of this one have come here.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), unsigned blocks, unsigned threads, cudaStream_t s, const A&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return FG_OK;
}

}  // namespace fg
