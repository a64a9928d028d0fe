// Launches that may begin before the stream's previous kernel has ended.
//
// A decode step is a chain of kernels of a few microseconds, and a kernel's
// launch takes about one of them.  Launched with programmatic stream
// serialization a kernel's CTAs are set up while the one before it ends; it
// must call wait_for_stream(), in every thread, before it touches memory.
// (Measured on one B200: an append of a 128-token step 5.1 -> 4.8 us, of one
// token 3.9 -> 3.6 us into the 4-bit cache.)
#pragma once

#include <cuda_runtime.h>

namespace gqa {

// Returns once every kernel before this one in the stream has ended and its
// memory is visible (at once for a kernel launched the ordinary way).
__device__ __forceinline__ void wait_for_stream() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// A load of what an earlier kernel may have written.  Read-only (.nc) loads
// are for data that stays the same while the kernel exists, and a kernel
// launched early exists while the one before it still writes.
template <class T>
__device__ __forceinline__ T ld_plain(const T* p) {
  return *p;
}

template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), int grid, int threads, size_t smem,
                         cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

}  // namespace gqa
