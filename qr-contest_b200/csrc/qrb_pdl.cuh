// qrb200 -- kernels that are launched while the one before them in the stream still runs.
//
// A layer's kernels are short and follow one another, and between two of them the GPU waits a
// microsecond or more for the next to be launched and set up.  Launched with programmatic stream
// serialization, a kernel may start once every block of the one before has called allow_next() (or has
// ended); it sets itself up and then waits in after_previous() until everything before it in the
// stream has completed and is visible.  So no thread touches global memory before after_previous(), and
// a kernel calls allow_next() when its loads are done: blocks that wait take places, and with the call
// at the start, blocks of the next kernels but one settled unevenly between this one's (one token
// 4096 x 4096 in 8 bits: 8.2 us, with the call after the loads 6.2).  Without the launch attribute both do
// nothing.
#pragma once
#include <cuda_runtime.h>

namespace qrb {

__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that way (early) or when all before it is done; cluster: blocks of a cluster along
// x (0: as the kernel says).
template <typename... P, typename... A>
inline cudaError_t launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                 unsigned cluster, bool early, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = early;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

}  // namespace qrb
