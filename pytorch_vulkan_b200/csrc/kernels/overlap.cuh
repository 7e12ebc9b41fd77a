// Launches whose start overlaps the end of the launch before them in the stream.
//
// A kernel that calls wait_for_last() before anything else and lets the next one
// come at once may be scheduled while the last one's blocks finish: the two to
// three microseconds between dependent launches are spent in the shadow of the
// last one.  wait_for_last() returns when all of the last launch's work is done
// and visible, so no thread may read or write global memory that has not met it, or
// a barrier behind one that has; kernels without it are not affected, whichever
// side of these they are on.  A kernel that allocates tensor memory does so before
// it lets the next one come: that one's blocks could take the memory first, and
// hold it until this launch has ended, which waits for them.
// A stream of calls of the C functions, us with and without: 8-bit layer 1 x 4096 ->
// 4096 5.7 and 8.2, 300 x 1000 -> 5001 8.1 and 10.3, 128 x 4096 -> 4096 10.0 and 12.3;
// log probabilities of 8192 x 1000 9.7 and 12.3, of 1 x 32768 with 20 alternatives
// 7.8 and 10.3; norm of 2047 x 5000 to 8 bits and back 25.5 and 30.7, with gradients
// 8192 x 4096 101 and 107.  (Launches with a long list of tensors as their argument
// gain nothing: the host is the bound.)
#pragma once
#include "common.cuh"

namespace pvb2 {

__device__ __forceinline__ void let_next_come() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// `cluster`: blocks of one, 0 where the kernel itself says so or has none
template <typename... P, typename... A>
static cudaError_t launch_over(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
                               unsigned cluster, const A&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace pvb2
