// Launches that may start while the stream's previous kernel still runs: the
// kernel sets itself up, then waits (grid_wait) before its first access to
// global memory, so that its set-up overlaps that kernel's end. Every kernel
// launched this way waits, hence a kernel that has waited may rely on all the
// earlier ones, and every access of a kernel comes after theirs. A call takes
// 0.3 to 1 us less in a row of them (16 x 8192 x 3584 7.85 -> 6.8 us).
#pragma once

#include <cuda_runtime.h>

#include <utility>

namespace megacu_b200 {

// Waits until the stream's earlier kernels have completed and their writes
// are visible.
__device__ __forceinline__ void grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Lets the next kernel start once every CTA of this one has started.
__device__ __forceinline__ void grid_start_next() {
  asm volatile("griddepcontrol.launch_dependents;");
}

template <class... P, class... A>
cudaError_t launch_chained(void (*kernel)(P...), unsigned grid, unsigned threads,
                           std::size_t smem, cudaStream_t stream, unsigned cluster, A &&...args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(std::forward<A>(args))...);
}

}  // namespace megacu_b200
