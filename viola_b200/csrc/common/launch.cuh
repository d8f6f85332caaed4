// Launch of a kernel that begins while the kernel before it in the stream ends, and the count of launches.
#pragma once
#include <cuda_runtime.h>
#include <atomic>

namespace vb {

// kernels launched so far by the entries of experts.cu and block_norm.cu (vb_block_launches)
inline std::atomic<long long> launches{0};
inline void count_launch() { launches.fetch_add(1, std::memory_order_relaxed); }

// The kernel may start once every block of the one before it has called cudaTriggerProgrammaticLaunchCompletion (or has
// ended); it calls cudaGridDependencySynchronize before it reads what that one writes, and before it writes anything.  What it
// reads earlier must have been there when that one began, so the one before is always the caller's own ordinary launch.
template <typename... P, typename... A>
void launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, static_cast<P>(args)...);
  count_launch();
}

}  // namespace vb
