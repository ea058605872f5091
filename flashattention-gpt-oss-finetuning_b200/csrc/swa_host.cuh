// swa_host.cuh -- host-side helpers that the translation units with extern "C" entry points share.
#pragma once

#include <cuda_runtime.h>

#include <atomic>

namespace swa {

// Allow a kernel `bytes` of dynamic shared memory: set once per device and kernel type K (each
// instance of a kernel has a Tag of its own; the attribute stays for the life of the context).
template <typename Tag, typename K> cudaError_t allow_smem(K kernel, int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// SwaStatus of a CUDA call; keeps its text for swa_last_cuda_error.
int host_record(cudaError_t e);

// The current device's flag for pages and lengths out of range (nullptr: lookup failed).
int* page_error_ptr();

}  // namespace swa
