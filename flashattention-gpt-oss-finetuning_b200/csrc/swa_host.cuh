// swa_host.cuh -- host-side helpers that the translation units with extern "C" entry points share.
#pragma once

#include <cuda_runtime.h>

namespace swa {

// SwaStatus of a CUDA call; keeps its text for swa_last_cuda_error.
int host_record(cudaError_t e);

// The current device's flag for pages and lengths out of range (nullptr: lookup failed).
int* page_error_ptr();

}  // namespace swa
