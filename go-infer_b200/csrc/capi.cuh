// capi.cuh -- the library's device context (capi.cu) for the other files that
// define entry points of include/goinfer_cuda.h.
#pragma once

#include <cuda_runtime.h>

#include <mutex>

namespace gi {

struct CapiCtx {
  int sm_count = 0;
  cudaStream_t stream = nullptr;  // the library's own
};

// Held for the length of an entry point.
std::mutex& capi_mutex();
// Binds the calling thread to the library's device (mutex held); a status
// code, with its text set, when gi_cuda_init has not succeeded.
int capi_ready(CapiCtx* c);
// Sets gi_cuda_last_error's text and returns `code`.
int capi_fail(int code, const char* what, cudaError_t e = cudaSuccess);

}  // namespace gi
