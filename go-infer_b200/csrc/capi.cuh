// capi.cuh -- the library's device context (capi.cu) for the other files that
// define entry points of include/goinfer_cuda.h.
#pragma once

#include <cuda_runtime.h>

#include <functional>
#include <mutex>

#include "model.cuh"

namespace gi {

struct CapiCtx {
  int sm_count = 0;
  cudaStream_t stream = nullptr;  // the library's own
  int* error = nullptr;           // set by kernels whose bounded waits give up
};

// Held for the length of an entry point.
std::mutex& capi_mutex();
// Binds the calling thread to the library's device (mutex held); a status
// code, with its text set, when gi_cuda_init has not succeeded.
int capi_ready(CapiCtx* c);
// A gi_cuda_model_t.
struct ModelHandle {
  DecodeModel m;
  uint32_t* pinned = nullptr;  // prompt tokens staged for the per-step copies
  size_t pinned_cap = 0;
  StepState* pinned_state = nullptr;
  ~ModelHandle() {
    if (pinned) cudaFreeHost(pinned);
    if (pinned_state) cudaFreeHost(pinned_state);
  }
};

// gi_cuda_model_generate (mutex held, checked pointers).  begin(steps, stream),
// if given, sets the steps up after the checks; its status code ends the call.
int model_generate(ModelHandle* h, const int32_t* tokens, uint32_t n_tokens, uint32_t start_pos, uint32_t n_gen,
                   const std::function<int(int, cudaStream_t)>& begin, uint32_t* out_tokens, float* out_logits,
                   float* decode_ms);
// -6, with its text set, when a bounded wait has given up since this was last
// asked (a look at host memory; mutex held).
int capi_device_error();
// Sets gi_cuda_last_error's text and returns `code`.
int capi_fail(int code, const char* what, cudaError_t e = cudaSuccess);

}  // namespace gi
