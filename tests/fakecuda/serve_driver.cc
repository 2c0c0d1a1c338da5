// The serving entry points (go-infer_b200/csrc/capi_serve.cu) over the fake
// runtime: stand-ins for their launches count the calls, and one reports a
// wait that gave up as a kernel would, through the error word.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "../../include/goinfer_cuda.h"
#include "model.cuh"
#include "serve.cuh"

namespace {
int launches = 0;
bool expire = false;
int last_tokens = -1;
}  // namespace

namespace gi {
int attn_prepare_device() { return 0; }
int sample_prepare_device() { return 0; }
bool attn_head_dim_ok(int hd) { return hd == 64; }
size_t attn_workspace(const KvCache&, const Attn&, int) { return 256; }
int64_t kv_cache_layout(int, int64_t n, int64_t page, int64_t kv, int64_t hd, int64_t at[4]) {
  at[0] = at[2] = at[3] = 0;
  at[1] = 2 * n * page * kv * hd;
  return 2 * at[1];
}
void rope_freqs(int, int, double, double, double, double, double, double*, double*) {}
cudaError_t kv_write_launch(const KvCache&, const float*, size_t, const float*, size_t, const int32_t*, int n,
                            const float*, size_t, float*, int, const int32_t*, const Rope&, int, cudaStream_t) {
  ++launches;
  last_tokens = n;
  return cudaSuccess;
}
cudaError_t kv_read_launch(const KvCache&, float*, float*, const int32_t*, int n, int, cudaStream_t) {
  ++launches;
  last_tokens = n;
  return cudaSuccess;
}
cudaError_t attn_launch(const KvCache&, const Attn& a, int, cudaStream_t) {
  ++launches;
  if (expire) *a.error = 1;
  expire = false;
  return cudaSuccess;
}
cudaError_t sample_launch(const Sample&, int, cudaStream_t) {
  ++launches;
  return cudaSuccess;
}
int DecodeModel::set_kv_cache(int) { return -2; }
int DecodeModel::start_sampling(const StepSampling&, const float*, int, cudaStream_t) { return -2; }
}  // namespace gi

#define CHECK(x)                                            \
  do {                                                      \
    if (!(x)) {                                             \
      std::printf("line %d: %s (%s)\n", __LINE__, #x, gi_cuda_last_error()); \
      return 1;                                             \
    }                                                       \
  } while (0)

int main() {
  CHECK(gi_cuda_init() == 0);
  void* mem = nullptr;
  CHECK(cudaMalloc(&mem, 1 << 20) == cudaSuccess);
  float* f = static_cast<float*>(mem);
  const int32_t* idx = static_cast<const int32_t*>(mem);
  const gi_cuda_kv_cache_t cache = {GI_TYPE_F16, 4, 16, 1, 64, mem, 1 << 20};
  const gi_cuda_attn_t attn = {1, 4, 1, 0, 1.f};
  auto write = [&](uint32_t n) {
    return gi_cuda_kv_write_dev(&cache, f, 64, f, 64, idx, n, nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr);
  };
  auto read = [&](uint32_t n) { return gi_cuda_kv_read_dev(&cache, f, f, idx, n, nullptr); };
  auto attend = [&] {
    return gi_cuda_attn_dev(&cache, &attn, f, f, 1, 1, nullptr, idx, idx, 1, nullptr, mem, 1 << 20, nullptr);
  };
  auto sample = [&] {
    return gi_cuda_sample_dev(static_cast<int32_t*>(mem), nullptr, f, 8, 1, 8, f, nullptr, nullptr, nullptr, nullptr,
                              nullptr);
  };

  // A wait that gave up in a serving call is reported by the next one, whichever it is, which launches nothing.
  for (int next = 0; next < 4; ++next) {
    auto call = [&] { return next == 0 ? write(1) : next == 1 ? read(1) : next == 2 ? attend() : sample(); };
    launches = 0;
    expire = true;
    CHECK(attend() == 0 && launches == 1);
    CHECK(call() == GI_ERR_TIMEOUT && launches == 1);
    CHECK(std::strstr(gi_cuda_last_error(), "timed out"));
    CHECK(call() == 0 && launches == 2);
  }
  cudaFree(mem);
  std::printf("ok\n");
  return 0;
}
