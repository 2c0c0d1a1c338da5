// serve.cuh -- the operators between a batch's projections and its next
// tokens: rotary positions and the paged KV cache (kvcache.cu), attention
// over it (paged_attn.cu) and sampling (sample.cu).  Argument checks are in
// capi.cu; the launchers here get checked arguments and return a
// cudaError_t of the launch.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

struct __half;  // cuda_fp16.h

namespace gi {

constexpr int kTypeF16 = 1;  // GGML id (pkg/gguf/types.go:25-52)

// A layer's paged cache.  Values: [page][kv head][offset][head_dim], K then
// V; Q8_0 adds fp16 scales of 32 values each, K then V.  A value is the half
// itself, or code * scale rounded to half (see kvcache.cu).
struct KvCache {
  int type = 0;  // kTypeF16 or kTypeQ8_0
  int n_kv_heads = 0, head_dim = 0, page_size = 0, n_pages = 0;
  int page_shift = 0;  // log2(page_size)
  uint8_t *k = nullptr, *v = nullptr;
  __half *ks = nullptr, *vs = nullptr;
};

struct Rope {
  int dim = 0;  // rotated dimensions of a head (even; 0 = none)
  int interleaved = 0;
  const double* freqs = nullptr;  // dim / 2 angles per position
  double mscale = 1.0;
};

// Byte offsets of a cache's four parts in its block; returns the block's size.
int64_t kv_cache_layout(int type, int64_t n_pages, int64_t page_size, int64_t n_kv_heads, int64_t head_dim,
                        int64_t at[4]);

// Frequencies of gi_rope_freqs (include/goinfer_cuda.h), checked arguments.
void rope_freqs(int scaling, int dim, double theta, double factor, double low, double high, double orig_ctx,
                double* freqs, double* mscale);

cudaError_t kv_write_launch(const KvCache& c, const float* k, size_t k_stride, const float* v, size_t v_stride,
                            const int32_t* slots, int n_tokens, const float* q, size_t q_stride, float* q_out,
                            int n_heads, const int32_t* positions, const Rope& rope, int sm_count, cudaStream_t s);
cudaError_t kv_read_launch(const KvCache& c, float* k, float* v, const int32_t* slots, int n_tokens, int sm_count,
                           cudaStream_t s);

struct Attn {
  int n_heads = 0, max_tokens = 0, max_q_len = 0, prefix_len = 0;
  float scale = 0.f;
  float* out = nullptr;  // [n_tokens][n_heads][head_dim]
  const float* q = nullptr;
  int n_seqs = 0, n_tokens = 0;
  const int32_t* q_start = nullptr;  // [n_seqs + 1], or null: one token per sequence
  const int32_t* kv_len = nullptr;   // [n_seqs]
  const int32_t* pages = nullptr;    // [n_seqs][pages_stride]
  int pages_stride = 0;
  const int32_t* prefix_pages = nullptr;
  void* ws = nullptr;
  int* error = nullptr;  // the library's error word
};

int attn_prepare_device();
// Head dimensions paged_attn.cu has kernels for.
bool attn_head_dim_ok(int head_dim);
size_t attn_workspace(const KvCache& c, const Attn& a, int sm_count);
cudaError_t attn_launch(const KvCache& c, const Attn& a, int sm_count, cudaStream_t s);

struct Sample {
  int32_t* ids = nullptr;
  float* prob = nullptr;  // may be null
  const float* logits = nullptr;
  size_t stride = 0;  // floats between rows
  int rows = 0, vocab = 0;
  const float* u = nullptr;
  const float* temperature = nullptr;  // null: 1
  const int32_t* top_k = nullptr;      // null: all
  const float* top_p = nullptr;        // null: 1
  const float* min_p = nullptr;        // null: 0
};

int sample_prepare_device();
cudaError_t sample_launch(const Sample& p, int sm_count, cudaStream_t s);

}  // namespace gi
