// capi_serve.cu -- the entry points of include/goinfer_cuda.h that serve a
// batch from a paged KV cache: argument checks and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "../../include/goinfer_cuda.h"
#include "capi.cuh"
#include "serve.cuh"

namespace {

int fail(int code, const char* what, cudaError_t e = cudaSuccess) { return gi::capi_fail(code, what, e); }

#define GI_CUDA_TRY(call, what)                       \
  do {                                                \
    cudaError_t e_ = (call);                          \
    if (e_ != cudaSuccess) return fail(-5, what, e_); \
  } while (0)

constexpr uint32_t kMaxServeHeads = 1024;
constexpr uint32_t kMaxPositions = INT32_MAX - 255;  // of a sequence: the end of its last tile fits an int
constexpr uint32_t kMaxServeTokens = 1u << 30;  // the launches' sums of them and their blocks fit an int

bool cache_shape_ok(const gi_cuda_kv_cache_t& c) {
  return (c.type == GI_TYPE_F16 || c.type == GI_TYPE_Q8_0) && c.n_pages && c.page_size >= 16 &&
         c.page_size <= 65536 && !(c.page_size & (c.page_size - 1)) &&
         (uint64_t)c.n_pages * c.page_size <= INT32_MAX && c.n_kv_heads && c.n_kv_heads <= kMaxServeHeads &&
         c.head_dim && c.head_dim % 32 == 0 && c.head_dim <= 256;
}

int kv_cache_ref(const gi_cuda_kv_cache_t* c, gi::KvCache* out) {
  if (!c) return fail(-4, "null cache");
  if (c->type != GI_TYPE_F16 && c->type != GI_TYPE_Q8_0) return fail(-2, "unsupported cache type");
  if (!cache_shape_ok(*c)) return fail(-4, "unsupported cache shape");
  int64_t at[4];
  const int64_t need = gi::kv_cache_layout(c->type, c->n_pages, c->page_size, c->n_kv_heads, c->head_dim, at);
  if (!c->data || c->bytes < (size_t)need) return fail(-3, "cache data missing or too small");
  if (reinterpret_cast<uintptr_t>(c->data) & 255) return fail(-4, "cache data must be 256-byte aligned");
  uint8_t* p = static_cast<uint8_t*>(c->data);
  out->type = c->type;
  out->n_kv_heads = (int)c->n_kv_heads;
  out->head_dim = (int)c->head_dim;
  out->page_size = (int)c->page_size;
  out->n_pages = (int)c->n_pages;
  out->page_shift = 0;
  while ((1u << out->page_shift) < c->page_size) ++out->page_shift;
  out->k = p + at[0];
  out->v = p + at[1];
  out->ks = reinterpret_cast<__half*>(p + at[2]);
  out->vs = reinterpret_cast<__half*>(p + at[3]);
  return 0;
}

int attn_ref(const gi::KvCache& c, const gi_cuda_attn_t* d, gi::Attn* a) {
  if (!d) return fail(-4, "null attention description");
  if (!gi::attn_head_dim_ok(c.head_dim)) return fail(-4, "attention takes head dims 64, 96, 128 and 256");
  if (!d->n_heads || d->n_heads > kMaxServeHeads || d->n_heads % c.n_kv_heads)
    return fail(-4, "n_heads must be a multiple of the cache's n_kv_heads");
  if (!d->max_tokens || !d->max_q_len || d->max_q_len > d->max_tokens ||
      (uint64_t)d->max_tokens * d->n_heads > (1u << 30))
    return fail(-4, "max_tokens or max_q_len out of range");
  if (d->prefix_len > (uint64_t)c.n_pages * c.page_size || d->prefix_len > kMaxPositions)
    return fail(-4, "prefix longer than the cache or 2^31 - 256 positions");
  a->n_heads = (int)d->n_heads;
  a->max_tokens = (int)d->max_tokens;
  a->max_q_len = (int)d->max_q_len;
  a->prefix_len = (int)d->prefix_len;
  a->scale = d->scale;
  return 0;
}

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

cudaStream_t stream_of(const gi::CapiCtx& ctx, void* s) { return s ? static_cast<cudaStream_t>(s) : ctx.stream; }

// The device is bound and the kernels' attributes are set.
int serve_ready(gi::CapiCtx* ctx) {
  static bool prepared = false;  // under the mutex
  if (int rc = gi::capi_ready(ctx)) return rc;
  if (!prepared && (gi::attn_prepare_device() || gi::sample_prepare_device()))
    return fail(-5, "kernel attribute set-up", cudaGetLastError());
  prepared = true;
  return 0;
}

// The same for a call that launches.  What it launches ends after it has returned, so a wait that gave up there is
// reported by the next call: programs that make no others would not learn of it.
int launch_ready(gi::CapiCtx* ctx) {
  if (int rc = serve_ready(ctx)) return rc;
  return gi::capi_device_error();
}

}  // namespace

extern "C" {

int gi_rope_freqs(int scaling, uint32_t dim, double theta, double factor, double low, double high, double orig_ctx,
                  double* freqs, double* mscale) {
  if (!freqs || !mscale || dim < 2 || dim % 2 || !(theta > 0)) return fail(-4, "bad rotary arguments");
  if (scaling < GI_ROPE_NONE || scaling > GI_ROPE_YARN) return fail(-2, "unknown rotary scaling");
  if (scaling != GI_ROPE_NONE && !(factor > 0)) return fail(-4, "rotary scaling needs a positive factor");
  if (scaling >= GI_ROPE_LLAMA3 && (!(low > 0) || !(high > low) || !(orig_ctx > 0)))
    return fail(-4, "rotary scaling needs 0 < low < high and orig_ctx");
  gi::rope_freqs(scaling, (int)dim, theta, factor, low, high, orig_ctx, freqs, mscale);
  return 0;
}

int64_t gi_kv_cache_bytes(int type, uint32_t n_pages, uint32_t page_size, uint32_t n_kv_heads, uint32_t head_dim) {
  gi_cuda_kv_cache_t c = {type, n_pages, page_size, n_kv_heads, head_dim, nullptr, 0};
  int64_t at[4];
  return cache_shape_ok(c) ? gi::kv_cache_layout(type, n_pages, page_size, n_kv_heads, head_dim, at) : -1;
}

int gi_cuda_kv_write_dev(const gi_cuda_kv_cache_t* cache, const float* k, size_t k_stride, const float* v,
                         size_t v_stride, const int32_t* slots, uint32_t n_tokens, const float* q, size_t q_stride,
                         float* q_out, uint32_t n_heads, const int32_t* positions, const gi_cuda_rope_t* rope,
                         void* stream) {
  gi::KvCache c;
  if (int rc = kv_cache_ref(cache, &c)) return rc;
  if (!k || !v || !slots || (q && !q_out)) return fail(-4, "null device pointer");
  if (!q) n_heads = 0;
  if (q && (!n_heads || n_heads > kMaxServeHeads)) return fail(-4, "n_heads out of range");
  if (n_tokens > kMaxServeTokens) return fail(-4, "too many tokens");
  if (misaligned(k) || misaligned(v) || misaligned(q) || misaligned(q_out) || k_stride % 4 || v_stride % 4 ||
      (q && q_stride % 4))
    return fail(-4, "rows must be 16-byte aligned");
  const size_t kv_row = (size_t)c.n_kv_heads * c.head_dim;
  if (n_tokens > 1 && (k_stride < kv_row || v_stride < kv_row || (q && q_stride < (size_t)n_heads * c.head_dim)))
    return fail(-4, "a stride is shorter than its row");
  gi::Rope r;
  if (rope && rope->dim) {
    if (!rope->freqs || !positions) return fail(-4, "rotary positions need freqs and positions");
    if (rope->dim % 2 || rope->dim > cache->head_dim) return fail(-4, "rotary dim must be even and at most head_dim");
    r.dim = (int)rope->dim;
    r.interleaved = rope->interleaved != 0;
    r.freqs = rope->freqs;
    r.mscale = rope->mscale;
  }
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = launch_ready(&ctx)) return rc;
  if (!n_tokens) return 0;
  GI_CUDA_TRY(gi::kv_write_launch(c, k, k_stride, v, v_stride, slots, (int)n_tokens, q, q_stride, q_out, (int)n_heads,
                                  positions, r, ctx.sm_count, stream_of(ctx, stream)),
              "cache write");
  return 0;
}

int gi_cuda_kv_read_dev(const gi_cuda_kv_cache_t* cache, float* k, float* v, const int32_t* slots, uint32_t n_tokens,
                        void* stream) {
  gi::KvCache c;
  if (int rc = kv_cache_ref(cache, &c)) return rc;
  if (!k || !v || !slots) return fail(-4, "null device pointer");
  if (n_tokens > kMaxServeTokens) return fail(-4, "too many tokens");
  if (misaligned(k) || misaligned(v)) return fail(-4, "rows must be 16-byte aligned");
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = launch_ready(&ctx)) return rc;
  if (!n_tokens) return 0;
  GI_CUDA_TRY(gi::kv_read_launch(c, k, v, slots, (int)n_tokens, ctx.sm_count, stream_of(ctx, stream)), "cache read");
  return 0;
}

int64_t gi_cuda_attn_workspace(const gi_cuda_kv_cache_t* cache, const gi_cuda_attn_t* attn) {
  gi::KvCache c;
  gi::Attn a;
  if (int rc = kv_cache_ref(cache, &c)) return rc;
  if (int rc = attn_ref(c, attn, &a)) return rc;
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = serve_ready(&ctx)) return rc;
  return (int64_t)gi::attn_workspace(c, a, ctx.sm_count);
}

int gi_cuda_attn_dev(const gi_cuda_kv_cache_t* cache, const gi_cuda_attn_t* attn, float* out, const float* q,
                     uint32_t n_seqs, uint32_t n_tokens, const int32_t* q_start, const int32_t* kv_len,
                     const int32_t* pages, uint32_t pages_stride, const int32_t* prefix_pages, void* workspace,
                     size_t workspace_bytes, void* stream) {
  gi::KvCache c;
  gi::Attn a;
  if (int rc = kv_cache_ref(cache, &c)) return rc;
  if (int rc = attn_ref(c, attn, &a)) return rc;
  if (!out || !q || !kv_len || !pages || (a.prefix_len && !prefix_pages)) return fail(-4, "null device pointer");
  if (n_tokens > attn->max_tokens) return fail(-4, "more tokens than the call was described for");
  if (n_seqs > attn->max_tokens) return fail(-4, "more sequences than max_tokens");
  if (!q_start && n_tokens != n_seqs) return fail(-4, "without q_start a sequence has one token");
  if (!pages_stride || (uint64_t)pages_stride * c.page_size > kMaxPositions)
    return fail(-4, "pages_stride out of range");
  if (misaligned(out) || misaligned(q)) return fail(-4, "rows must be 16-byte aligned");
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = launch_ready(&ctx)) return rc;
  const size_t need = gi::attn_workspace(c, a, ctx.sm_count);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(-4, "workspace missing, too small or not 256-byte aligned");
  if (!n_seqs || !n_tokens) return 0;
  a.out = out;
  a.q = q;
  a.n_seqs = (int)n_seqs;
  a.n_tokens = (int)n_tokens;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.pages = pages;
  a.pages_stride = (int)pages_stride;
  a.prefix_pages = prefix_pages;
  a.ws = workspace;
  a.error = ctx.error;
  GI_CUDA_TRY(gi::attn_launch(c, a, ctx.sm_count, stream_of(ctx, stream)), "attention");
  return 0;
}

int gi_cuda_sample_dev(int32_t* ids, float* prob, const float* logits, size_t logits_stride, uint32_t rows,
                       uint32_t vocab, const float* u, const float* temperature, const int32_t* top_k,
                       const float* top_p, const float* min_p, void* stream) {
  if (!vocab || vocab > (1u << 20)) return fail(-4, "vocab out of range");
  if (!ids || !logits || !u) return fail(-4, "null device pointer");
  if (rows > (1u << 20) || (rows > 1 && logits_stride < vocab)) return fail(-4, "rows or logits_stride out of range");
  gi::Sample p;
  p.ids = ids;
  p.prob = prob;
  p.logits = logits;
  p.stride = logits_stride;
  p.rows = (int)rows;
  p.vocab = (int)vocab;
  p.u = u;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = launch_ready(&ctx)) return rc;
  if (!rows) return 0;
  GI_CUDA_TRY(gi::sample_launch(p, ctx.sm_count, stream_of(ctx, stream)), "sampling");
  return 0;
}

int gi_cuda_model_set_kv_cache(gi_cuda_model_t model, int type) {
  if (type != GI_TYPE_F32 && type != GI_TYPE_F16 && type != GI_TYPE_Q8_0) return fail(-2, "unsupported cache type");
  if (!model) return fail(-4, "null model");
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = serve_ready(&ctx)) return rc;
  gi::ModelHandle* h = static_cast<gi::ModelHandle*>(model);
  GI_CUDA_TRY(cudaStreamSynchronize(ctx.stream), "cache type");
  h->m.drop_graphs();  // captured with the other cache
  int rc = -5;
  try {
    rc = h->m.set_kv_cache(type);
  } catch (...) {  // no memory for the tables on the host
  }
  if (rc == -2) return fail(rc, "the persistent layers and tensor parallelism need the float32 cache");
  if (rc == -4) return fail(rc, "F16 and Q8_0 caches take head dims 64, 96, 128 and 256");
  if (rc) return fail(rc, "cache buffers", cudaGetLastError());
  h->m.reset_cache(ctx.stream);
  GI_CUDA_TRY(cudaStreamSynchronize(ctx.stream), "empty cache");
  return 0;
}

int gi_cuda_model_generate_sampled(gi_cuda_model_t model, const int32_t* tokens, uint32_t n_tokens,
                                   uint32_t start_pos, uint32_t n_gen, float temperature, int32_t top_k, float top_p,
                                   float min_p, const float* u, uint32_t* out_tokens, float* out_logits,
                                   float* decode_ms) {
  if (!model || !tokens || !out_tokens || !u || n_tokens < 1 || n_gen < 1) return fail(-4, "bad generate arguments");
  std::lock_guard<std::mutex> lk(gi::capi_mutex());
  gi::CapiCtx ctx;
  if (int rc = serve_ready(&ctx)) return rc;
  gi::ModelHandle* h = static_cast<gi::ModelHandle*>(model);
  if (h->m.cfg().vocab > (1 << 20)) return fail(-4, "vocab out of range");
  gi::StepSampling p;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  auto begin = [&](int steps, cudaStream_t s) {
    std::vector<float> all((size_t)steps, 0.f);  // the prompt's steps pick nothing that is used
    std::copy(u, u + n_gen, all.begin() + (n_tokens - 1));
    const int rc = h->m.start_sampling(p, all.data(), steps, s);
    if (rc == -2) return fail(rc, "sampling under tensor parallelism");
    return rc ? fail(rc, "sampling buffers", cudaGetLastError()) : 0;
  };
  int rc = 0;
  try {
    rc = gi::model_generate(h, tokens, n_tokens, start_pos, n_gen, begin, out_tokens, out_logits, decode_ms);
  } catch (...) {
    rc = fail(-5, "no host memory for the uniform numbers");
  }
  h->m.stop_sampling();
  return rc;
}

}  // extern "C"
