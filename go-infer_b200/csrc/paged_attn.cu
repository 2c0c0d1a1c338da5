// paged_attn.cu -- grouped-query attention of a ragged batch over the paged
// KV cache, with an optional prefix that every sequence sees (the work of
// AttentionGQABatch over paged_kv.go's pages and prefix_cache.go's shared
// prompts).
//
// Sequence b has len = kv_len[b] cached positions in its own pages, the last
// `new` of which are its tokens q_start[b] .. q_start[b+1] - 1 of this call.
// Token j of them sees the whole prefix and its own positions below
// len - new + j + 1; with nothing to see its row is 0.  Softmax statistics
// and sums are float32.
#include "common.cuh"
#include "gemv.cuh"
#include "serve.cuh"

namespace gi {
namespace {

constexpr int kAttnThreads = 256;

GI_DEVINL float cached(const KvCache& c, const uint8_t* plane, const __half* scales, size_t at) {
  if (c.type == kTypeF16) return __half2float(reinterpret_cast<const __half*>(plane)[at]);
  return __half2float(__hmul(__int2half_rn(reinterpret_cast<const int8_t*>(plane)[at]), scales[at >> 5]));
}

// One (token, head) per block; a warp takes every 8th position and holds
// head_dim / 32 dimensions per lane.
template <int HD>
__global__ void __launch_bounds__(kAttnThreads) attn_rows_kernel(KvCache c, Attn a) {
  constexpr int E = HD / 32, W = kAttnThreads / 32;
  __shared__ float so[W][HD], sm[W], sl[W];
  const int token = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = h / (a.n_heads / c.n_kv_heads);
  int b = 0, start = 0, end = 0;
  for (; b < a.n_seqs; ++b) {
    start = a.q_start ? a.q_start[b] : b;
    end = a.q_start ? a.q_start[b + 1] : b + 1;
    if (token >= start && token < end) break;
  }
  if (b == a.n_seqs) return;  // behind the last sequence
  const int own = max(0, min(a.kv_len[b], a.pages_stride * c.page_size));
  const int seen = max(0, min(own, own - (end - start) + (token - start) + 1));
  const size_t row = ((size_t)token * a.n_heads + h) * HD;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = a.q[row + lane + 32 * e] * a.scale;
    o[e] = 0.f;
  }
  for (int t = warp; t < a.prefix_len + seen; t += W) {
    const int p = t < a.prefix_len ? t : t - a.prefix_len;
    const int page = t < a.prefix_len ? a.prefix_pages[p >> c.page_shift]
                                      : a.pages[(size_t)b * a.pages_stride + (p >> c.page_shift)];
    if (page < 0 || page >= c.n_pages) continue;
    const size_t at =
        (((size_t)page * c.n_kv_heads + g) << c.page_shift | (p & (c.page_size - 1))) * HD + lane;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], cached(c, c.k, c.ks, at + 32 * e), s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : expf(m - mn), w = expf(s - mn);
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * cached(c, c.v, c.vs, at + 32 * e);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane + 32 * e] = o[e];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < W; ++w) L += sm[w] == -INFINITY ? 0.f : sl[w] * expf(sm[w] - M);
  for (int d = threadIdx.x; d < HD; d += kAttnThreads) {
    float x = 0.f;
    for (int w = 0; w < W; ++w) x += sm[w] == -INFINITY ? 0.f : so[w][d] * expf(sm[w] - M);
    a.out[row + d] = L > 0.f ? x / L : 0.f;
  }
}

}  // namespace

int attn_prepare_device() { return 0; }

bool attn_head_dim_ok(int hd) { return hd == 64 || hd == 96 || hd == 128 || hd == 256; }

size_t attn_workspace(const KvCache&, const Attn&, int) { return 0; }

cudaError_t attn_launch(const KvCache& c, const Attn& a, int, cudaStream_t s) {
  const dim3 grid(a.n_tokens, a.n_heads);
  switch (c.head_dim) {
    case 64: attn_rows_kernel<64><<<grid, kAttnThreads, 0, s>>>(c, a); break;
    case 96: attn_rows_kernel<96><<<grid, kAttnThreads, 0, s>>>(c, a); break;
    case 128: attn_rows_kernel<128><<<grid, kAttnThreads, 0, s>>>(c, a); break;
    default: attn_rows_kernel<256><<<grid, kAttnThreads, 0, s>>>(c, a); break;
  }
  return cudaGetLastError();
}

}  // namespace gi
