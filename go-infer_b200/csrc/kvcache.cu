// kvcache.cu -- rotary positions, the paged KV cache as it is written, and
// its rows read back (the work of ApplyRoPE, pkg/math/kernels.go:22-36, and
// of pkg/engine/kvcache.go's F16 / Q8_0 rings and paged_kv.go's pages, for a
// batch of tokens).
//
// Rotation: pair i of a head turns by a = pos * freq_i.  a, cos a and sin a
// are taken in double, because at position 10^5 float32 leaves a few
// hundredths of a radian; the factors are rounded to float32 once and applied as
// attn.cuh does, r0 = x0 c - x1 s and r1 = x0 s + x1 c with every operation
// rounded by itself, so a cache written here holds the same K as the
// decode step's.
//
// Q8_0: the framework's own block rule (quantize.cu, QuantizeQ8_0): 32
// values, d = max|x| / 127 with its fp16 mantissa cut off, code =
// round-half-away(clamp(x / d)).  A cached value is code * d rounded to half
// precision (at most 2^-11 of the value, 1/8 of the half step of a code near
// 127), because the attention's tensor-core products take halves; every
// reader uses that same value.  What would not be finite is not stored: NaN is
// written as 0 and magnitudes end at 65504, so one bad token cannot reach
// the other rows of a batch through P * V.
#include <cmath>

#include "../../include/goinfer_cuda.h"
#include "common.cuh"
#include "gemv.cuh"
#include "paged.cuh"
#include "serve.cuh"

namespace gi {
namespace {

using paged::codes_to_h2;

constexpr int kWriteThreads = 256;
constexpr int kReadAhead = 4;
constexpr int kMaxHeadDim = 256;

// fp32 >= 0 -> fp16 bits by cutting the mantissa (go-infer's FP32ToFP16);
// x <= 65504 / 127, so no overflow.
GI_DEVINL uint32_t f16_cut(float x) {
  const uint32_t b = __float_as_uint(x);
  const int e = (int)(b >> 23) - 112;
  if (e > 0) return ((uint32_t)e << 10) | ((b >> 13) & 0x3FFu);
  if (e < -10) return 0u;
  return ((b & 0x7FFFFFu) | 0x800000u) >> (14 - e);
}

// i / d for 8 <= d and i d < 2^34: the kernels below divide twice per 16 bytes of
// output, and integer division alone kept their issue slots 80 % busy.
struct Divide {
  uint32_t m;
  explicit Divide(uint32_t d) : m((uint32_t)((1ull << 34) / d + 1)) {}
  GI_DEVINL int operator()(int i) const { return (int)(__umulhi((uint32_t)i, m) >> 2); }
};

GI_DEVINL float finite_half(float x) { return x != x ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

// A block's token: 4-value chunks of its q heads, K heads and V heads, one
// per thread and step.  Chunk t of a head holds dimensions 4t .. 4t + 3, so
// the 8 lanes of an aligned group of 8 hold one Q8_0 block.
template <int TYPE>
__global__ void __launch_bounds__(kWriteThreads) kv_write_kernel(
    KvCache c, const float* __restrict__ k, size_t k_stride, const float* __restrict__ v, size_t v_stride,
    const int32_t* __restrict__ slots, const float* __restrict__ q, size_t q_stride, float* __restrict__ q_out,
    int n_heads, const int32_t* __restrict__ positions, Rope rope, int per_block, Divide by_hd4) {
  __shared__ float2 cs[kMaxHeadDim / 2];
  griddep_wait();
  griddep_launch_dependents();
  const int token = blockIdx.x;
  const int half = rope.dim >> 1;
  if (half) {
    const double pos = (double)positions[token];
    for (int i = threadIdx.x; i < half; i += kWriteThreads) {
      double sn, cn;
      sincos(pos * rope.freqs[i], &sn, &cn);
      cs[i] = make_float2((float)(cn * rope.mscale), (float)(sn * rope.mscale));
    }
    __syncthreads();
  }
  const int hd4 = c.head_dim >> 2;
  const int q_chunks = n_heads * hd4, kv_chunks = c.n_kv_heads * hd4;
  const int slot = slots[token];
  const bool kept = slot >= 0 && (slot >> c.page_shift) < c.n_pages;
  const int end = min(q_chunks + (kept ? 2 * kv_chunks : 0), (int)(blockIdx.y + 1) * per_block);
  for (int i = blockIdx.y * per_block + threadIdx.x; i < end; i += kWriteThreads) {
    const int part = i < q_chunks ? 0 : i < q_chunks + kv_chunks ? 1 : 2;  // q, K or V
    const int j = part == 0 ? i : part == 1 ? i - q_chunks : i - q_chunks - kv_chunks;
    const float* row = part == 0 ? q + (size_t)token * q_stride
                       : part == 1 ? k + (size_t)token * k_stride : v + (size_t)token * v_stride;
    const int head = by_hd4(j), d = (j - head * hd4) * 4;
    row += head * c.head_dim;
    const float4 own = *reinterpret_cast<const float4*>(row + d);
    float x[4] = {own.x, own.y, own.z, own.w};
    if (part < 2 && d < rope.dim) {
      if (rope.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          if (d + e >= rope.dim) break;
          const float2 r = cs[(d + e) >> 1];
          const float x0 = x[e], x1 = x[e + 1];
          x[e] = __fsub_rn(__fmul_rn(x0, r.x), __fmul_rn(x1, r.y));
          x[e + 1] = __fadd_rn(__fmul_rn(x0, r.y), __fmul_rn(x1, r.x));
        }
      } else if ((half & 3) == 0) {  // the partners are a whole chunk
        const bool low = d < half;
        const float4 o = *reinterpret_cast<const float4*>(row + (low ? d + half : d - half));
        const float p[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 r = cs[(low ? d : d - half) + e];
          x[e] = low ? __fsub_rn(__fmul_rn(x[e], r.x), __fmul_rn(p[e], r.y))
                     : __fadd_rn(__fmul_rn(p[e], r.y), __fmul_rn(x[e], r.x));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int de = d + e;
          if (de >= rope.dim) break;
          const bool low = de < half;
          const float p = row[low ? de + half : de - half];
          const float2 r = cs[low ? de : de - half];
          x[e] = low ? __fsub_rn(__fmul_rn(x[e], r.x), __fmul_rn(p, r.y))
                     : __fadd_rn(__fmul_rn(p, r.y), __fmul_rn(x[e], r.x));
        }
      }
    }
    if (part == 0) {
      *reinterpret_cast<float4*>(q_out + ((size_t)token * n_heads + head) * c.head_dim + d) =
          make_float4(x[0], x[1], x[2], x[3]);
      continue;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = finite_half(x[e]);
    const size_t at =
        (((size_t)(slot >> c.page_shift) * c.n_kv_heads + head) << c.page_shift | (slot & (c.page_size - 1))) *
            c.head_dim + d;
    uint8_t* plane = part == 1 ? c.k : c.v;
    if (TYPE == kTypeF16) {
      *reinterpret_cast<uint2*>(plane + 2 * at) = make_uint2(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]));
      continue;
    }
    float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    const unsigned group = 0xFFu << (threadIdx.x & 24);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(group, m, o));
    const uint32_t h = f16_cut(__fdiv_rn(m, 127.f));
    const float scale = __half2float(__ushort_as_half((unsigned short)h));
    const float inv = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = fminf(fmaxf(__fmul_rn(x[e], inv), -128.f), 127.f);
      codes |= ((uint32_t)(int)roundf(y) & 0xFFu) << (8 * e);
    }
    *reinterpret_cast<uint32_t*>(plane + at) = codes;
    if ((threadIdx.x & 7) == 0) (part == 1 ? c.ks : c.vs)[at >> 5] = __ushort_as_half((unsigned short)h);
  }
}

// A CTA's tokens: 4-value chunks of their K and V rows, kReadAhead per thread
// and step with all loads before the first store.  Whole tokens, in the order
// of the output: 30011 tokens of 8 heads of 128 take 54 us (5.8 TB/s).  It took
// 72 us while indexes were divided by division, and 79 us in another order, 16
// tokens of one head in a row, which lie side by side in the cache.
template <int TYPE>
__global__ void __launch_bounds__(kWriteThreads) kv_read_kernel(KvCache c, float* __restrict__ k,
                                                                float* __restrict__ v,
                                                                const int32_t* __restrict__ slots, int n_tokens,
                                                                int per_cta, int span, Divide by_row,
                                                                Divide by_hd4) {
  const int hd4 = c.head_dim >> 2, row4 = c.n_kv_heads * hd4;
  const int first = blockIdx.x * per_cta;
  const int end = min(min(per_cta, n_tokens - first) * 2 * row4, (int)(blockIdx.y + 1) * span);
  for (int i0 = blockIdx.y * span + threadIdx.x; i0 < end; i0 += kReadAhead * kWriteThreads) {
    float* to[kReadAhead];
    uint2 w[kReadAhead];
    __half scale[kReadAhead];
#pragma unroll
    for (int a = 0; a < kReadAhead; ++a) {
      const int i = i0 + a * kWriteThreads;
      to[a] = nullptr;
      if (i >= end) continue;
      const int local = by_row(i), token = first + local;
      int j = i - local * 2 * row4;
      const bool is_v = j >= row4;
      if (is_v) j -= row4;
      const int head = by_hd4(j), d = (j - head * hd4) * 4;
      const int slot = __ldg(slots + token);
      if (slot < 0 || (slot >> c.page_shift) >= c.n_pages) continue;
      const size_t at =
          (((size_t)(slot >> c.page_shift) * c.n_kv_heads + head) << c.page_shift | (slot & (c.page_size - 1))) *
              c.head_dim + d;
      const uint8_t* plane = is_v ? c.v : c.k;
      if (TYPE == kTypeF16) {
        w[a] = __ldg(reinterpret_cast<const uint2*>(plane + 2 * at));
      } else {
        w[a].x = __ldg(reinterpret_cast<const uint32_t*>(plane + at));
        scale[a] = (is_v ? c.vs : c.ks)[at >> 5];
      }
      to[a] = (is_v ? v : k) + ((size_t)token * c.n_kv_heads + head) * c.head_dim + d;
    }
#pragma unroll
    for (int a = 0; a < kReadAhead; ++a) {
      if (!to[a]) continue;
      uint2 h = w[a];
      if (TYPE == kTypeQ8_0) {
        uint32_t lo, hi;
        codes_to_h2(w[a].x, lo, hi);
        const uint32_t s = __half_as_ushort(scale[a]), s2 = s | (s << 16);
        h = make_uint2(hmul2_u32(lo, s2), hmul2_u32(hi, s2));
      }
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
      __stcs(reinterpret_cast<float4*>(to[a]), make_float4(x.x, x.y, y.x, y.y));
    }
  }
}

}  // namespace

int64_t kv_cache_layout(int type, int64_t n_pages, int64_t page_size, int64_t n_kv_heads, int64_t head_dim,
                        int64_t at[4]) {
  const int64_t n = n_pages * page_size * n_kv_heads * head_dim;
  auto up = [](int64_t b) { return (b + 255) & ~(int64_t)255; };
  const int64_t val = up(type == kTypeF16 ? 2 * n : n), sc = type == kTypeF16 ? 0 : up(n / 32 * 2);
  at[0] = 0;
  at[1] = val;
  at[2] = 2 * val;
  at[3] = 2 * val + sc;
  return 2 * (val + sc);
}

void rope_freqs(int scaling, int dim, double theta, double factor, double low, double high, double orig_ctx,
                double* freqs, double* mscale) {
  const double two_pi = 6.283185307179586476925286766559;
  *mscale = scaling == GI_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
  // yarn: the (fractional) pair whose angle turns n times over orig_ctx positions
  auto pair_of = [&](double n) { return dim * std::log(orig_ctx / (n * two_pi)) / (2.0 * std::log(theta)); };
  const double first = scaling == GI_ROPE_YARN ? std::fmax(std::floor(pair_of(high)), 0.0) : 0.0;
  const double last = scaling == GI_ROPE_YARN ? std::fmin(std::ceil(pair_of(low)), dim - 1.0) : 0.0;
  for (int i = 0; i < dim / 2; ++i) {
    const double f = 1.0 / std::pow(theta, 2.0 * i / dim);  // as the decode step's table (kernels.go:25-29)
    double r = f;
    if (scaling == GI_ROPE_LINEAR) {
      r = f / factor;
    } else if (scaling == GI_ROPE_LLAMA3) {
      const double wave = two_pi / f, keep = (orig_ctx / wave - low) / (high - low);
      if (wave > orig_ctx / low) r = f / factor;
      else if (wave >= orig_ctx / high) r = (1.0 - keep) * f / factor + keep * f;
    } else if (scaling == GI_ROPE_YARN) {
      const double ramp = std::fmin(std::fmax((i - first) / std::fmax(last - first, 0.001), 0.0), 1.0);
      r = f / factor * ramp + f * (1.0 - ramp);
    }
    freqs[i] = r;
  }
}

cudaError_t kv_write_launch(const KvCache& c, const float* k, size_t k_stride, const float* v, size_t v_stride,
                            const int32_t* slots, int n_tokens, const float* q, size_t q_stride, float* q_out,
                            int n_heads, const int32_t* positions, const Rope& rope, int sm_count, cudaStream_t s) {
  const int chunks = (n_heads + 2 * c.n_kv_heads) * (c.head_dim / 4);
  int parts = (chunks + kWriteThreads - 1) / kWriteThreads;
  const int want = (4 * sm_count + n_tokens - 1) / n_tokens;
  if (parts > want) parts = want;
  const int per = ((chunks + parts - 1) / parts + kWriteThreads - 1) / kWriteThreads * kWriteThreads;
  const dim3 grid(n_tokens, (chunks + per - 1) / per);
  if (c.type == kTypeF16)
    kv_write_kernel<kTypeF16><<<grid, kWriteThreads, 0, s>>>(c, k, k_stride, v, v_stride, slots, q, q_stride, q_out,
                                                             n_heads, positions, rope, per,
                                                             Divide(c.head_dim / 4));
  else
    kv_write_kernel<kTypeQ8_0><<<grid, kWriteThreads, 0, s>>>(c, k, k_stride, v, v_stride, slots, q, q_stride, q_out,
                                                              n_heads, positions, rope, per,
                                                             Divide(c.head_dim / 4));
  return cudaGetLastError();
}

cudaError_t kv_read_launch(const KvCache& c, float* k, float* v, const int32_t* slots, int n_tokens, int sm_count,
                           cudaStream_t s) {
  // Tokens per CTA: enough for a step of every thread, while there is a CTA for every SM; with fewer tokens than
  // SMs a token is spread over CTAs.
  const int chunks = 2 * c.n_kv_heads * (c.head_dim / 4);
  int per = kReadAhead * kWriteThreads / chunks;
  if (per > n_tokens / sm_count) per = n_tokens / sm_count;
  if (per < 1) per = 1;
  int span = per * chunks;
  if (n_tokens < sm_count) span = (span * n_tokens / sm_count / kWriteThreads + 1) * kWriteThreads;
  const dim3 grid((unsigned)((n_tokens + per - 1) / per), (unsigned)((per * chunks + span - 1) / span));
  if (c.type == kTypeF16)
    kv_read_kernel<kTypeF16><<<grid, kWriteThreads, 0, s>>>(c, k, v, slots, n_tokens, per, span, Divide(chunks),
                                                         Divide(c.head_dim / 4));
  else
    kv_read_kernel<kTypeQ8_0><<<grid, kWriteThreads, 0, s>>>(c, k, v, slots, n_tokens, per, span, Divide(chunks),
                                                         Divide(c.head_dim / 4));
  return cudaGetLastError();
}

}  // namespace gi
