// paged.cuh -- what the kernels of paged_attn.cu and wide_attn.cu share: the
// rows and positions of a launch, and the line of tiles that its CTAs cut
// into equal runs.
#pragma once

#include "common.cuh"
#include "serve.cuh"

namespace gi {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

GI_DEVINL float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 16 bytes to shared memory, of which the first `bytes` (16 or 0) are read.
GI_DEVINL void cp_async16_or_zero(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Four int8 codes as two half2 (exact): 0x6400 + (c + 128) is the half
// 1152 + c.
GI_DEVINL void codes_to_h2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  lo = hsub2_u32(prmt(w, 0x64646464u, 0x4140), 0x64806480u);
  hi = hsub2_u32(prmt(w, 0x64646464u, 0x4342), 0x64806480u);
}

// The positions and rows one launch covers: every sequence's own positions,
// or the shared prefix as one sequence whose rows are all tokens.
struct Pass {
  const float* q;
  float* out;   // rows of whole units: finished, or with ml not null the sums alone
  float2* ml;   // [token][head] (m, sum) of whole units
  float* parts;  // of units cut between CTAs, two slots per CTA
  long long* line;  // [0] tiles per CTA, [1 + b] sequence b's first tile
  const int32_t *q_start, *kv_len, *pages;
  int pages_stride, n_seqs, n_tokens, n_heads;
  int prefix;  // > 0: the prefix pass, of that many positions; n_seqs still counts the sequences
  float scale;
  int unit_cost;  // see span_of
  int beside;     // launched to run beside the kernel before it, whose results it does not read
};

struct Seq {
  int start, fresh, len;  // first token, new tokens, positions
};

GI_DEVINL Seq seq_of(const Pass& p, int b, int page_shift) {
  Seq s;
  const int first = p.prefix ? 0 : b, last = p.prefix ? p.n_seqs : b + 1;
  s.start = max(0, min(p.q_start ? p.q_start[first] : first, p.n_tokens));
  s.fresh = max(s.start, min(p.q_start ? p.q_start[last] : last, p.n_tokens)) - s.start;
  s.len = p.prefix ? p.prefix : max(0, min(p.kv_len[b], p.pages_stride << page_shift));
  return s;
}

// Positions of the sequence that new token j sees.
GI_DEVINL int seen_by(const Pass& p, const Seq& s, int j) {
  return p.prefix ? s.len : max(0, min(s.len, s.len - s.fresh + j + 1));
}

// a / b, which fits an int; a >= 0
GI_DEVINL int quotient(long long a, int b) {
  return a < (1ll << 32) ? (int)((uint32_t)a / (uint32_t)b) : (int)(a / b);
}

// A sequence's units: rt row tiles per kv head; a unit takes unit_cost places
// of the line (its start and end) and then one for each of its tl tiles.
struct Span {
  int rt, tl, unit;  // unit: places of one
  long long places;
};
GI_DEVINL Span span_of(const Pass& p, const Seq& s, int group, int kv_heads, int rows, int tt) {
  Span n;
  n.rt = (s.fresh * group + rows - 1) / rows;  // rows: a power of two; n_tokens * n_heads fits an int
  n.tl = max(1, (s.len + tt - 1) / tt);
  n.unit = n.tl + p.unit_cost;
  n.places = (long long)n.rt * n.unit * kv_heads;
  return n;
}

// A pass's tiles: query rows of a unit, positions of a tile, floats of a part.
struct Rows {
  int rows, tt, part;
};

// A CTA's run of the line: places [pos, end), beginning in sequence b, whose first place is `first`.
struct Run {
  long long pos, end, first;
  int b;
};

// Cuts the line into equal runs, at least `least` places each; false for a CTA
// without one.  By every thread of the CTA; CTA 0 writes p.line.
template <int THREADS>
GI_DEVINL bool run_of_line(const KvCache& c, const Pass& p, int group, int rows, int tt, int least, Run* run) {
  constexpr int W = THREADS / 32;
  __shared__ long long s_scan[W], s_first;
  __shared__ int s_seq;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n_seqs = p.prefix ? 1 : p.n_seqs;
  const int per = (n_seqs + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, n_seqs), b1 = min(b0 + per, n_seqs);
  long long mine = 0;
  for (int b = b0; b < b1; ++b)
    mine += span_of(p, seq_of(p, b, c.page_shift), group, c.n_kv_heads, rows, tt).places;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  const long long chunk = max((total + gridDim.x - 1) / (long long)gridDim.x, (long long)least);
  run->pos = (long long)blockIdx.x * chunk;
  run->end = min(total, run->pos + chunk);
  if (blockIdx.x == 0) {
    if (tid == 0) p.line[0] = chunk;
    long long at = before;
    for (int b = b0; b < b1; ++b) {
      p.line[1 + b] = at;
      at += span_of(p, seq_of(p, b, c.page_shift), group, c.n_kv_heads, rows, tt).places;
    }
  }
  if (run->pos >= run->end) return false;
  if (run->pos >= before && run->pos < before + mine) {
    long long at = before;
    int b = b0;
    for (;; ++b) {
      const long long n = span_of(p, seq_of(p, b, c.page_shift), group, c.n_kv_heads, rows, tt).places;
      if (run->pos < at + n) break;
      at += n;
    }
    s_seq = b;
    s_first = at;
  }
  __syncthreads();
  run->b = s_seq;
  run->first = s_first;
  return true;
}

// wide_attn.cu: a pass in units of 128 query rows.
bool wide_ok(int head_dim, int rows);  // whether it is for units that could have `rows` rows
Rows wide_rows(int head_dim);
int wide_cost();  // Pass::unit_cost of its passes
int wide_prepare();
cudaError_t wide_launch(const KvCache& c, const Pass& p, int sm_count, int* error, cudaStream_t s);

}  // namespace paged
}  // namespace gi
