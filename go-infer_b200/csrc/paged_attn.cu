// paged_attn.cu -- grouped-query attention of a ragged batch over the paged
// KV cache, with an optional prefix that every sequence sees (the work of
// AttentionGQABatch over paged_kv.go's pages and prefix_cache.go's shared
// prompts).
//
// Sequence b has len = kv_len[b] cached positions in its own pages, the last
// `new` of which are its tokens q_start[b] .. q_start[b+1] - 1 of this call.
// Token j of them sees the whole prefix and its own positions below
// len - new + j + 1; with nothing to see its row is 0.  A row of q that is not
// finite becomes NaN: its scores are, no maximum takes them up (m stays -inf),
// but its sums are NaN, and they are joined whatever m is.
//
// out = sum_t p_t v_t / sum_t p_t, p_t = 2^(s_t - m), s_t = log2(e) scale q.k_t,
// in one pass over the positions with the running maximum m: a tile of
// positions raises m, and what was summed before shrinks by 2^(m_old - m_new).
//
// The products run on the fp16 tensor cores (mma m16n8k16, float32 sums) and
// keep float32's precision where it counts: the cache's values are halves
// already (kvcache.cu), q and p are split into a half and the half of its
// remainder (22 bits).  The 16 rows of an MMA are the high parts of 8 query
// rows over their low parts, so a row's two sums end in one thread.
// q rows are scaled by a power of two to just under 2^14 and p to at most 2^14, which
// keeps the remainders in half's normal range.  An MMA chain is one
// tile long; the running sum over tiles is a float32 FMA, because the tensor
// cores cut their sums instead of rounding them and a chain of thousands of
// positions would drift.
//
// Units of many rows go to wide_attn.cu.
//
// Bound: single tokens read the cache once (HBM).  A unit of work is (sequence, kv
// head, 8 * MT query rows of that head's group): it reads a position once for
// all its rows.  The units' tiles form one line that is cut into equal runs, one per
// CTA, so unequal lengths cost nothing and one long sequence fills the GPU; a
// unit that is cut leaves parts (m, sum, row) that attn_merge_kernel joins in
// order.  Each of a CTA's 4 warps takes every 4th tile of the run through a
// cp.async ring of its own and meets the others only at the end of a unit.
#include "common.cuh"
#include "gemv.cuh"
#include "paged.cuh"
#include "serve.cuh"

namespace gi {
namespace {

using namespace paged;

constexpr int kWarps = 4, kAttnThreads = 32 * kWarps;
constexpr int kMergeThreads = 128;
// A unit's place on the line: kUnitCost tiles for its start and end (its
// queries, the joining of the warps: 9 to 10 thousand clocks, a tile about 900
// per CTA), then its tl tiles.  Without them the CTAs whose runs hold many
// short sequences end last: a batch of 62 sequences of 1 to 8192 positions
// took 135 us instead of 127.
constexpr int kUnitCost = 8;

GI_DEVINL void ldsm_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

// D = A(16x16 f16, row) * B(16x8 f16, col): the first of a chain.
GI_DEVINL void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// The scales of one position's blocks 0 .. N - 1, two halves a register.
template <int N>
GI_DEVINL void load_scales(uint32_t addr, uint32_t (&w)[(N + 1) / 2]) {
  if (N == 2) {
    w[0] = lds32(addr);
  } else if (N == 4) {
    const uint64_t x = lds64(addr);
    w[0] = (uint32_t)x, w[(N + 1) / 2 - 1] = (uint32_t)(x >> 32);
  } else if (N == 8) {
    const uint4 x = lds128(addr);
    w[0] = x.x, w[1 % ((N + 1) / 2)] = x.y, w[2 % ((N + 1) / 2)] = x.z, w[3 % ((N + 1) / 2)] = x.w;
  } else {  // 3: six bytes, even alignment
    w[0] = lds16(addr) | (lds16(addr + 2) << 16);
    w[(N + 1) / 2 - 1] = lds16(addr + 4);
  }
}

__host__ __device__ constexpr int pow2_up(int n) { return n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

// HD head dim, MT groups of 8 query rows per unit, TT positions per tile, NS
// tiles in a warp's ring.
template <int HD, int TYPE, int MT, int TT, int NS>
struct Tile {
  static constexpr int kRows = 8 * MT;
  static constexpr int kElem = TYPE == kTypeF16 ? 2 : 1;
  static constexpr int kPitch = pow2_up(HD * kElem);      // bytes of a position's row in shared memory
  static constexpr int kChunks = HD * kElem / 16;         // 16-byte chunks of a row
  static constexpr int kScaleBytes = TYPE == kTypeF16 ? 0 : HD / 16;  // a position's scales
  static constexpr int kPlane = TT * kPitch, kScales = TT * kScaleBytes;
  static constexpr int kStage = 2 * (kPlane + kScales);
  static constexpr int kQ = MT * (HD / 16) * 512;
  static constexpr int kMerge = kWarps * kRows * HD * 4;
  static constexpr int kRing = kWarps * NS * kStage > kMerge ? kWarps * NS * kStage : kMerge;
  static constexpr int kSmem = kRing + kQ + kWarps * kRows * 8 + kRows * 4;
  static constexpr int kPart = kRows * (HD + 2);  // floats of a part

  // Chunk of row r that holds logical chunk c.  The reads of one instruction
  // touch rows 0, 1, 4, 5, 8, 9, 12, 13 (K) or 0, 4, 8, 12 (V codes); the
  // exclusive-or puts them in different banks.
  GI_DEVINL static int chunk(int r, int c) {
    if (TYPE == kTypeF16) return c ^ (((r & 1) << 2) | ((r >> 2) & 3));
    if (HD == 64) return c ^ (((r >> 2) & 1) << 1);
    return c ^ ((((r ^ (r >> 3)) & 1) | (((r >> 2) & 1) << 1)) << 1);
  }
};

template <int HD, int TYPE, int MT, int TT, int NS, int MINB>
__global__ void __launch_bounds__(kAttnThreads, MINB) attn_tiles_kernel(KvCache c, Pass p) {
  using T = Tile<HD, TYPE, MT, TT, NS>;
  constexpr int NT = TT / 8, NG = TT / 16, NB = HD / 32;
  extern __shared__ __align__(128) uint8_t sm[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / c.n_kv_heads;
  // ---- this CTA's run of the line of tiles ----
  if (!p.beside) griddep_wait();
  griddep_launch_dependents();
  Run run;
  if (!run_of_line<kAttnThreads>(c, p, group, T::kRows, TT, kWarps, &run)) {
    if (p.beside) griddep_wait();  // its end is also the end of the kernel it ran beside
    return;
  }
  long long pos = run.pos, first = run.first;
  const long long end = run.end;
  int b = run.b;

  uint8_t* ring = sm + warp * NS * T::kStage;
  uint8_t* sq = sm + T::kRing;
  float2* s_ml = reinterpret_cast<float2*>(sq + T::kQ);           // [warp][row]
  float* s_fac = reinterpret_cast<float*>(s_ml + kWarps * T::kRows);  // [row]
  const uint32_t ring_u = smem_u32(ring), sq_u = smem_u32(sq);

  while (pos < end) {
    Seq s = seq_of(p, b, c.page_shift);
    Span n = span_of(p, s, group, c.n_kv_heads, T::kRows, TT);
    while (pos >= first + n.places) {
      first += n.places;
      s = seq_of(p, ++b, c.page_shift);
      n = span_of(p, s, group, c.n_kv_heads, T::kRows, TT);
    }
    const long long rel = pos - first;
    const int unit = quotient(rel, n.unit), at0 = (int)(rel - (long long)unit * n.unit);
    const int h = unit / n.rt, row0 = (unit - h * n.rt) * T::kRows;
    const int at1 = (int)min(at0 + (end - pos), (long long)n.unit);
    pos += at1 - at0;
    const int tile0 = max(at0 - p.unit_cost, 0), count = at1 - p.unit_cost - tile0;
    if (count <= 0) break;  // the run ends before the unit's first tile
    const bool whole = count == n.tl;
    const int n_rows = min(T::kRows, s.fresh * group - row0);
    const int seen_first = seen_by(p, s, row0 / group), seen_last = seen_by(p, s, (row0 + n_rows - 1) / group);
    const int tile_end = min(tile0 + count, (seen_last + TT - 1) / TT);
    const int32_t* pages = p.pages + (p.prefix ? 0 : (size_t)b * p.pages_stride);

    // Copies a tile into stage `st`; returns a bit per 16 positions whose page is not in the cache.
    auto issue = [&](int tile, int st) {
      uint32_t bad = 0;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        const int p0 = tile * TT + gr * 16;
        const int page = p0 < s.len ? __ldg(pages + (p0 >> c.page_shift)) : -1;
        const bool ok = (unsigned)page < (unsigned)c.n_pages;
        if (!ok) bad |= 1u << gr;
        const size_t at =
            ((size_t)(ok ? page : 0) * c.n_kv_heads + h << c.page_shift) + (ok ? p0 & (c.page_size - 1) : 0);
        const uint32_t dst = ring_u + st * T::kStage;
        const int left = ok ? s.len - p0 : 0;  // positions of the 16 that exist
#pragma unroll
        for (int i = lane; i < 16 * T::kChunks; i += 32) {
          const int r = i / T::kChunks, ch = i - r * T::kChunks;
          const uint32_t d = dst + (gr * 16 + r) * T::kPitch + T::chunk(r, ch) * 16;
          const size_t src = at * HD * T::kElem + (size_t)i * 16;
          const int bytes = r < left ? 16 : 0;
          cp_async16_or_zero(d, c.k + src, bytes);
          cp_async16_or_zero(d + T::kPlane, c.v + src, bytes);
        }
        if (TYPE == kTypeQ8_0) {
          const uint32_t ds = dst + 2 * T::kPlane + gr * 16 * T::kScaleBytes;
          for (int i = lane; i < T::kScaleBytes; i += 32) {
            const size_t src = at * T::kScaleBytes + (size_t)i * 16;
            const int bytes = i * 16 < left * T::kScaleBytes ? 16 : 0;
            cp_async16_or_zero(ds + i * 16, reinterpret_cast<const uint8_t*>(c.ks) + src, bytes);
            cp_async16_or_zero(ds + T::kScales + i * 16, reinterpret_cast<const uint8_t*>(c.vs) + src, bytes);
          }
        }
      }
      return bad;
    };

    int tile = tile0 + warp;
    uint32_t bad[NS];  // of the stage `st + i`
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) {
      bad[i] = tile + i * kWarps < tile_end ? issue(tile + i * kWarps, i) : 0u;
      cp_async_commit();
    }

    // ---- the unit's queries as MMA operands: a power of two under 2^14 per row, high and low halves ----
#pragma unroll 2
    for (int r = warp; r < T::kRows; r += kWarps) {
      const int row = row0 + r;
      const bool real = r < n_rows;
      const float* q = p.q + ((size_t)(s.start + (real ? row / group : 0)) * p.n_heads + (size_t)h * group +
                              (real ? row % group : 0)) * HD;
      float2 x[(HD / 2 + 31) / 32];
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < (HD / 2 + 31) / 32; ++i) {
        const int d2 = lane + 32 * i;
        x[i] = real && d2 < HD / 2 ? reinterpret_cast<const float2*>(q)[d2] : make_float2(0.f, 0.f);
        m = fmaxf(m, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
      }
      m = warp_max(m);
      const int ex = (int)(__float_as_uint(m) >> 23) - 127;  // m in [2^ex, 2^(ex + 1))
      const int sh = m > 0.f ? min(13 - ex, 126) : 0;
      const float up = exp2i(sh);
      if (lane == 0) s_fac[r] = p.scale * kLog2e * exp2i(-sh);
#pragma unroll
      for (int i = 0; i < (HD / 2 + 31) / 32; ++i) {
        const int d = 2 * (lane + 32 * i);
        if (d >= HD) break;
        // dimension d is byte d % 8 of quad d % 32 / 8's part of block d / 32
        const int ks = (d >> 5) * 2 + ((d >> 2) & 1), reg = (d & 2);
        const uint32_t hi = pack_h2(x[i].x * up, x[i].y * up);
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        const uint32_t lo = pack_h2(x[i].x * up - back.x, x[i].y * up - back.y);
        uint32_t* w = reinterpret_cast<uint32_t*>(
            sq + (((r >> 3) * (HD / 16) + ks) * 32 + (r & 7) * 4 + ((d >> 3) & 3)) * 16);
        w[reg] = hi;
        w[reg + 1] = lo;
      }
    }
    __syncthreads();

    float o[MT][HD / 8][2], m[MT], l[MT], fac[MT];
    int seen[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = mt * 8 + g;
      m[mt] = -INFINITY;
      l[mt] = 0.f;
      fac[mt] = s_fac[r];
      seen[mt] = seen_by(p, s, (row0 + min(r, n_rows - 1)) / group);
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) o[mt][i][0] = o[mt][i][1] = 0.f;
    }

    for (int st = 0; tile < tile_end; tile += kWarps, st = st + 1 == NS ? 0 : st + 1) {
      const uint32_t bad_now = bad[0];
#pragma unroll
      for (int i = 0; i < NS - 2; ++i) bad[i] = bad[i + 1];
      bad[NS - 2] = 0;
      if (tile + (NS - 1) * kWarps < tile_end) bad[NS - 2] = issue(tile + (NS - 1) * kWarps, st == 0 ? NS - 1 : st - 1);
      cp_async_commit();
      cp_async_wait<NS - 1>();
      __syncwarp();
      const uint32_t ku = ring_u + st * T::kStage, vu = ku + T::kPlane, ksu = vu + T::kPlane, vsu = ksu + T::kScales;
      const int p0 = tile * TT;
      if (TYPE == kTypeQ8_0 && p0 + TT > s.len) {  // scales of positions that do not exist may hold anything
        for (int i = lane; i < TT * (HD / 32); i += 32)
          if (p0 + i / (HD / 32) >= s.len)
            *reinterpret_cast<__half*>(ring + st * T::kStage + 2 * T::kPlane + T::kScales + 2 * i) = __half(0.f);
        __syncwarp();
      }

      // S = q K^T: column g of MMA nt is position 16 (nt / 2) + 4 (g / 2) + g % 2 + 2 (nt % 2)
      float sc[MT][NT][4];
      uint32_t kd[NT][(NB + 1) / 2];
      if (TYPE == kTypeQ8_0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          load_scales<NB>(ksu + (16 * (nt >> 1) + 4 * (g >> 1) + (g & 1) + 2 * (nt & 1)) * T::kScaleBytes, kd[nt]);
      }
#pragma unroll
      for (int blk = 0; blk < NB; ++blk) {
        uint4 a[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int k = 0; k < 2; ++k) a[mt][k] = lds128(sq_u + ((mt * (HD / 16) + 2 * blk + k) * 32 + lane) * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int r = 4 * (g >> 1) + (g & 1) + 2 * (nt & 1), row = 16 * (nt >> 1) + r;
          uint32_t kb[4];
          if (TYPE == kTypeF16) {
            const uint4 w = lds128(ku + row * T::kPitch + T::chunk(r, 4 * blk + t) * 16);
            kb[0] = w.x, kb[1] = w.y, kb[2] = w.z, kb[3] = w.w;
          } else {
            const uint64_t w = lds64(ku + row * T::kPitch + T::chunk(r, 2 * blk + (t >> 1)) * 16 + (t & 1) * 8);
            const uint32_t d2 = prmt(kd[nt][blk >> 1], 0u, blk & 1 ? 0x3232 : 0x1010);
            codes_to_h2((uint32_t)w, kb[0], kb[1]);
            codes_to_h2((uint32_t)(w >> 32), kb[2], kb[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) kb[i] = hmul2_u32(kb[i], d2);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            if (blk == 0) mma_16816_first(sc[mt][nt], a[mt][0].x, a[mt][0].y, a[mt][0].z, a[mt][0].w, kb[0], kb[1]);
            else mma_16816(sc[mt][nt], a[mt][0].x, a[mt][0].y, a[mt][0].z, a[mt][0].w, kb[0], kb[1]);
            mma_16816(sc[mt][nt], a[mt][1].x, a[mt][1].y, a[mt][1].z, a[mt][1].w, kb[2], kb[3]);
          }
        }
      }

      // softmax: this thread's positions of row g are 16 (nt / 2) + 4 t + 2 (nt % 2) + {0, 1}
      uint32_t pf[MT][NG][4];
      float alpha[MT];
      const bool masked = p0 + TT > seen_first || bad_now;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float top = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x = (sc[mt][nt][i] + sc[mt][nt][i + 2]) * fac[mt];
            if (masked) {
              const int at = p0 + 16 * (nt >> 1) + 4 * t + 2 * (nt & 1) + i;
              if (at >= seen[mt] || ((bad_now >> (nt >> 1)) & 1)) x = -INFINITY;
            }
            sc[mt][nt][i] = x;
            top = fmaxf(top, x);
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[mt], top), base = mn == -INFINITY ? 0.f : mn;
        alpha[mt] = exp2_approx(m[mt] - base);
        m[mt] = mn;
        float sum = 0.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float x = exp2_approx(sc[mt][nt][0] - base) * 16384.f, y = exp2_approx(sc[mt][nt][1] - base) * 16384.f;
          sum += x + y;
          const uint32_t hi = pack_h2(x, y);
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          pf[mt][nt >> 1][2 * (nt & 1)] = hi;
          pf[mt][nt >> 1][2 * (nt & 1) + 1] = pack_h2(x - back.x, y - back.y);
        }
        l[mt] = l[mt] * alpha[mt] + sum;
      }

      // O += P V
      uint32_t vd[NG][4][(NB + 1) / 2];
      if (TYPE == kTypeQ8_0) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
          for (int i = 0; i < 4; ++i) load_scales<NB>(vsu + (16 * gr + 4 * t + i) * T::kScaleBytes, vd[gr][i]);
      }
#pragma unroll
      for (int blk = 0; blk < NB; ++blk) {
        float acc[MT][4][4];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          uint32_t vb[4][2];
          if (TYPE == kTypeF16) {  // MMA j: dimensions 32 blk + 8 j + (0 .. 7)
            const int i8 = lane & 7, mat = lane >> 3;
            const int r = 4 * (i8 >> 1) + (i8 & 1) + 2 * (mat & 1), row = 16 * gr + r;
#pragma unroll
            for (int j = 0; j < 4; j += 2)
              ldsm_x4_trans(vu + row * T::kPitch + T::chunk(r, 4 * blk + j + (mat >> 1)) * 16, vb[j][0], vb[j][1],
                            vb[j + 1][0], vb[j + 1][1]);
          } else {  // MMA j: dimensions 32 blk + 4 (0 .. 7) + j
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 4 * t + i, row = 16 * gr + r;
              w[i] = lds32(vu + row * T::kPitch + T::chunk(r, 2 * blk + (g >> 2)) * 16 + (g & 3) * 4);
            }
            const uint32_t sel = blk & 1 ? 0x7632 : 0x5410;
            const uint32_t d01 = prmt(vd[gr][0][blk >> 1], vd[gr][1][blk >> 1], sel);
            const uint32_t d23 = prmt(vd[gr][2][blk >> 1], vd[gr][3][blk >> 1], sel);
            uint32_t x[4], y[4];
            codes_to_h2(prmt(w[0], w[1], 0x5140), x[0], x[1]);  // dimensions 0, 1 of positions 0, 1
            codes_to_h2(prmt(w[0], w[1], 0x7362), x[2], x[3]);
            codes_to_h2(prmt(w[2], w[3], 0x5140), y[0], y[1]);
            codes_to_h2(prmt(w[2], w[3], 0x7362), y[2], y[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              vb[j][0] = hmul2_u32(x[j], d01);
              vb[j][1] = hmul2_u32(y[j], d23);
            }
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (gr == 0)
                mma_16816_first(acc[mt][j], pf[mt][gr][0], pf[mt][gr][1], pf[mt][gr][2], pf[mt][gr][3], vb[j][0], vb[j][1]);
              else
                mma_16816(acc[mt][j], pf[mt][gr][0], pf[mt][gr][1], pf[mt][gr][2], pf[mt][gr][3], vb[j][0], vb[j][1]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              o[mt][4 * blk + j][i] = fmaf(o[mt][4 * blk + j][i], alpha[mt], acc[mt][j][i] + acc[mt][j][i + 2]);
      }
      __syncwarp();
    }
    cp_async_wait<0>();

    // ---- the four warps' sums joined ----
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 1);
      l[mt] += __shfl_xor_sync(0xffffffffu, l[mt], 2);
      if (t == 0) s_ml[warp * T::kRows + mt * 8 + g] = make_float2(m[mt], l[mt]);
    }
    __syncthreads();  // also: every ring is free
    float* s_o = reinterpret_cast<float*>(sm) + (size_t)warp * T::kRows * HD;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = mt * 8 + g;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w * T::kRows + r].x);
      const float f = top == -INFINITY ? 0.f : exp2_approx(m[mt] - top);
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const int blk = i >> 2, j = i & 3;
        if (TYPE == kTypeF16) {
          *reinterpret_cast<float2*>(s_o + r * HD + 8 * i + 2 * t) = make_float2(o[mt][i][0] * f, o[mt][i][1] * f);
        } else {
          s_o[r * HD + 32 * blk + 8 * t + j] = o[mt][i][0] * f;
          s_o[r * HD + 32 * blk + 8 * t + 4 + j] = o[mt][i][1] * f;
        }
      }
    }
    __syncthreads();
    float* part = p.parts + (size_t)(2 * blockIdx.x + (tile0 > 0 ? 0 : 1)) * T::kPart;
    for (int i = tid; i < n_rows * (HD / 4); i += kAttnThreads) {
      const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w * T::kRows + r].x);
      const float base = top == -INFINITY ? 0.f : top;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 e = s_ml[w * T::kRows + r];
        sum += e.y * exp2_approx(e.x - base);
        const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm) +
                                                          ((size_t)w * T::kRows + r) * HD + d);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
      if (!whole) {
        *reinterpret_cast<float4*>(part + r * HD + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(part + T::kRows * HD + 2 * r) = make_float2(top, sum);
        continue;
      }
      const int row = row0 + r;
      const size_t at = (size_t)(s.start + row / group) * p.n_heads + (size_t)h * group + row % group;
      if (p.ml) {
        if (d == 0) p.ml[at] = make_float2(top, sum);
      } else {
        const float f = sum > 0.f ? 1.f / sum : 0.f;
        x.x *= f, x.y *= f, x.z *= f, x.w *= f;
      }
      *reinterpret_cast<float4*>(p.out + at * HD + d) = x;
    }
    __syncthreads();
  }
  if (p.beside) griddep_wait();
}

// Joins row (token, head) of the passes' parts, in the order of the
// positions: the prefix, then the sequence's own.  One CTA per (token, kv head).
// Parts come in groups of kAhead, whose loads are in flight together: a row of one
// long sequence has a dozen parts, and each would cost an L2 round trip.
__global__ void __launch_bounds__(kMergeThreads) attn_merge_kernel(KvCache c, Pass own, Rows ro, Pass pre, Rows rp,
                                                                   float* __restrict__ out) {
  constexpr int kAhead = 8;
  __shared__ int s_b;
  const int token = blockIdx.x, h = blockIdx.y, group = own.n_heads / c.n_kv_heads, hd = c.head_dim;
  griddep_wait();
  griddep_launch_dependents();
  int b = token < own.n_seqs ? token : -1;
  if (own.q_start) {  // the last sequence that starts at or before the token and has it
    if (threadIdx.x < 32) {
      int lo = 0, hi = own.n_seqs;  // the answer is in [lo, hi): 32 probes a step
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (int)threadIdx.x * step;
        const unsigned below = __ballot_sync(0xffffffffu, at < hi && own.q_start[at] <= token);
        const int last = 31 - __clz((int)below);
        if (last < 0) break;  // before the first sequence
        hi = min(hi, lo + (last + 1) * step);
        lo += last * step;
      }
      if (threadIdx.x == 0) s_b = own.q_start[lo] <= token && token < own.q_start[lo + 1] ? lo : -1;
    }
    __syncthreads();
    b = s_b;
  }
  if (b < 0) return;
  struct Source {
    Seq s;
    Span n;
    long long chunk, line;
  } src[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 0 && !pre.prefix) continue;
    const Pass& p = k ? own : pre;
    const Rows& w = k ? ro : rp;
    src[k].s = seq_of(p, k ? b : 0, c.page_shift);
    // Only a q_start that does not ascend leaves a token outside the prefix pass's rows: it has no place on that line.
    if (k == 0 && (token < src[k].s.start || token - src[k].s.start >= src[k].s.fresh)) return;
    src[k].n = span_of(p, src[k].s, group, c.n_kv_heads, w.rows, w.tt);
    src[k].chunk = p.line[0];
    src[k].line = p.line[1 + (k ? b : 0)];
  }
  for (int i = threadIdx.x; i < group * (hd / 4); i += kMergeThreads) {
    const int hg = i / (hd / 4), d = (i - hg * (hd / 4)) * 4;
    const size_t at = (size_t)token * own.n_heads + (size_t)h * group + hg;
    float top = -INFINITY, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    bool done = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 0 && !pre.prefix) continue;
      const Pass& p = k ? own : pre;
      const Rows& w = k ? ro : rp;
      const Source& q = src[k];
      const int row = (token - q.s.start) * group + hg, r = row % w.rows;
      const long long u1 = q.line + ((long long)h * q.n.rt + row / w.rows + 1) * q.n.unit, u0 = u1 - q.n.tl;
      const int i0 = quotient(u0, (int)q.chunk), i1 = quotient(u1 - 1, (int)q.chunk);
      if (i0 == i1 && !p.ml) {  // finished by its CTA
        done = true;
        break;
      }
      for (int c0 = i0; c0 <= i1; c0 += kAhead) {
        float2 e[kAhead];
        float4 y[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int ci = c0 + a;
          e[a] = make_float2(-INFINITY, 0.f);
          y[a] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (ci > i1) continue;
          if (i0 == i1) {  // a whole unit's sums
            e[a] = p.ml[at];
            y[a] = *reinterpret_cast<const float4*>(p.out + at * hd + d);
          } else {
            const float* part = p.parts + (size_t)(2 * ci + (ci * q.chunk > u0 ? 0 : 1)) * w.part;
            e[a] = *reinterpret_cast<const float2*>(part + w.rows * hd + 2 * r);
            y[a] = *reinterpret_cast<const float4*>(part + r * hd + d);
          }
        }
        float mn = top;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) mn = fmaxf(mn, e[a].x);
        const float base = mn == -INFINITY ? 0.f : mn;  // nothing seen, or not a number
        const float f0 = exp2_approx(top - base);
        x.x *= f0, x.y *= f0, x.z *= f0, x.w *= f0;
        sum *= f0;
        top = mn;
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const float f = exp2_approx(e[a].x - base);
          x.x = fmaf(y[a].x, f, x.x), x.y = fmaf(y[a].y, f, x.y);
          x.z = fmaf(y[a].z, f, x.z), x.w = fmaf(y[a].w, f, x.w);
          sum = fmaf(e[a].y, f, sum);
        }
      }
    }
    if (done) continue;
    const float f = sum > 0.f ? 1.f / sum : 0.f;
    *reinterpret_cast<float4*>(out + at * hd + d) = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
  }
}

// ---- launch choices -----------------------------------------------------------
typedef void (*TilesKernel)(KvCache, Pass);
struct Choice {
  TilesKernel fn;  // null: wide_attn.cu
  int smem, per_sm;
  Rows rows;
};

template <int HD, int TYPE, int MT, int TT, int NS, int MINB>
Choice choice() {
  using T = Tile<HD, TYPE, MT, TT, NS>;
  return {attn_tiles_kernel<HD, TYPE, MT, TT, NS, MINB>, T::kSmem, MINB, {T::kRows, TT, T::kPart}};
}

// The kernel for units of `rows` query rows.
template <int HD, int TYPE>
Choice choose(int rows) {
  constexpr int wide = TYPE == kTypeF16 || HD == 256 ? 16 : 32;
  constexpr int few = HD == 256 ? (TYPE == kTypeF16 ? 1 : 2) : 3;
  if (rows <= 8) return choice<HD, TYPE, 1, wide, 2, few>();
  if (rows <= 16 || HD == 256) return choice<HD, TYPE, 2, 16, 2, HD == 256 ? 1 : 3>();
  return choice<HD, TYPE, HD == 256 ? 2 : 4, 16, 2, HD == 256 ? 1 : 2>();
}

Choice choose(const KvCache& c, int rows) {
  if (wide_ok(c.head_dim, rows)) return {nullptr, 0, 1, wide_rows(c.head_dim)};
  const bool f16 = c.type == kTypeF16;
  switch (c.head_dim) {
    case 64: return f16 ? choose<64, kTypeF16>(rows) : choose<64, kTypeQ8_0>(rows);
    case 96: return f16 ? choose<96, kTypeF16>(rows) : choose<96, kTypeQ8_0>(rows);
    case 128: return f16 ? choose<128, kTypeF16>(rows) : choose<128, kTypeQ8_0>(rows);
    default: return f16 ? choose<256, kTypeF16>(rows) : choose<256, kTypeQ8_0>(rows);
  }
}

// A launch whose CTAs may come up before the kernel in front of it has ended (`early`; they wait where they
// read its results), or after it.
template <typename... K, typename... A>
cudaError_t launch_after(dim3 grid, int threads, int smem, cudaStream_t s, bool early, void (*k)(K...), A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, static_cast<K>(args)...);
}

// The workspace: each pass's line and parts, and with a prefix the whole units' sums of both.
struct Layout {
  size_t line[2], parts[2], ml[2], sums, bytes;
};
Layout layout(const KvCache& c, const Attn& a, const Choice& own, const Choice& pre, int sm_count) {
  Layout w = {};
  auto take = [&](size_t bytes) {
    const size_t at = w.bytes;
    w.bytes += (bytes + 255) & ~(size_t)255;
    return at;
  };
  const size_t rows = (size_t)a.max_tokens * a.n_heads;
  w.line[0] = take(8 * ((size_t)a.max_tokens + 1));
  w.parts[0] = take(sizeof(float) * 2 * own.per_sm * sm_count * own.rows.part);
  if (a.prefix_len) {
    w.line[1] = take(16);
    w.parts[1] = take(sizeof(float) * 2 * pre.per_sm * sm_count * pre.rows.part);
    for (size_t& m : w.ml) m = take(8 * rows);
    w.sums = take(sizeof(float) * rows * c.head_dim);
  }
  return w;
}

int rows_of(long long tokens, int group) { return (int)(tokens * group < 1024 ? tokens * group : 1024); }

template <int HD, int TYPE>
int prepare() {
  for (int rows : {8, 16, 32}) {
    const Choice k = choose<HD, TYPE>(rows);
    if (cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem) != cudaSuccess) return -5;
  }
  return 0;
}

}  // namespace

int attn_prepare_device() {
  return prepare<64, kTypeF16>() || prepare<64, kTypeQ8_0>() || prepare<96, kTypeF16>() || prepare<96, kTypeQ8_0>() ||
                 prepare<128, kTypeF16>() || prepare<128, kTypeQ8_0>() || prepare<256, kTypeF16>() ||
                 prepare<256, kTypeQ8_0>() || wide_prepare()
             ? -5
             : 0;
}

bool attn_head_dim_ok(int hd) { return hd == 64 || hd == 96 || hd == 128 || hd == 256; }

size_t attn_workspace(const KvCache& c, const Attn& a, int sm_count) {
  const int group = a.n_heads / c.n_kv_heads;
  return layout(c, a, choose(c, rows_of(a.max_q_len, group)), choose(c, rows_of(a.max_tokens, group)), sm_count).bytes;
}

cudaError_t attn_launch(const KvCache& c, const Attn& a, int sm_count, cudaStream_t s) {
  const int group = a.n_heads / c.n_kv_heads;
  const Choice ko = choose(c, rows_of(a.max_q_len, group)), kp = choose(c, rows_of(a.max_tokens, group));
  const Layout w = layout(c, a, ko, kp, sm_count);
  uint8_t* ws = static_cast<uint8_t*>(a.ws);
  Pass own = {};
  own.q = a.q;
  own.out = a.out;
  own.ml = a.prefix_len ? reinterpret_cast<float2*>(ws + w.ml[0]) : nullptr;
  own.parts = reinterpret_cast<float*>(ws + w.parts[0]);
  own.line = reinterpret_cast<long long*>(ws + w.line[0]);
  own.q_start = a.q_start;
  own.kv_len = a.kv_len;
  own.pages = a.pages;
  own.pages_stride = a.pages_stride;
  own.n_seqs = a.n_seqs;
  own.n_tokens = a.n_tokens;
  own.n_heads = a.n_heads;
  own.scale = a.scale;
  own.unit_cost = kUnitCost;
  Pass pre = own;
  pre.prefix = a.prefix_len;
  if (a.prefix_len) {
    pre.out = reinterpret_cast<float*>(ws + w.sums);
    pre.ml = reinterpret_cast<float2*>(ws + w.ml[1]);
    pre.parts = reinterpret_cast<float*>(ws + w.parts[1]);
    pre.line = reinterpret_cast<long long*>(ws + w.line[1]);
    pre.pages = a.prefix_pages;
  }
  auto run = [&](const Choice& k, Pass& p) {
    if (!k.fn) {
      p.unit_cost = wide_cost();
      return wide_launch(c, p, sm_count, a.error, s);
    }
    return launch_after(k.per_sm * sm_count, kAttnThreads, k.smem, s, p.beside != 0, k.fn, c, p);
  };
  // The own positions' kernel needs nothing of the prefix's: it fills the SMs as that one's CTAs end.
  own.beside = a.prefix_len && ko.fn;
  if (a.prefix_len)
    if (cudaError_t e = run(kp, pre)) return e;
  if (cudaError_t e = run(ko, own)) return e;
  // the merge's CTAs come up while the tiles' drain; they wait for all of it before they read
  return launch_after(dim3(a.n_tokens, c.n_kv_heads), kMergeThreads, 0, s, true, attn_merge_kernel, c, own, ko.rows, pre,
                      kp.rows, a.out);
}

}  // namespace gi
