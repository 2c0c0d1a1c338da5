// wide_attn.cu -- attention over the paged cache for units of many query
// rows (a prompt's chunk, a shared prefix under a batch): the same operator,
// line of tiles and parts as paged_attn.cu, on the 5th-generation tensor
// cores.
//
// Bound: the tensor cores.  A tile is 128 query rows x 128 positions; it
// takes 2 x 128 x 128 x head_dim products for S = q K^T and as many for
// P V, twice each, because q and P are split into two halves (22 bits, see
// paged_attn.cu): about 2200 clocks at head dim 128.  Beside them run the
// softmax (one thread per half row, no shuffles: a row is a tensor-memory
// lane) and the conversion of the cache's values into operand tiles, by warps
// of their own:
//   warps 0-7    softmax: row 32 (w % 4) + lane, positions 64 (w / 4) + 0..63
//                of the tile; also the queries, the running sums, the output
//   warps 8-11   K, 12-14 V^T: the tiles' groups of 16 positions in turn, global
//                -> a ring of raw groups (cp.async) -> halves in the operand
//                tiles, 128-byte swizzle
//   warp 15      tcgen05.mma (one thread), tensor memory
// (16 warps: a thread can have 128 registers)
// K and V^T are K-major operands: V is transposed on its way through
// registers, where Q8_0 codes become halves in any case.  P takes the place
// of S in tensor memory (16 columns of S become 8 of high and 8 of low
// halves) and is the A operand of P V from there.
// Tensor memory, 128 columns each: S/P twice, P V, the queries' high and low
// halves (the A operand of S, so that an S product reads only K from shared
// memory).
// P V of one tile starts from zero; the running sum over tiles is a float32
// FMA in the softmax threads' registers, so rounding does not grow with the
// length (the tensor cores cut their sums).
// Every wait for a barrier in memory is bounded in time; on expiry the CTA sets
// *error, its roles leave, the products in flight are awaited (again bounded),
// tensor memory is freed.  The softmax warps also meet at a named barrier, which
// cannot give up: there they vote, and leave all together or not at all, since
// one warp's wait may expire in the moment in which another's is over.
#include "common.cuh"
#include "gemv.cuh"
#include "paged.cuh"
#include "serve.cuh"
#include "tc.cuh"

namespace gi {
namespace {

using namespace paged;
using namespace tc;

constexpr int kRows = 128, kTok = 128;
constexpr int kSoftWarps = 8, kKWarps = 4, kVWarps = 3, kLoadWarps = kKWarps + kVWarps;
constexpr int kGroups = kTok / 16;  // of 16 positions, what a loading warp takes at a time
constexpr int kWideThreads = 32 * (kSoftWarps + kLoadWarps + 1);
// Tiles that a unit's start and end take.  With 0 / 1 / 2 / 4 / 8: 7 chunks of up to 512 on up to 4000 positions
// 313 / 304 / 292 / 286 / 294 us, 60 of up to 64 on up to 2000 350 / 311 / 267 / 224 / 230 (32/8 heads of 128, Q8_0);
// 200 of up to 32 on up to 500 245 / 236 / 212 / 208 / 221 (heads of 64, F16).
constexpr int kWideCost = 4;
constexpr int kTmem = 512;

template <int HD, int TYPE>
struct Wide {
  static constexpr int kElem = TYPE == kTypeF16 ? 2 : 1;
  static constexpr int kOperand = kTok * HD * 2;       // bytes of a K tile: sub-tiles of 64 dimensions
  static constexpr int kV = HD * kTok * 2;             // bytes of a V^T tile: two sub-tiles of 64 positions
  static constexpr int kData = 16 * HD * kElem;        // bytes of a group of 16 positions in the cache
  static constexpr int kSlot = kData + (TYPE == kTypeF16 ? 0 : HD);  // with its scales
  static constexpr int kSlots = TYPE == kTypeF16 ? 2 : 4;            // groups a loading warp has in flight
  static constexpr int kK = 0, kVt = 2 * kOperand, kRing = kVt + 2 * kV;
  static constexpr int kEnd = kRing + kLoadWarps * kSlots * kSlot;
  static constexpr int kSmem = kEnd + 1024 /* alignment */ + 8192;
  static constexpr int kPart = kRows * (HD + 2);
  static constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kTok >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  static constexpr uint32_t kIdescO = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
};

GI_DEVINL void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// 32 lanes x 32 columns from tensor memory, waited for in place.
GI_DEVINL void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// tc.cuh's products, by the lane of a converged warp for which `mine` is 1:
// the warp computes the operands' descriptors together, in uniform
// registers, and only the instruction itself is predicated.  Issued from
// inside an `if (lane == 0)` each product costs some 130 clocks of moves.
GI_DEVINL void mma_ts_by(uint32_t mine, uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; "
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate), "r"(mine)
      : "memory");
}
GI_DEVINL void commit_by(uint32_t mine, uint32_t bar) {
  asm volatile(
      "{ .reg .pred q; setp.ne.b32 q, %1, 0; "
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar),
      "r"(mine)
      : "memory");
}

// Named barrier of the softmax warps.
GI_DEVINL void soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kSoftWarps) : "memory"); }
// The same with a vote: whether `ok` holds in every thread, the same answer for all.
GI_DEVINL bool soft_vote(bool ok) {
  uint32_t all;
  asm volatile(
      "{ .reg .pred p, q; setp.ne.b32 p, %1, 0; bar.red.and.pred q, 1, %2, p; selp.u32 %0, 1, 0, q; }"
      : "=r"(all)
      : "r"((uint32_t)ok), "n"(32 * kSoftWarps)
      : "memory");
  return all != 0;
}

// A unit of this CTA's run.
struct Unit {
  Seq s;
  int h, row0, n_rows, tile0, tiles, seen_first, b;
  bool whole;
};

// The run's units in order; every role walks them by itself.
struct Walk {
  long long pos, end, first;
  int b;
  __device__ __noinline__ bool next(const KvCache& c, const Pass& p, int group, Unit* u) {
    if (pos >= end) return false;
    Seq s = seq_of(p, b, c.page_shift);
    Span n = span_of(p, s, group, c.n_kv_heads, kRows, kTok);
    while (pos >= first + n.places) {
      first += n.places;
      s = seq_of(p, ++b, c.page_shift);
      n = span_of(p, s, group, c.n_kv_heads, kRows, kTok);
    }
    const long long rel = pos - first;
    const int unit = quotient(rel, n.unit), at0 = (int)(rel - (long long)unit * n.unit);
    const int at1 = (int)min(at0 + (end - pos), (long long)n.unit);
    pos += at1 - at0;
    const int tile0 = max(at0 - p.unit_cost, 0), count = at1 - p.unit_cost - tile0;
    if (count <= 0) return false;  // the run ends before the unit's first tile
    u->s = s;
    u->b = b;
    u->h = unit / n.rt;
    u->row0 = (unit - u->h * n.rt) * kRows;
    u->n_rows = min(kRows, s.fresh * group - u->row0);
    u->tile0 = tile0;
    u->whole = count == n.tl;
    u->seen_first = seen_by(p, s, u->row0 / group);
    const int seen_last = seen_by(p, s, (u->row0 + u->n_rows - 1) / group);
    u->tiles = max(0, min(tile0 + count, (seen_last + kTok - 1) / kTok) - tile0);
    return true;
  }
};

// The rest of a wait that was not over at once: bounded in time; false ends the role.
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* stop, int* error) {
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
    for (int i = 0; i < 16; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*stop) return false;
    if (globaltimer_ns() - t0 > kWaitNs) {
      *stop = 1;
      atomicExch(error, 1);
      return false;
    }
  }
}

// The roles' loops share the SM's instruction cache: unrolled to the full, they ran at a
// quarter of the speed.
template <int HD, int TYPE>
__global__ void __launch_bounds__(kWideThreads, 1) wide_kernel(KvCache c, Pass p, int* error) {
  using W = Wide<HD, TYPE>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  float2* s_ml = reinterpret_cast<float2*>(sm + W::kEnd);          // [2][row]: a half row's statistics
  float* s_max = reinterpret_cast<float*>(s_ml + 2 * kRows);       // [tile parity][half][row]
  uint8_t* s_bad = reinterpret_cast<uint8_t*>(s_max + 4 * kRows);  // [tile % 4][16-position group]
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_bad + 32);
  volatile int* s_stop = reinterpret_cast<volatile int*>(s_tmem + 1);
  const uint32_t bars = smem_u32(s_tmem + 4);  // 8-byte aligned: everything above is a multiple of 16 bytes
  Unit* s_unit = reinterpret_cast<Unit*>(s_tmem + 4 + 2 * 18);  // the softmax warps' unit
  // barriers, [tile parity] each but the queries'
  auto k_full = [&](int i) { return bars + 8 * i; };
  auto pv_full = [&](int i) { return bars + 8 * (2 + i); };  // V^T is there and P, which comes after P V of the tile before is taken
  auto k_free = [&](int i) { return bars + 8 * (4 + i); };
  auto v_free = [&](int i) { return bars + 8 * (6 + i); };
  auto s_full = [&](int i) { return bars + 8 * (8 + i); };
  auto o_full = [&](int i) { return bars + 8 * (10 + i); };
  const uint32_t q_full = bars + 8 * 12, last = bars + 8 * 13;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = p.n_heads / c.n_kv_heads;

  griddep_wait();
  griddep_launch_dependents();
  Run run;
  if (!run_of_line<kWideThreads>(c, p, group, kRows, kTok, 1, &run)) return;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full(i), kGroups);
      mbar_init(pv_full(i), kGroups + kSoftWarps);
      mbar_init(k_free(i), 1);
      mbar_init(v_free(i), 1);
      mbar_init(s_full(i), 1);
      mbar_init(o_full(i), 1);
    }
    mbar_init(q_full, kSoftWarps);
    mbar_init(last, 1);
    fence_mbar_init();
    *s_stop = 0;
  }
  if (warp == kSoftWarps + kLoadWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)),
                 "r"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(s_tmem);
  auto s_col = [&](int i) { return tmem + i * kTok; };
  const uint32_t o_col = tmem + 2 * kTok, q_col = o_col + 128;  // P V; the queries' high, then low halves

  // By every lane of a warp, which leaves together; false ends the role.
  auto wait = [&](uint32_t bar, uint32_t parity) {
    const bool ok = mbar_try_wait(bar, parity) || wait_on(bar, parity, s_stop, error);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  Walk walk = {run.pos, run.end, run.first, run.b};
  Unit u;
  int tile_no = 0;  // tiles of all units so far: buffer tile_no & 1, use tile_no >> 1 of it
  auto phase = [](int i) { return (uint32_t)(i >> 1) & 1u; };

  if (warp >= kSoftWarps + kLoadWarps) {
    // ---- the products ----
    int unit_no = 0;
    bool ok = true;
    const uint32_t mine = lane == 0, tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
    while (ok && walk.next(c, p, group, &u)) {
      if (!u.tiles) continue;  // no queries come: their writer may be at most one phase ahead
      if (!(ok = wait(q_full, unit_no & 1))) break;
      ++unit_no;
      // S of tile i goes before P V of tile i - 1, which waits for the softmax
      for (int i = 0; i <= u.tiles && ok && u.tiles; ++i) {
        if (i < u.tiles) {
          const int n = tile_no + i;
          if (i >= 2) ok = wait(o_full(n & 1), phase(n - 2));  // P of tile n - 2 is read: S may come in its place
          ok = ok && wait(k_full(n & 1), phase(n));
          if (!ok) break;
          tc_fence_after();
          const int buf = __shfl_sync(0xffffffffu, n & 1, 0);
          const uint32_t d = tmem_u + buf * kTok;
          const uint32_t q = tmem_u + 2 * kTok + 128;
          const uint64_t k = desc_sw128(base + W::kK + buf * W::kOperand);
#pragma unroll
          for (int part = 0; part < 2; ++part)  // the low halves first: each step cuts the sum, and theirs is small
#pragma unroll
            for (int e = 0; e < HD / 16; ++e) {
              const int off = (e >> 2) * (kTok * 128 / 16) + (e & 3) * 2;
              mma_ts_by(mine, d, q + (1 - part) * (HD / 2) + 8 * e, k + off, W::kIdescS, part | e);
            }
          commit_by(mine, s_full(buf));
          commit_by(mine, k_free(buf));
        }
        if (i > 0) {
          const int n = tile_no + i - 1;
          ok = wait(pv_full(n & 1), phase(n));
          if (!ok) break;
          tc_fence_after();
          const int buf = __shfl_sync(0xffffffffu, n & 1, 0);
          const uint32_t d = tmem_u + 2 * kTok, a = tmem_u + buf * kTok;
          const uint64_t v = desc_sw128(base + W::kVt + buf * W::kV);
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int e = 0; e < kTok / 16; ++e)
              mma_ts_by(mine, d, a + 16 * e + 8 * (1 - part), v + (e >> 2) * (HD * 128 / 16) + (e & 3) * 2, W::kIdescO,
                        part | e);
          commit_by(mine, o_full(buf));
          commit_by(mine, v_free(buf));
        }
      }
      tile_no += u.tiles;
    }
    // nothing may be in flight when the others leave
    if (lane == 0) {
      mma_commit(last);
      if (!wait_phase(last, 0)) atomicExch(error, 1);
    }
    __syncwarp();
  } else if (warp >= kSoftWarps) {
    // ---- operand tiles: a warp takes every 4th group of K, or every 3rd of V ----
    constexpr int kE = W::kElem;
    constexpr int kLoads = W::kData / 512;       // 16-byte copies of a group per lane
    constexpr int kDims = HD / 32;               // dimensions of V per lane
    constexpr int kVWords = kDims * kE >= 4 ? kDims * kE / 4 : 1;
    constexpr int kScaleWords = HD / 64;  // words of a position's scales
    const bool is_k = warp < kSoftWarps + kKWarps;
    const int step = is_k ? kKWarps : kVWarps, id = is_k ? warp - kSoftWarps : warp - kSoftWarps - kKWarps;
    const uint32_t slots = base + W::kRing + (warp - kSoftWarps) * W::kSlots * W::kSlot;
    // The warp's groups of a unit in turn: group g of the unit's 8 * tiles is
    // its if (8 tile_no + g) % step == id.  kSlots of them are on their way
    // into the warp's slots; 32 pages are looked up at a time, one per lane, so
    // that a group's copies do not wait for its page.
    int page = 0, page_of = 0;  // of group page_of + lane * step
    uint32_t bads = 0;          // bit s: slot s's group has no such page
    auto look_up = [&](int g) {
      page_of = g;
      const int p0 = u.tile0 * kTok + 16 * (g + lane * step);
      const int32_t* pages = p.pages + (p.prefix ? 0 : (size_t)u.b * p.pages_stride);
      page = p0 < u.s.len && p0 >= 0 ? __ldg(pages + (p0 >> c.page_shift)) : 0;
    };
    auto copy = [&](int g, int slot) {
      if (g >= page_of + 32 * step) look_up(g);
      const int p0 = u.tile0 * kTok + 16 * g, pg = __shfl_sync(0xffffffffu, page, (g - page_of) / step);
      const bool bad = (unsigned)pg >= (unsigned)c.n_pages;
      bads = (bads & ~(1u << slot)) | (uint32_t)bad << slot;
      const int left = bad ? 0 : u.s.len - p0;
      const size_t at = (((size_t)(bad ? 0 : pg) * c.n_kv_heads + u.h) << c.page_shift) + (p0 & (c.page_size - 1));
      const uint8_t* src = (is_k ? c.k : c.v) + at * HD * kE;
      const uint32_t dst = slots + slot * W::kSlot;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int ch = 32 * i + lane;
        cp_async16_or_zero(dst + 16 * ch, src + 16 * ch, ch / (HD * kE / 16) < left ? 16 : 0);
      }
      if (TYPE == kTypeQ8_0 && lane < HD / 16)  // 16 bytes: the scales of 256 / HD positions
        cp_async16_or_zero(dst + W::kData + 16 * lane,
                           reinterpret_cast<const uint8_t*>(is_k ? c.ks : c.vs) + at * (HD / 16) + 16 * lane,
                           16 * lane < left * (HD / 16) ? 16 : 0);
    };
    // word `lane` of a slot's scales; 0 for positions that do not exist, whatever lies there
    auto scales_of = [&](int g, int slot) {
      uint32_t w = 0;
      if (TYPE == kTypeQ8_0 && lane < 16 * kScaleWords &&
          u.tile0 * kTok + 16 * g + lane / kScaleWords < ((bads >> slot) & 1 ? 0 : u.s.len))
        w = lds32(slots + slot * W::kSlot + W::kData + 4 * lane);
      return w;
    };
    // scale of position r, block b, from the lanes' words
    auto scale_word = [&](uint32_t words, int r, int b) {
      return __shfl_sync(0xffffffffu, words, r * kScaleWords + (b >> 1));
    };
    auto put_k = [&](uint32_t from, uint32_t scales, int tile, int w) {
      const uint32_t dst = base + W::kK + (tile & 1) * W::kOperand;
#pragma unroll
      for (int l = 0; l < kLoads; ++l) {
        const int ch = 32 * l + lane, per = HD * kE / 16, r = ch / per, row = 16 * w + r, q = ch - r * per;
        const uint4 x = lds128(from + 16 * ch);
        if (TYPE == kTypeF16) {  // 8 values: one 16-byte unit
          sts128(dst + (q >> 3) * (kTok * 128) + sw128_off(row, q & 7), x.x, x.y, x.z, x.w);
        } else {  // 16 codes: two units, all of one block
          const int b = q >> 1;
          const uint32_t d2 = prmt(scale_word(scales, r, b), 0u, b & 1 ? 0x3232 : 0x1010);
          uint32_t o[8];
          codes_to_h2(x.x, o[0], o[1]);
          codes_to_h2(x.y, o[2], o[3]);
          codes_to_h2(x.z, o[4], o[5]);
          codes_to_h2(x.w, o[6], o[7]);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = hmul2_u32(o[e], d2);
          const uint32_t t = dst + (q >> 2) * (kTok * 128);
          const int unit = 2 * (q & 3);
          sts128(t + sw128_off(row, unit), o[0], o[1], o[2], o[3]);
          sts128(t + sw128_off(row, unit + 1), o[4], o[5], o[6], o[7]);
        }
      }
    };
    auto put_v = [&](uint32_t from, uint32_t scales, int tile, int w) {
      // 64 positions per sub-tile
      const uint32_t dst = base + W::kVt + (tile & 1) * W::kV + (w >> 2) * (HD * 128);
      const int b = lane * kDims / 32;  // this lane's block of 32 dimensions
      // a lane's rows come in an order of its own, so that eight lanes that store together hold
      // eight rows that differ mod 8 and with them, by the swizzle, eight 16-byte units of the banks
      const uint32_t turn = TYPE != kTypeF16 && kDims == 4 ? (lane >> 1) & 3 : (lane >> 2) & 1;
      const uint32_t first = TYPE == kTypeF16 ? 0x5410 ^ (turn * 0x2222) : (0x5140 ^ (turn * 0x1111));
      const uint32_t second = first ^ 0x2222;
      auto row_of = [&](int e) {
        return TYPE == kTypeF16 ? 64 * (e >> 1) + 2 * lane + ((e & 1) ^ turn) : lane * kDims + (e ^ turn);
      };
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 8 positions: one 16-byte unit of each of the lane's rows
        uint32_t x[8][kVWords], o[kDims][4];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t a = from + (8 * half + r) * HD * kE + lane * (TYPE == kTypeF16 ? 4 : kDims);
#pragma unroll
          for (int i = 0; i < kVWords; ++i) x[r][i] = TYPE != kTypeF16 && kDims == 2 ? lds16(a) : lds32(a + 128 * i);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (TYPE == kTypeF16) {
#pragma unroll
            for (int e = 0; e < kDims / 2; ++e) {
              o[2 * e][q] = prmt(x[2 * q][e], x[2 * q + 1][e], first);
              o[2 * e + 1][q] = prmt(x[2 * q][e], x[2 * q + 1][e], second);
            }
          } else {
            const int r = 8 * half + 2 * q;
            const uint32_t d = prmt(scale_word(scales, r, b), scale_word(scales, r + 1, b), b & 1 ? 0x7632 : 0x5410);
            uint32_t x0, x1;
            codes_to_h2(prmt(x[2 * q][0], x[2 * q + 1][0], first), x0, x1);
            o[0][q] = hmul2_u32(x0, d);
            o[1][q] = hmul2_u32(x1, d);
            if (kDims == 4) {
              codes_to_h2(prmt(x[2 * q][0], x[2 * q + 1][0], second), x0, x1);
              o[2 % kDims][q] = hmul2_u32(x0, d);
              o[3 % kDims][q] = hmul2_u32(x1, d);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < kDims; ++e)
          sts128(dst + sw128_off(row_of(e), 2 * (w & 3) + half), o[e][0], o[e][1], o[e][2], o[e][3]);
      }
    };
    bool go = true;
    while (go && walk.next(c, p, group, &u)) {
      const int n_groups = u.tiles * kGroups;
      const int g0 = ((id - tile_no * kGroups) % step + step) % step;  // this warp's first
      if (g0 < n_groups) look_up(g0);
#pragma unroll 1
      for (int s = 0; s < W::kSlots; ++s) {
        if (g0 + s * step < n_groups) copy(g0 + s * step, s);
        cp_async_commit();
      }
      int slot = 0;
#pragma unroll 1
      for (int g = g0; g < n_groups; g += step) {
        const int n = tile_no + g / kGroups, w = g % kGroups;
        cp_async_wait<W::kSlots - 1>();
        __syncwarp();
        if (!(go = wait(is_k ? k_free(n & 1) : v_free(n & 1), phase(n) ^ 1))) break;
        const uint32_t from = slots + slot * W::kSlot, scales = scales_of(g, slot);
        if (is_k) {
          if (lane == 0) s_bad[8 * (n & 3) + w] = (bads >> slot) & 1;  // read until the softmax of this tile is done
          put_k(from, scales, n, w);
        } else {
          put_v(from, scales, n, w);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(is_k ? k_full(n & 1) : pv_full(n & 1));
        if (g + W::kSlots * step < n_groups) copy(g + W::kSlots * step, slot);
        cp_async_commit();
        slot = slot + 1 == W::kSlots ? 0 : slot + 1;
      }
      cp_async_wait<0>();
      tile_no += u.tiles;
    }
  } else {
    // ---- softmax ----
    const int half = warp >> 2, r = 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    constexpr int kOut = HD / 2;  // this thread's dimensions of the output
    bool ok = true;
    // thread 0 walks and shows the unit: the others keep no state of the walk in registers
    while (ok) {
      if (tid == 0) {
        s_unit->tiles = -1;
        if (walk.next(c, p, group, &u)) *s_unit = u;
      }
      soft_sync();
      const int tiles = s_unit->tiles;
      if (tiles < 0) break;
      // queries: a power of two per row that puts the largest just under 2^14, then
      // high and low halves into tensor memory, the A operand of S
      float fac = 0.f;
      if (tiles) {
        const int row = s_unit->row0 + r;
        const bool real = r < s_unit->n_rows;
        const float4* q = reinterpret_cast<const float4*>(
            p.q + ((size_t)(s_unit->s.start + (real ? row / group : 0)) * p.n_heads + (size_t)s_unit->h * group +
                   (real ? row % group : 0)) * HD + half * kOut);
        float x[kOut], m = 0.f;
#pragma unroll
        for (int i = 0; i < kOut / 4; ++i) {
          const float4 y = real ? __ldg(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
          x[4 * i] = y.x, x[4 * i + 1] = y.y, x[4 * i + 2] = y.z, x[4 * i + 3] = y.w;
        }
#pragma unroll
        for (int i = 0; i < kOut; ++i) m = fmaxf(m, fabsf(x[i]));
        s_max[half * kRows + r] = m;
        soft_sync();
        m = fmaxf(m, s_max[(half ^ 1) * kRows + r]);
        const int ex = (int)(__float_as_uint(m) >> 23) - 127;
        const int sh = m > 0.f ? min(13 - ex, 126) : 0;
        const float up = p.scale < 0.f ? -exp2i(sh) : exp2i(sh);  // the scale's sign with q: the factor on S is >= 0
        fac = fabsf(p.scale) * kLog2e * exp2i(-sh);
#pragma unroll
        for (int i = 0; i < kOut; i += 32) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x0 = x[i + 2 * e] * up, x1 = x[i + 2 * e + 1] * up;
            hi[e] = pack_h2(x0, x1);
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
            lo[e] = pack_h2(x0 - back.x, x1 - back.y);
          }
          const uint32_t to = q_col + lanes + (half * kOut + i) / 2;
          tmem_st16(to, hi);
          tmem_st16(to + HD / 2, lo);
        }
        tmem_wait_st();
        tc_fence_before();
        soft_sync();  // s_max is read
        if (lane == 0) mbar_arrive(q_full);
      }
      const int seen = seen_by(p, s_unit->s, (s_unit->row0 + min(r, s_unit->n_rows - 1)) / group) - s_unit->tile0 * kTok;
      const int seen_first = s_unit->seen_first - s_unit->tile0 * kTok;  // positions from the first tile's on
      float o[kOut], m = -INFINITY, l = 0.f, alpha = 0.f;  // m: of the products, before the factor
#pragma unroll
      for (int i = 0; i < kOut; ++i) o[i] = 0.f;
      // A wait that gave up is taken to the next vote: no warp leaves on its own, and
      // until then it touches neither tensor memory nor the barriers.
      for (int i = 0; i <= tiles && tiles; ++i) {
        const int n_i = tile_no + i, p0 = i * kTok + 64 * half;
        const uint32_t s = s_col(n_i & 1) + lanes + 64 * half;
        uint32_t bad = 0;
        bool masked = false;
        float alpha_n = 0.f, zero = 0.f;
        // positions j .. j + 15 of the 64 that this row sees
        auto limit = [&](int j) { return (bad >> (8 * (j >> 4))) & 1 ? 0 : seen - p0 - j; };
        if (i < tiles) {
          const int n = n_i;
          ok = ok && wait(s_full(n & 1), phase(n));
          tc_fence_after();
          bad = *reinterpret_cast<const volatile uint32_t*>(s_bad + 8 * (n & 3) + 4 * half);
          masked = p0 + 64 > seen_first || bad;  // uniform in the warp
          float top = -INFINITY;
#pragma unroll 1
          for (int j = ok ? 0 : 64; j < 64; j += 32) {
            float x[32];
            tmem_ld32(s + j, x);
            if (masked) {
              const int l0 = limit(j), l1 = limit(j + 16);
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                x[e] = e < l0 ? x[e] : -INFINITY;
                x[16 + e] = e < l1 ? x[16 + e] : -INFINITY;
              }
            }
            float t2 = x[1];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              top = fmaxf(top, x[e]);
              t2 = fmaxf(t2, x[e + 1]);
            }
            top = fmaxf(top, t2);
          }
          s_max[((n & 1) * 2 + half) * kRows + r] = top;
          if (!(ok = soft_vote(ok))) break;
          top = fmaxf(top, s_max[((n & 1) * 2 + (half ^ 1)) * kRows + r]);
          top = fmaxf(m, top);
          zero = top == -INFINITY ? 0.f : top;
          alpha_n = m == -INFINITY ? 0.f : exp2_approx((m - zero) * fac);
          m = top;
        }
        if (i > 0) {  // o = o alpha + P V of the tile before, before this tile's P lets the next one begin
          const int n = tile_no + i - 1;
          ok = ok && wait(o_full(n & 1), phase(n));
          if (!ok) continue;
          tc_fence_after();
#pragma unroll
          for (int d = 0; d < kOut; d += 32) {
            float x[32];
            tmem_ld32(o_col + lanes + half * kOut + d, x);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[d + e] = fmaf(o[d + e], alpha, x[e]);
          }
          tc_fence_before();
        }
        if (i < tiles) {
          float sum = 0.f, sum2 = 0.f;
          // The maximum is taken off before the factor, so the largest weight is 1 exactly, however large the
          // scores are: x fac - zero fac in one FMA leaves the rounding of zero fac, which is past half's range
          // from scores of 2^25 on.  P at most 2^14, by a product, which rounds nothing; inside the exponent the
          // power would be rounded to 2^-21 of a weight.
#pragma unroll 1
          for (int j = 0; j < 64; j += 16) {
            float x[16];
            uint32_t w[16];
            tmem_ld16(s + j, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = exp2_approx((x[e] - zero) * fac) * 16384.f;
            if (masked) {
              const int l0 = limit(j);
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = e < l0 ? x[e] : 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sum += x[2 * e];
              sum2 += x[2 * e + 1];
              w[e] = pack_h2(x[2 * e], x[2 * e + 1]);
              const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
              w[8 + e] = pack_h2(x[2 * e] - back.x, x[2 * e + 1] - back.y);
            }
            tmem_st16(s + j, w);
          }
          sum += sum2;
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pv_full(n_i & 1));
          l = l * alpha_n + sum;
        }
        alpha = alpha_n;
      }
      tile_no += tiles;

      // ---- the row: finished, its sums, or a part ----
      s_ml[half * kRows + r] = make_float2(m, l);
      if (!(ok = soft_vote(ok))) break;
      float sum = l + s_ml[(half ^ 1) * kRows + r].y;
      const int row = s_unit->row0 + r;
      const bool real = r < s_unit->n_rows;
      const size_t at =
          (size_t)(s_unit->s.start + row / group) * p.n_heads + (size_t)s_unit->h * group + row % group;
      // What is joined with other parts is for the maximum in powers of two, m fac rounded: 2^(what was rounded off)
      // goes to the sums, unless it is more than they bear (then scores are whole steps of 32 and more apart).
      const float m2 = m == -INFINITY ? m : m * fac, rest = fmaf(m, fac, -m2);
      float f = fabsf(rest) <= 16.f ? exp2f(rest) : 1.f;
      sum *= f;
      float* out = p.out + at * HD + half * kOut;
      if (!s_unit->whole) {
        float* part = p.parts + (size_t)(2 * blockIdx.x + (s_unit->tile0 > 0 ? 0 : 1)) * W::kPart;
        out = part + r * HD + half * kOut;
        if (half == 0 && real) *reinterpret_cast<float2*>(part + kRows * HD + 2 * r) = make_float2(m2, sum);
      } else if (p.ml) {
        if (half == 0 && real) p.ml[at] = make_float2(m2, sum);
      } else {
        f = sum > 0.f ? f / sum : 0.f;
      }
      if (real) {
#pragma unroll
        for (int i = 0; i < kOut; i += 4)
          *reinterpret_cast<float4*>(out + i) = make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
      }
      soft_sync();  // s_unit, s_ml and s_max are read
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kSoftWarps + kLoadWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmem) : "memory");
}

template <int HD, int TYPE>
cudaError_t launch_wide(const KvCache& c, const Pass& p, int sm_count, int* error, cudaStream_t s) {
  wide_kernel<HD, TYPE><<<sm_count, kWideThreads, Wide<HD, TYPE>::kSmem, s>>>(c, p, error);
  return cudaGetLastError();
}

template <int HD, int TYPE>
bool prepare_wide() {
  return cudaFuncSetAttribute(wide_kernel<HD, TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Wide<HD, TYPE>::kSmem) ==
         cudaSuccess;
}

}  // namespace

namespace paged {

// Head dim 128 from 48 rows on: 4 sequences of 8000 positions, 8 kv heads, Q8_0, take 54 / 55 / 56 / 97 us here
// with 48 / 64 / 96 / 256 rows per unit, and 63 / 58 / 65 / 211 us in units of at most 32 rows (paged_attn.cu); a
// prefix of 8192 under 48 / 64 sequences 35 / 39 and 41 / 45 us.  Sequences of 500 positions lose up to 2 us by it
// (48 rows: 20.7 against 18.2).  Head dim 64, half the work per tile, from 64 rows on: 47 against 51 us with 64
// rows, but 44 against 39 with 48.
bool wide_ok(int head_dim, int rows) { return (head_dim == 128 && rows >= 48) || (head_dim == 64 && rows >= 64); }

Rows wide_rows(int head_dim) { return {kRows, kTok, kRows * (head_dim + 2)}; }

int wide_prepare() {
  return prepare_wide<64, kTypeF16>() && prepare_wide<64, kTypeQ8_0>() && prepare_wide<128, kTypeF16>() &&
                 prepare_wide<128, kTypeQ8_0>()
             ? 0
             : -5;
}

cudaError_t wide_launch(const KvCache& c, const Pass& p, int sm_count, int* error, cudaStream_t s) {
  const bool f16 = c.type == kTypeF16;
  if (c.head_dim == 64)
    return f16 ? launch_wide<64, kTypeF16>(c, p, sm_count, error, s)
               : launch_wide<64, kTypeQ8_0>(c, p, sm_count, error, s);
  return f16 ? launch_wide<128, kTypeF16>(c, p, sm_count, error, s)
             : launch_wide<128, kTypeQ8_0>(c, p, sm_count, error, s);
}

int wide_cost() { return kWideCost; }

}  // namespace paged
}  // namespace gi
