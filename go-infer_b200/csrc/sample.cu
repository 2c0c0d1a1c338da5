// sample.cu -- the next token of each row of logits: temperature, top-k,
// top-p and min-p, and the pick by a given uniform number (the work of
// pkg/sampler for a batch; greedy rows take the first maximum as
// sampler.go:86-96 does).
//
// Definition, for a row with candidates (logits above -inf; NaN is none):
//   weight  W_i = rint(2^42 exp((l_i - max) / T)), exp in double, so W is a
//           64-bit integer and every sum of weights is exact: no order of
//           additions can move a border;
//   order   by logit, larger first, equal ones by index, lower first;
//   top-k   the first k of the order;
//   top-p   of these the shortest beginning with sum >= ceil(p * sum of all);
//   min-p   of these those with W >= ceil(min_p * 2^42);
//   pick    in index order the first whose running sum exceeds
//           floor(u * sum).
//
// No sort: a border of the order is found by counting.  The candidates (or
// their weights) are summed into 256 bins that are linear in the logit, the
// bin that holds the border is searched further (256 bins of the order's own
// integer range) until at most 128 candidates are left, and of those every
// thread takes one and sums what comes before it.  A top-k that leaves at
// most 128 is finished on that list alone.  Once a border's bin is known and
// at most 2048 candidates lie before its end, they are packed in index order
// into one CTA, which goes on alone.
//
// Bound: one row is latency (a few cluster barriers), many rows are the read of
// the logits and the double-precision exponentials of rows without top-k.  A
// row is spread over a cluster of CTAs, each of which keeps its slice of the row
// in shared memory; bins, lists and sums are exchanged through distributed
// shared memory.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"
#include "serve.cuh"

namespace cg = cooperative_groups;

namespace gi {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kSampleWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = 128;            // candidates that are ranked directly, each against all
constexpr int kMaxCluster = 8;
constexpr int kLoads = 4;             // 16-byte loads a thread has in flight
constexpr int kPack = 64;             // survivors a warp can pack
constexpr int kFlat = 2048;           // survivors of a row that one CTA takes over
constexpr int kMaxSlice = 44 * 1024;  // logits a CTA keeps in shared memory (176 KB)
constexpr int kMaxSums = (1 << 20) / kMaxCluster / 128;  // sums of 128 neighbours of the longest slice
constexpr int kFracBits = 42;         // a weight of 1 is 2^42
constexpr u64 kOne = 1ull << kFracBits;

// Monotone key of a float: larger float, larger key; -0 as +0; 0 for what is
// no candidate (-inf and NaN).
GI_DEVINL uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
GI_DEVINL float float_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// Place in the order: smaller comes first.
GI_DEVINL u64 place_of(float x, int index) { return (u64)~key_of(x) << 32 | (uint32_t)index; }
GI_DEVINL float logit_at(u64 place) { return float_of(~(uint32_t)(place >> 32)); }

// rint(2^42 exp((x - top) / T)) by Tang's table method: exp(y) = 2^(n/64) e^r
// with |r| <= ln2 / 128; 2^(j/64) from a table, e^r - 1 by its Taylor sum to
// r^5 (next term below 2^-57); 1/T once per row instead of a division.  The
// result is within 1 of the definition's.  No branches, so that a thread's
// four logits overlap; 0 for what is no candidate.
struct Weigh {
  float top;
  double inv_t;
  const double* table;  // 2^(j / 64), shared memory

  GI_DEVINL u64 operator()(float x) const {
    const double y = fmax(((double)x - (double)top) * inv_t, -31.0);  // 2^42 e^-31 < 1/2; not a number counts as -31
    const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double z = fma(y, 92.33248261689366, magic);  // 64 / ln 2
    const int n = __double2loint(z);
    const double nd = z - magic;
    const double r = fma(nd, -1.162596423439437e-12, fma(nd, -0.010830424695086549, y));  // ln 2 / 64: 33 bits and the rest
    double q = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    q = fma(r, q, 1.0 / 6.0);
    q = fma(r, q, 0.5);
    q = fma(r, q, 1.0);
    const double s = table[n & 63];
    const double v = fma(s, q * r, s);  // in [0.99, 2.01)
    const double w = __hiloint2double(__double2hiint(v) + (((n >> 6) + kFracBits) << 20), __double2loint(v));
    const u64 rounded = (u64)(__double_as_longlong(w + magic) - __double_as_longlong(magic));
    return top == INFINITY ? (x == INFINITY ? kOne : 0ull) : rounded;
  }
};

GI_DEVINL u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
GI_DEVINL u64 warp_scan64(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}
// Smallest a and largest b over the lanes of groups of `width`.
template <typename A>
GI_DEVINL void warp_least_most(A& a, A& b, int width) {
  for (int o = width / 2; o > 0; o >>= 1) {
    a = min(a, __shfl_xor_sync(0xffffffffu, a, o));
    b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
  }
}

struct alignas(16) Item {
  u64 place, weight;
};

// What a CTA shows the others of its cluster.  Everything that is written
// again in a later step exists twice, used in turn: the barrier of the
// step between tells that all have read it.
struct Shown {
  uint32_t count[2][kBins], lo[2][kBins], hi[2][kBins];  // candidates and weights of the bins
  u64 first, sum;      // smallest place; weight that stays
  uint32_t least;      // smallest key of a candidate
  u64 range[2][2];     // smallest and largest place of a bin
  int n_items;
  u64 items[kList];    // places
  // what each warp has packed of its stretch of the slice, and the number (kPack + 1: too many)
  int pack_n[kSampleWarps];
  float pack_v[kSampleWarps][kPack];
  int pack_i[kSampleWarps][kPack];
};

struct Shared {
  Shown shown;
  Item list[kList];
  u64 bin_count[kBins], bin_weight[kBins];  // of the whole row
  u64 part[kSampleWarps], part2[kSampleWarps];
  double table[64];
  u64 found_before;
  u64 answer;
  int found_bin;
  union {  // the row's survivors in index order, or the pick's sums of a slice
    struct {
      alignas(16) float flat_v[kFlat];
      alignas(16) int flat_i[kFlat];
    };
    u64 sums[kMaxSums];
  };
};

static_assert(offsetof(Shared, flat_v) % 16 == 0 && offsetof(Shared, flat_i) % 16 == 0, "read as float4 and int4");

// Sum over the block, for every thread.
GI_DEVINL u64 block_sum(u64 v, u64* part) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) v += part[w];
  return v;
}

// Sum over the threads before this one, and over all.
GI_DEVINL u64 block_scan(u64 v, u64* part, u64* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 incl = warp_scan64(v, lane);
  __syncthreads();
  if (lane == 31) part[warp] = incl;
  __syncthreads();
  u64 before = incl - v, all = 0;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) {
    if (w < warp) before += part[w];
    all += part[w];
  }
  *total = all;
  return before;
}

// RES: the slice is in shared memory, else it is read from global memory each time.
template <bool RES>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(Sample p, int slice) {
  extern __shared__ __align__(16) float row_sm[];
  __shared__ __align__(16) Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), row = blockIdx.x / (int)cluster.num_blocks();
  int ranks = (int)cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = min(rank * slice, p.vocab), n = min(slice, p.vocab - i0);  // this CTA's logits
  const float* g = p.logits + (size_t)row * p.stride + i0;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;
  Weigh weigh = {0.f, 0.0, s.table};

  int flat = -1;  // >= 0: this CTA alone goes on, with so many survivors in s.flat_*
  auto barrier = [&] {
    if (flat >= 0) __syncthreads();
    else cluster.sync();
  };
  // f(what the cluster's CTA r shows, r) for every r, unrolled so that the remote loads are in flight together
  auto each_rank = [&](auto f) {
    if (flat >= 0) {
      f(static_cast<const Shown*>(&s.shown), 0);
      return;
    }
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r)
      if (r < ranks) f(static_cast<const Shown*>(cluster.map_shared_rank(&s.shown, r)), r);
  };
  // Four logits from index i (a multiple of 4) of the slice on; -inf behind its end.
  const bool aligned = (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  auto from_global = [&](int i) {
    if (aligned && i + 4 <= n) return __ldg(reinterpret_cast<const float4*>(g + i));
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = i + e < n ? __ldg(g + i + e) : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
  };
  // Four neighbours of the slice, or of the flat survivors; -inf behind their end.
  auto four = [&](int j, float (&v)[4], int (&i)[4]) {
    float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (flat >= 0) {
      int4 x = make_int4(0, 0, 0, 0);
      if (j < flat) {
        q = *reinterpret_cast<const float4*>(s.flat_v + j);
        x = *reinterpret_cast<const int4*>(s.flat_i + j);
      }
      i[0] = x.x, i[1] = x.y, i[2] = x.z, i[3] = x.w;
    } else {
      if (j < n) q = RES ? *reinterpret_cast<const float4*>(row_sm + j) : from_global(j);
#pragma unroll
      for (int e = 0; e < 4; ++e) i[e] = i0 + j + e;
    }
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  };
  // f(four logits, their indexes) over the slice or the flat survivors
  auto each = [&](auto f) {
    const int end = flat >= 0 ? flat : n;
#pragma unroll 2
    for (int j = 4 * tid; j < end; j += 4 * kThreads) {
      float v[4];
      int i[4];
      four(j, v, i);
      f(v, i);
    }
  };

  // ---- the slice into shared memory; first place, smallest candidate ----
  float best = -INFINITY, low = INFINITY;
  int best_i = -1;
  for (int j = 4 * tid; j < n; j += 4 * kLoads * kThreads) {
    float4 q[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int i = j + 4 * u * kThreads;
      q[u] = i < n ? from_global(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int i = j + 4 * u * kThreads;
      if (RES && i < n) *reinterpret_cast<float4*>(row_sm + i) = q[u];
      const float v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (v[e] > best) {  // the first maximum stays
          best = v[e];
          best_i = i + e;
        }
        if (v[e] > -INFINITY) low = fminf(low, v[e]);
      }
    }
  }
  if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
  for (int i = tid; i < 2 * kBins; i += kThreads) s.shown.count[0][i] = s.shown.lo[0][i] = s.shown.hi[0][i] = 0;
  // (place, ~key): both smallest
  u64 first = best_i < 0 ? ~0ull : place_of(best, i0 + best_i), least = best_i < 0 ? 0ull : ~key_of(low);
  warp_least_most(first, least, 32);
  if (lane == 0) {
    s.part[warp] = first;
    s.part2[warp] = least;
  }
  if (tid == 0) s.shown.n_items = 0;
  __syncthreads();
  if (warp == 0) {
    first = s.part[lane & (kSampleWarps - 1)];
    least = s.part2[lane & (kSampleWarps - 1)];
    warp_least_most(first, least, kSampleWarps);
    if (lane == 0) {
      s.shown.first = first;
      s.shown.least = (uint32_t)least;
    }
  }
  cluster.sync();
  first = ~0ull;
  least = 0ull;
  each_rank([&](const Shown* o, int) {
    first = min(first, o->first);
    least = max(least, (u64)o->least);
  });
  if (first == ~0ull || !(t > 0.f)) {
    if (rank == 0 && tid == 0) {
      p.ids[row] = first == ~0ull ? -1 : (int32_t)(uint32_t)first;
      if (p.prob) p.prob[row] = first == ~0ull ? 0.f : 1.f;
    }
    cluster.sync();  // nobody reads a CTA that is gone
    return;
  }
  const float top = logit_at(first);
  weigh.top = top;
  weigh.inv_t = 1.0 / (double)t;
  // Bins linear in the logit; halves, because the difference may pass the
  // largest float.  With an infinite top only infinite logits weigh: they are bin 0.
  const float reach = 0.5f * top - 0.5f * float_of(~(uint32_t)least);
  const float per_bin = top == INFINITY ? 1e-36f : reach > 0.f ? fminf(255.99f / reach, 3.0e38f) : 0.f;
  const float half_top = top == INFINITY ? 2.5e38f : 0.5f * top;
  auto scaled = [&](float v) { return fmaxf(fmaf(-0.5f, v, half_top) * per_bin, 0.f); };
  auto bin_of = [&](float v) { return min((int)scaled(v), kBins - 1); };  // of a candidate
  // a candidate of bins up to b
  auto up_to = [&](float v, int b) { return v > -INFINITY && (b >= kBins - 1 || scaled(v) < (float)(b + 1)); };

  int turn = 0;      // which of the twice-kept buffers
  u64 cut = ~0ull;   // survivors: places <= cut

  // Bins of the row's survivors: by logit, or (BY_PLACE) those in [from, cut] by (place - from) >> shift.
  // Leaves the whole row's bins in s.bin_*.
  auto bins = [&](auto by_place, auto weights, u64 from, u64 to, int shift) {
    constexpr bool kPlace = decltype(by_place)::value, kWeights = decltype(weights)::value;
    constexpr bool kCounts = kPlace || !kWeights;
    Shown& o = s.shown;
    each([&](const float (&v)[4], const int (&i)[4]) {
      int b[4];
      u64 w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        b[e] = v[e] > -INFINITY ? bin_of(v[e]) : -1;
        if (kPlace || cut != ~0ull) {
          const u64 place = place_of(v[e], i[e]);
          if (place < from || place > to) b[e] = -1;
          else if (kPlace) b[e] = (int)((place - from) >> shift);
        }
        if (kWeights) w[e] = weigh(v[e]);
      }
      if (kCounts) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (b[e] >= 0) atomicAdd(&o.count[turn][b[e]], 1u);
      }
      if (kWeights) {  // a 64-bit sum in two words: the low word's carry goes up
        uint32_t up[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t l = b[e] >= 0 ? (uint32_t)w[e] : 0u;
          const uint32_t old = l ? atomicAdd(&o.lo[turn][b[e]], l) : 0u;
          up[e] = (b[e] >= 0 ? (uint32_t)(w[e] >> 32) : 0u) + (old + l < old ? 1u : 0u);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (up[e]) atomicAdd(&o.hi[turn][b[e]], up[e]);
      }
    });
    barrier();
    if (tid < kBins) {
      u64 c = 0, w = 0;
      each_rank([&](const Shown* q, int) {
        if (kCounts) c += q->count[turn][tid];
        if (kWeights) w += (u64)q->hi[turn][tid] << 32 | q->lo[turn][tid];
      });
      s.bin_count[tid] = c;
      s.bin_weight[tid] = w;
    }
    turn ^= 1;
    // the buffers of the next step: their readers have passed this step's barrier
    if (tid < kBins) o.count[turn][tid] = o.lo[turn][tid] = o.hi[turn][tid] = 0;
    __syncthreads();
  };
  // The bin in which the running sum (of counts or weights) reaches `need`, and the sum before it.
  auto locate = [&](bool weights, u64 need) {
    const u64 mine = tid < kBins ? (weights ? s.bin_weight[tid] : s.bin_count[tid]) : 0ull;
    u64 all;
    const u64 before = block_scan(mine, s.part, &all);
    if (tid < kBins && before < need && need <= before + mine) {
      s.found_bin = tid;
      s.found_before = before;
    }
    __syncthreads();
    return all;
  };
  // The row's survivors that `take` accepts, at most kList, into s.list of
  // every CTA, each with its weight.
  auto gather = [&](auto take) {
    each([&](const float (&v)[4], const int (&i)[4]) {
      bool in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = take(v[e], i[e]);
      if (!(in[0] | in[1] | in[2] | in[3])) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u64 place = place_of(v[e], i[e]);
        if (in[e] && place <= cut) s.shown.items[atomicAdd(&s.shown.n_items, 1)] = place;
      }
    });
    barrier();
    int at = 0, m[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) m[r] = 0;
    each_rank([&](const Shown* q, int r) { m[r] = q->n_items; });
    u64 place = ~0ull;  // thread at + j takes item j of rank r
    each_rank([&](const Shown* q, int r) {
      if (tid >= at && tid < at + m[r]) place = q->items[tid - at];
      at += m[r];
    });
    if (tid < kList) s.list[tid] = {place, place == ~0ull ? 0ull : weigh(logit_at(place))};
    barrier();  // the items are read: they may be written again
    if (tid == 0) s.shown.n_items = 0;
    __syncthreads();
    return at;
  };
  // Packs the row's candidates of bins up to b into rank 0,
  // which goes on alone: false for the other CTAs, which are done.  Nothing
  // happens when a warp or the row has too many.
  auto pack = [&](int b) {
    if (flat >= 0) return true;
    const int stretch = ((n + kSampleWarps - 1) / kSampleWarps + 127) & ~127;
    const int w0 = min(warp * stretch, n), w1 = min(w0 + stretch, n);
    int have = 0;
#pragma unroll 2
    for (int j0 = w0; j0 < w1; j0 += 128) {
      float v[4];
      int i[4];
      four(j0 + 4 * lane, v, i);  // -inf from the slice's end; a stretch ends on a multiple of 128 or there
      unsigned in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = __ballot_sync(0xffffffffu, up_to(v[e], b));
      if (!(in[0] | in[1] | in[2] | in[3])) continue;
      const unsigned lower = (1u << lane) - 1u;
      int at = have + __popc(in[0] & lower) + __popc(in[1] & lower) + __popc(in[2] & lower) + __popc(in[3] & lower);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((in[e] >> lane) & 1) {
          if (at < kPack) {
            s.shown.pack_v[warp][at] = v[e];
            s.shown.pack_i[warp][at] = i[e];
          }
          ++at;
        }
      have += __popc(in[0]) + __popc(in[1]) + __popc(in[2]) + __popc(in[3]);
      if (have > kPack) break;
    }
    if (lane == 0) s.shown.pack_n[warp] = min(have, kPack + 1);
    cluster.sync();
    // every CTA sees every warp's number: thread r * 16 + w that of warp w of rank r
    int m = 0;
    if (tid < ranks * kSampleWarps)
      m = cluster.map_shared_rank(&s.shown, tid / kSampleWarps)->pack_n[tid % kSampleWarps];
    if (__syncthreads_or(m > kPack)) return true;
    if (block_sum((u64)m, s.part) > kFlat) return true;
    if (rank == 0) {
      u64 all;
      const int before = (int)block_scan((u64)m, s.part, &all);
      if (tid < kMaxCluster * kSampleWarps) s.list[tid].place = (u64)before << 32 | (uint32_t)m;  // (no list is in use)
      __syncthreads();
      // warp w takes what the ranks' warps w have, all remote loads in flight together
      float v[kMaxCluster][kPack / 32];
      int i[kMaxCluster][kPack / 32];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        if (r >= ranks) break;
        const Shown* o = cluster.map_shared_rank(&s.shown, r);
        const int have_r = (int)(uint32_t)s.list[r * kSampleWarps + warp].place;
#pragma unroll
        for (int h = 0; h < kPack / 32; ++h)
          if (32 * h + lane < have_r) {
            v[r][h] = o->pack_v[warp][32 * h + lane];
            i[r][h] = o->pack_i[warp][32 * h + lane];
          }
      }
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        if (r >= ranks) break;
        const u64 e = s.list[r * kSampleWarps + warp].place;
#pragma unroll
        for (int h = 0; h < kPack / 32; ++h)
          if (32 * h + lane < (int)(uint32_t)e) {
            s.flat_v[(int)(e >> 32) + 32 * h + lane] = v[r][h];
            s.flat_i[(int)(e >> 32) + 32 * h + lane] = i[r][h];
          }
      }
      const int total = (int)all;
      if (tid < 3 && total + tid < kFlat) s.flat_v[total + tid] = -INFINITY;  // up to a multiple of 4
      flat = total;
    }
    cluster.sync();  // what was packed is read
    return rank == 0;
  };
  // cut = the place at which the running sum over the order reaches `need`,
  // found in bin b of the level-0 bins with `before` in front of it; in_bin: the bin's candidates (all ones: not counted).
  auto descend = [&](auto weights, u64 need, int b, u64 before, u64 in_bin) {
    constexpr bool kWeights = decltype(weights)::value;
    int m;
    if (in_bin <= kList) {
      m = gather([&](float v, int) { return v > -INFINITY && bin_of(v) == b; });
    } else {
      // smallest and largest place of the bin's survivors
      u64 lo = ~0ull, hi = 0;
      each([&](const float (&v)[4], const int (&i)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 place = place_of(v[e], i[e]);
          if (!(v[e] > -INFINITY) || bin_of(v[e]) != b || place > cut) continue;
          lo = min(lo, place);
          hi = max(hi, place);
        }
      });
      warp_least_most(lo, hi, 32);
      __syncthreads();
      if (lane == 0) {
        s.part[warp] = lo;
        s.part2[warp] = hi;
      }
      __syncthreads();
      if (warp == 0) {
        lo = s.part[lane & (kSampleWarps - 1)];
        hi = s.part2[lane & (kSampleWarps - 1)];
        warp_least_most(lo, hi, kSampleWarps);
        if (lane == 0) {
          s.shown.range[turn][0] = lo;
          s.shown.range[turn][1] = hi;
        }
      }
      barrier();
      each_rank([&](const Shown* q, int) {
        lo = min(lo, q->range[turn][0]);
        hi = max(hi, q->range[turn][1]);
      });
      u64 left;
      do {  // each turn leaves at most 1/128 of the range
        const int shift = max(0, 56 - __clzll((long long)(hi - lo)));  // (hi - lo) >> shift < 256
        bins(std::true_type(), weights, lo, hi, shift);
        locate(kWeights, need - before);
        const int d = s.found_bin;
        before += s.found_before;
        lo += (u64)d << shift;
        hi = min(hi, lo + ((1ull << shift) - 1));
        left = s.bin_count[d];
      } while (left > kList);
      m = gather([&](float v, int i) {
        const u64 place = place_of(v, i);
        return v > -INFINITY && place >= lo && place <= hi;
      });
    }
    if (tid < m) {
      const Item me = s.list[tid];
      u64 sum = before;
#pragma unroll 8
      for (int j = 0; j < m; ++j) {
        const Item e = s.list[j];
        if (e.place < me.place) sum += kWeights ? e.weight : 1ull;
      }
      if (sum < need && need <= sum + (kWeights ? me.weight : 1ull)) s.answer = me.place;
    }
    __syncthreads();
    cut = s.answer;
    __syncthreads();
  };
  auto needed = [&](u64 sum) {  // top-p's border
    const double want = ceil((double)top_p * (double)sum);
    return want >= 1.0 ? (u64)want : 1ull;
  };
  const u64 floor_w = min_p > 0.f ? (u64)ceil((double)fminf(min_p, 1.f) * (double)kOne) : 0ull;
  const double u = (double)fminf(fmaxf(p.u[row], 0.f), 1.f - 5.9604644775390625e-8f);
  auto target_of = [&](u64 sum) {
    const u64 w = (u64)floor(u * (double)sum);
    return w < sum ? w : sum - 1;
  };

  if (k > 0 && k < p.vocab) {
    bins(std::false_type(), std::false_type(), 0ull, ~0ull, 0);
    const u64 all = locate(false, (u64)k);
    if (all > (u64)k) {
      const int b = s.found_bin;
      const u64 ahead_of_b = s.found_before, in_b = s.bin_count[b];
      if (ahead_of_b + in_b <= kList) {
        // ---- the first k are on one list: rank 0 finishes on it ----
        const int m = gather([&](float v, int) { return up_to(v, b); });
        if (rank != 0) return;  // gather()'s last barrier: no CTA reads another any more
        const Item me = s.list[min(tid, kList - 1)];
        u64 before = 0;
        int ahead = 0;
        if (tid < m) {
#pragma unroll 8
          for (int j = 0; j < m; ++j) {
            const Item e = s.list[j];
            if (e.place < me.place) {
              before += e.weight;
              ++ahead;
            }
          }
        }
        bool stays = tid < m && ahead < k;
        if (top_p < 1.f) {
          const u64 sum = block_sum(stays ? me.weight : 0ull, s.part);
          stays = stays && before < needed(sum);
        }
        stays = stays && me.weight >= floor_w;
        __syncthreads();
        if (tid < kList) s.list[tid].weight = stays ? me.weight : 0ull;
        const u64 total = block_sum(stays ? me.weight : 0ull, s.part);  // its barriers order the list's writes too
        if (stays) {
          const u64 target = target_of(total);
          u64 run = 0;
#pragma unroll 8
          for (int j = 0; j < m; ++j) {
            const Item e = s.list[j];
            if ((uint32_t)e.place < (uint32_t)me.place) run += e.weight;
          }
          if (run <= target && target < run + me.weight) {
            p.ids[row] = (int32_t)(uint32_t)me.place;
            if (p.prob) p.prob[row] = (float)((double)me.weight / (double)total);
          }
        }
        return;
      }
      if (ahead_of_b + in_b <= kFlat && !pack(b)) return;
      descend(std::false_type(), (u64)k, b, ahead_of_b, in_b);
    }
  }
  if (top_p < 1.f) {
    bins(std::false_type(), std::true_type(), 0ull, cut, 0);
    const u64 sum = block_sum(tid < kBins ? s.bin_weight[tid] : 0ull, s.part);
    const u64 need = needed(sum);
    if (need < sum) {
      locate(true, need);
      const int b = s.found_bin;
      const u64 ahead_of_b = s.found_before;
      if (cut == ~0ull && !pack(b)) return;
      descend(std::true_type(), need, b, ahead_of_b, ~0ull);
    }
  }

  // ---- the pick: sums of 128 neighbours each, scanned in index order ----
  auto four_weights = [&](int group, u64 (&w)[4], int (&i)[4]) {
    float v[4];
    four(128 * group + 4 * lane, v, i);
    bool in = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (cut != ~0ull && place_of(v[e], i[e]) > cut) v[e] = -INFINITY;
      in |= v[e] > -INFINITY;
    }
    w[0] = w[1] = w[2] = w[3] = 0ull;
    if (!__any_sync(0xffffffffu, in)) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = weigh(v[e]);
      if (w[e] < floor_w) w[e] = 0ull;
    }
  };
  const int groups = ((flat >= 0 ? flat : n) + 127) / 128;
  u64* sums = flat >= 0 ? reinterpret_cast<u64*>(s.list) : s.sums;  // (no list is in use any more)
  __syncthreads();
#pragma unroll 2
  for (int e = warp; e < groups; e += kSampleWarps) {
    u64 w[4];
    int i[4];
    four_weights(e, w, i);
    const u64 sum = warp_sum64(w[0] + w[1] + w[2] + w[3]);
    if (lane == 0) sums[e] = sum;
  }
  __syncthreads();
  const int per = (groups + kThreads - 1) / kThreads;  // sums per thread: 1, or a few of a long slice
  u64 mine = 0;
  for (int e = tid * per; e < min(tid * per + per, groups); ++e) mine += sums[e];
  u64 here;
  u64 before = block_scan(mine, s.part, &here);
  u64 total = here, ahead = 0;
  if (flat < 0) {
    if (tid == 0) s.shown.sum = here;
    cluster.sync();
    total = 0;
    each_rank([&](const Shown* q, int r) {
      const u64 w = q->sum;
      if (r < rank) ahead += w;
      total += w;
    });
    cluster.sync();
  }
  const u64 target = target_of(total);
  if (target < ahead || target >= ahead + here) return;  // in another CTA's slice
  before += ahead;
  if (target >= before && target < before + mine) {
    int e = tid * per;
    while (target >= before + sums[e]) before += sums[e++];
    s.found_bin = e;
    s.found_before = before;
  }
  __syncthreads();
  if (warp != 0) return;
  u64 w[4];
  int i[4];
  four_weights(s.found_bin, w, i);
  const u64 sum = w[0] + w[1] + w[2] + w[3];
  u64 at = s.found_before + warp_scan64(sum, lane) - sum;
  if (target < at || target >= at + sum) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (target >= at && target < at + w[e]) {
      p.ids[row] = i[e];
      if (p.prob) p.prob[row] = (float)((double)w[e] / (double)total);
    }
    at += w[e];
  }
}

}  // namespace

int sample_prepare_device() {
  return cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kMaxSlice * (int)sizeof(float)) == cudaSuccess
             ? 0
             : -5;
}

cudaError_t sample_launch(const Sample& p, int sm_count, cudaStream_t s) {
  // CTAs per row: doubled while each keeps over 512 logits and at most 4 come
  // on an SM (64 rows of 128256: 66 us with 8, 85 us with 4), and while the
  // slice does not fit shared memory.
  int ranks = 1;
  while (ranks < kMaxCluster && (p.vocab > ranks * kMaxSlice ||
                                 (p.vocab > ranks * 1024 && p.rows * ranks <= 2 * sm_count)))
    ranks *= 2;
  const int slice = ((p.vocab + ranks - 1) / ranks + 3) & ~3;
  const bool resident = slice <= kMaxSlice;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ranks * (unsigned)p.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = resident ? sizeof(float) * slice : 0;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return resident ? cudaLaunchKernelEx(&cfg, sample_kernel<true>, p, slice)
                  : cudaLaunchKernelEx(&cfg, sample_kernel<false>, p, slice);
}

}  // namespace gi
