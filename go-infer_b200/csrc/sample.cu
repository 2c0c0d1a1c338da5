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
// integer range) until at most 512 candidates are left, and of those every
// thread takes one and sums what comes before it.  A top-k that leaves at
// most 512 is finished on that list alone.
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

#ifndef GI_F
#define GI_F 3ll
#endif
namespace cg = cooperative_groups;

namespace gi {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kSampleWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = kThreads;      // candidates that are ranked directly
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 48 * 1024;  // logits a CTA keeps in shared memory (192 KB)
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
GI_DEVINL u64 place_of(uint32_t key, uint32_t index) { return (u64)~key << 32 | index; }

// rint(2^42 exp((x - top) / T)) by Tang's table method: exp(y) = 2^(n/64) e^r
// with |r| <= ln2 / 128; 2^(j/64) from a table, e^r - 1 by its Taylor sum to
// r^5 (next term below 2^-57); 1/T once per row instead of a division.  The
// result is within 1 of the definition's.
struct Weigh {
  float top;
  double inv_t;
  const double* table;  // 2^(j / 64), shared memory

  GI_DEVINL u64 operator()(float x) const {
    if (top == INFINITY) return x == INFINITY ? kOne : 0ull;
    const double y = ((double)x - (double)top) * inv_t;
    if (!(y > -30.5)) return 0ull;  // below 2^-43.9
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
    return (u64)(__double_as_longlong(w + magic) - __double_as_longlong(magic));
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

struct Item {
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
};

struct Shared {
  Shown shown;
  Item list[kList];
  u64 bin_count[kBins], bin_weight[kBins];  // of the whole row
  u64 part[kSampleWarps + 1], part2[kSampleWarps + 1];
  double table[64];
  u64 found_before;
  u64 answer;
  int found_bin;
  u64 sums[kMaxSums];
};

GI_DEVINL void add64(uint32_t* lo, uint32_t* hi, u64 w) {
  const uint32_t l = (uint32_t)w, old = atomicAdd(lo, l);
  const uint32_t h = (uint32_t)(w >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(hi, h);
}

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
__global__ void __launch_bounds__(kThreads) sample_kernel(Sample p, int slice) {
  extern __shared__ __align__(16) float row_sm[];
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = min(rank * slice, p.vocab), n = min(slice, p.vocab - i0);  // this CTA's logits
  const float* g = p.logits + (size_t)row * p.stride + i0;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;

  // f(what the cluster's CTA r shows, r) for every r, unrolled so that the remote loads are in flight together
  auto each_rank = [&](auto f) {
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
  auto four_at = [&](int i) { return RES ? *reinterpret_cast<const float4*>(row_sm + i) : from_global(i); };
  // f(logit, its index) over the slice, four neighbours per thread and step.
  const int steps = (n + 4 * kThreads - 1) / (4 * kThreads);
  auto each = [&](auto f) {
#pragma unroll 2
    for (int r = 0; r < steps; ++r) {
      const int i = 4 * (r * kThreads + tid);
      if (i >= n) break;
      const float4 v = four_at(i);
      f(v.x, i0 + i), f(v.y, i0 + i + 1), f(v.z, i0 + i + 2), f(v.w, i0 + i + 3);
    }
  };

  // ---- the slice into shared memory; first place, smallest candidate ----
  float best = -INFINITY, low = INFINITY;
  int best_i = -1;
#pragma unroll 8
  for (int r = 0; r < steps; ++r) {
    const int i = 4 * (r * kThreads + tid);
    if (i >= n) break;
    const float4 q = from_global(i);
    if (RES) *reinterpret_cast<float4*>(row_sm + i) = q;
    const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (v[e] > best) {  // the first maximum stays
        best = v[e];
        best_i = i + e;
      }
      if (v[e] > -INFINITY) low = fminf(low, v[e]);
    }
  }
  if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
  for (int i = tid; i < 2 * kBins; i += kThreads) s.shown.count[0][i] = s.shown.lo[0][i] = s.shown.hi[0][i] = 0;
  u64 first = best_i < 0 ? ~0ull : place_of(key_of(best), (uint32_t)(i0 + best_i));
  uint32_t least = best_i < 0 ? ~0u : key_of(low);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  if (lane == 0) {
    s.part[warp] = first;
    s.part2[warp] = least;
  }
  if (tid == 0) s.shown.n_items = 0;
  __syncthreads();
  if (warp == 0) {
    first = s.part[lane & (kSampleWarps - 1)];
    least = (uint32_t)s.part2[lane & (kSampleWarps - 1)];
#pragma unroll
    for (int o = kSampleWarps / 2; o > 0; o >>= 1) {
      first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    if (lane == 0) {
      s.shown.first = first;
      s.shown.least = least;
    }
  }
  cluster.sync();
  first = ~0ull;
  least = ~0u;
  each_rank([&](const Shown* o, int) {
    first = min(first, o->first);
    least = min(least, o->least);
  });
  if (first == ~0ull || !(t > 0.f)) {
    if (rank == 0 && tid == 0) {
      p.ids[row] = first == ~0ull ? -1 : (int32_t)(uint32_t)first;
      if (p.prob) p.prob[row] = first == ~0ull ? 0.f : 1.f;
    }
    cluster.sync();  // nobody reads a CTA that is gone
    return;
  }
  const float top = float_of(~(uint32_t)(first >> 32));
  const Weigh weigh = {top, 1.0 / (double)t, s.table};
  const float reach = 0.5f * top - 0.5f * float_of(least);  // halves: the difference may pass the largest float
  const float per_bin = top == INFINITY ? 0.f : reach > 0.f ? fminf(255.99f / reach, 3.0e38f) : 0.f;
  auto bin_of = [&](float v) {  // linear in the logit; kBins for what is no candidate
    if (!(v > -INFINITY)) return kBins;
    if (top == INFINITY) return v == INFINITY ? 0 : kBins - 1;
    return min((int)((0.5f * top - 0.5f * v) * per_bin), kBins - 1);
  };

  int turn = 0;      // which of the twice-kept buffers
  u64 cut = ~0ull;   // survivors: places <= cut

  // Bins of the row's survivors: by logit, or (BY_PLACE) those in [from, to] by (place - from) >> shift.
  // Leaves the whole row's bins in s.bin_*.
  auto bins = [&](auto by_place, bool weights, u64 from, u64 to, int shift) {
    Shown& o = s.shown;
    each([&](float v, int i) {
      int b = bin_of(v);
      if (b == kBins) return;
      if (decltype(by_place)::value || cut != ~0ull) {
        const u64 place = place_of(key_of(v), (uint32_t)i);
        if (place < from || place > to) return;
        if (decltype(by_place)::value) b = (int)((place - from) >> shift);
      }
      atomicAdd(&o.count[turn][b], 1u);
      if (weights) add64(&o.lo[turn][b], &o.hi[turn][b], weigh(v));
    });
    cluster.sync();
    if (tid < kBins) {
      u64 c = 0, w = 0;
      each_rank([&](const Shown* q, int) {
        c += q->count[turn][tid];
        if (weights) w += (u64)q->hi[turn][tid] << 32 | q->lo[turn][tid];
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
  // every CTA, each with its weight; empty items up to a multiple of 8.
  auto gather = [&](auto take) {
    each([&](float v, int i) {
      if (!take(v, i)) return;
      const u64 place = place_of(key_of(v), (uint32_t)i);
      if (place <= cut) s.shown.items[atomicAdd(&s.shown.n_items, 1)] = place;
    });
    cluster.sync();
    int at = 0, m[kMaxCluster];
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) m[r] = 0;
    each_rank([&](const Shown* q, int r) { m[r] = q->n_items; });
    u64 place = ~0ull;  // thread at + j takes item j of rank r
    each_rank([&](const Shown* q, int r) {
      if (tid >= at && tid < at + m[r]) place = q->items[tid - at];
      at += m[r];
    });
    s.list[tid] = {place, place == ~0ull ? 0ull : weigh(float_of(~(uint32_t)(place >> 32)))};
    cluster.sync();  // the items are read: they may be written again
    if (tid == 0) s.shown.n_items = 0;
    __syncthreads();
    return at;
  };
  // cut = the place at which the running sum over the order reaches `need`; the level-0 bins are there and located.
  auto descend = [&](bool weights, u64 need) {
    int b = s.found_bin, m;
    u64 before = s.found_before;
    if (s.bin_count[b] <= kList) {
      m = gather([&](float v, int) { return bin_of(v) == b; });
    } else {
      // smallest and largest place of the bin's survivors
      u64 lo = ~0ull, hi = 0;
      each([&](float v, int i) {
        if (bin_of(v) != b) return;
        const u64 place = place_of(key_of(v), (uint32_t)i);
        if (place > cut) return;
        lo = min(lo, place);
        hi = max(hi, place);
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      __syncthreads();
      if (lane == 0) {
        s.part[warp] = lo;
        s.part2[warp] = hi;
      }
      __syncthreads();
      if (warp == 0) {
        lo = s.part[lane & (kSampleWarps - 1)];
        hi = s.part2[lane & (kSampleWarps - 1)];
#pragma unroll
        for (int o = kSampleWarps / 2; o > 0; o >>= 1) {
          lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        if (lane == 0) {
          s.shown.range[turn][0] = lo;
          s.shown.range[turn][1] = hi;
        }
      }
      cluster.sync();
      each_rank([&](const Shown* q, int) {
        lo = min(lo, q->range[turn][0]);
        hi = max(hi, q->range[turn][1]);
      });
      u64 left;
      do {  // each turn leaves at most 1/128 of the range
        const int shift = max(0, 56 - __clzll((long long)(hi - lo)));  // (hi - lo) >> shift < 256
        bins(std::true_type(), weights, lo, hi, shift);
        locate(weights, need - before);
        const int d = s.found_bin;
        before += s.found_before;
        lo += (u64)d << shift;
        hi = min(hi, lo + ((1ull << shift) - 1));
        left = s.bin_count[d];
      } while (left > kList);
      m = gather([&](float v, int i) {
        const u64 place = place_of(key_of(v), (uint32_t)i);
        return v > -INFINITY && place >= lo && place <= hi;
      });
    }
    if (tid < m) {
      const Item me = s.list[tid];
      u64 sum = before;
#pragma unroll 8
      for (int j = 0; j < m; ++j) {
        const Item e = s.list[j];
        if (e.place < me.place) sum += weights ? e.weight : 1ull;
      }
      if (sum < need && need <= sum + (weights ? me.weight : 1ull)) s.answer = me.place;
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
    bins(std::false_type(), false, 0ull, ~0ull, 0);
    const u64 all = locate(false, (u64)k);
    if (all > (u64)k) {
      const int b = s.found_bin;
      if (s.found_before + s.bin_count[b] <= kList) {
        // ---- the first k are on one list: finish on it ----
        const int m = gather([&](float v, int) { return bin_of(v) <= b; });
        const Item me = s.list[tid];
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
        s.list[tid].weight = stays ? me.weight : 0ull;
        const u64 total = block_sum(stays ? me.weight : 0ull, s.part);  // its barriers order the list's writes too
        if (stays && rank == 0) {
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
        return;  // gather()'s last barrier: no CTA reads another any more
      }
      descend(false, (u64)k);
    }
  }
  if (top_p < 1.f) {
    bins(std::false_type(), true, 0ull, cut, 0);
    const u64 sum = block_sum(tid < kBins ? s.bin_weight[tid] : 0ull, s.part);
    const u64 need = needed(sum);
    if (need < sum) {
      locate(true, need);
      descend(true, need);
    }
  }

  // ---- the pick: sums of 128 neighbours each (a warp's step), the sums scanned in index order ----
  auto stays_weight = [&](float v, int i) {
    if (!(v > -INFINITY) || place_of(key_of(v), (uint32_t)i) > cut) return 0ull;
    const u64 w = weigh(v);
    return w >= floor_w ? w : 0ull;
  };
  auto four_weights = [&](int i, u64 (&w)[4]) {
    const float4 v = i < n ? four_at(i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    w[0] = stays_weight(v.x, i0 + i), w[1] = stays_weight(v.y, i0 + i + 1);
    w[2] = stays_weight(v.z, i0 + i + 2), w[3] = stays_weight(v.w, i0 + i + 3);
  };
  for (int r = 0; r < steps; ++r) {
    u64 w[4];
    four_weights(4 * (r * kThreads + tid), w);
    const u64 sum = warp_sum64(w[0] + w[1] + w[2] + w[3]);
    if (lane == 0) s.sums[r * kSampleWarps + warp] = sum;
  }
  __syncthreads();
  const int per = (steps * kSampleWarps + kThreads - 1) / kThreads;  // sums per thread: 1, or a few of a long slice
  u64 mine = 0;
  for (int e = 0; e < per; ++e)
    if (tid * per + e < steps * kSampleWarps) mine += s.sums[tid * per + e];
  u64 here;
  u64 before = block_scan(mine, s.part, &here);
  if (tid == 0) s.shown.sum = here;
  cluster.sync();
  u64 total = 0, ahead = 0;
  each_rank([&](const Shown* q, int r) {
    const u64 w = q->sum;
    if (r < rank) ahead += w;
    total += w;
  });
  cluster.sync();
  const u64 target = target_of(total);
  if (target < ahead || target >= ahead + here) return;  // in another CTA's slice
  before += ahead;
  if (target >= before && target < before + mine) {
    int e = tid * per;
    while (target >= before + s.sums[e]) before += s.sums[e++];
    s.found_bin = e;
    s.found_before = before;
  }
  __syncthreads();
  if (warp != 0) return;
  const int i = 128 * s.found_bin + 4 * lane;
  u64 w[4];
  four_weights(i, w);
  const u64 sum = w[0] + w[1] + w[2] + w[3];
  u64 at = s.found_before + warp_scan64(sum, lane) - sum;
  if (target < at || target >= at + sum) return;
  int e = 0;
  while (target >= at + w[e]) at += w[e++];
  p.ids[row] = i0 + i + e;
  if (p.prob) p.prob[row] = (float)((double)w[e] / (double)total);
}

}  // namespace

int sample_prepare_device() {
  return cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kMaxSlice * (int)sizeof(float)) == cudaSuccess
             ? 0
             : -5;
}

cudaError_t sample_launch(const Sample& p, int sm_count, cudaStream_t s) {
  // CTAs per row: while a CTA keeps over 1024 logits and the grid fits the GPU, or the slice does not fit
  // shared memory
  int ranks = 1;
  while (ranks < kMaxCluster && (p.vocab > ranks * kMaxSlice ||
                                 (p.vocab > ranks * 1024 && (long long)p.rows * ranks * 2 <= GI_F * sm_count)))
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
