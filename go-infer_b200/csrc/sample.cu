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

#include "common.cuh"
#include "serve.cuh"

namespace cg = cooperative_groups;

namespace gi {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kSampleWarps = kThreads / 32;
constexpr int kBins = 256;
constexpr int kList = kThreads;      // candidates that are ranked directly
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 48 * 1024;  // logits a CTA keeps in shared memory (192 KB)
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
  u64 first, sum[2];   // smallest place; sums
  uint32_t least;      // smallest key of a candidate
  u64 range[2][2];     // smallest and largest place of a bin
  int n_items;
  Item items[kList];
};

struct Shared {
  Shown shown;
  Item list[kList];
  u64 bin_count[kBins], bin_weight[kBins];  // of the whole row
  u64 part[kSampleWarps + 1], part2[kSampleWarps + 1];
  double table[64];
  u64 found_before;
  u64 answer;
  int found_bin, n_list;
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

__global__ void __launch_bounds__(kThreads) sample_kernel(Sample p, int slice, int resident) {
  extern __shared__ __align__(16) float row_sm[];
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i0 = min(rank * slice, p.vocab), n = min(slice, p.vocab - i0);  // this CTA's logits
  const float* g = p.logits + (size_t)row * p.stride + i0;
  const float* x = resident ? row_sm : g;
  const float t = p.temperature ? p.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float min_p = p.min_p ? p.min_p[row] : 0.f;

  // ---- the slice into shared memory; first place, smallest key ----
  u64 first = ~0ull;
  uint32_t least = ~0u;
  auto look = [&](float v, int i) {
    const uint32_t key = key_of(v);
    if (key == 0u) return;
    first = min(first, place_of(key, (uint32_t)(i0 + i)));
    least = min(least, key);
  };
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(g) & 15) == 0) {
    for (int i = tid; i < n / 4; i += kThreads) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(g) + i);
      if (resident) reinterpret_cast<float4*>(row_sm)[i] = v;
      look(v.x, 4 * i), look(v.y, 4 * i + 1), look(v.z, 4 * i + 2), look(v.w, 4 * i + 3);
    }
    done = n & ~3;
  }
  for (int i = done + tid; i < n; i += kThreads) {
    const float v = __ldg(g + i);
    if (resident) row_sm[i] = v;
    look(v, i);
  }
  if (tid < 64) s.table[tid] = exp2((double)tid / 64.0);
  for (int i = tid; i < 2 * kBins; i += kThreads) s.shown.count[0][i] = s.shown.lo[0][i] = s.shown.hi[0][i] = 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  if (lane == 0) {
    s.part[warp] = first;
    s.part2[warp] = least;
  }
  if (tid == 0) s.shown.n_items = s.n_list = 0;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kSampleWarps; ++w) {
      first = min(first, s.part[w]);
      least = min(least, (uint32_t)s.part2[w]);
    }
    s.shown.first = first;
    s.shown.least = least;
  }
  cluster.sync();
  first = ~0ull;
  least = ~0u;
  for (int r = 0; r < ranks; ++r) {
    const Shown* o = cluster.map_shared_rank(&s.shown, r);
    first = min(first, o->first);
    least = min(least, o->least);
  }
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
  auto bin_of = [&](float v) {  // linear in the logit
    if (top == INFINITY) return v == INFINITY ? 0 : kBins - 1;
    return min((int)((0.5f * top - 0.5f * v) * per_bin), kBins - 1);
  };

  int turn = 0;      // which of the twice-kept buffers
  u64 cut = ~0ull;   // survivors: places <= cut

  // Bins of the row's survivors in [from, to]: by logit (shift < 0), or by
  // (place - from) >> shift.  Leaves the whole row's bins in s.bin_*.
  auto bins = [&](bool weights, u64 from, u64 to, int shift) {
    Shown& o = s.shown;
    for (int i = tid; i < n; i += kThreads) {
      const float v = x[i];
      const uint32_t key = key_of(v);
      if (key == 0u) continue;
      const u64 place = place_of(key, (uint32_t)(i0 + i));
      if (place < from || place > to) continue;
      const int b = shift < 0 ? bin_of(v) : (int)((place - from) >> shift);
      atomicAdd(&o.count[turn][b], 1u);
      if (weights) add64(&o.lo[turn][b], &o.hi[turn][b], weigh(v));
    }
    cluster.sync();
    if (tid < kBins) {
      u64 c = 0, w = 0;
      for (int r = 0; r < ranks; ++r) {
        const Shown* q = cluster.map_shared_rank(&s.shown, r);
        c += q->count[turn][tid];
        if (weights) w += (u64)q->hi[turn][tid] << 32 | q->lo[turn][tid];
      }
      s.bin_count[tid] = c;
      s.bin_weight[tid] = w;
    }
    turn ^= 1;
    // the buffers of the next step: their readers have passed this step's barrier
    for (int i = tid; i < kBins; i += kThreads) o.count[turn][i] = o.lo[turn][i] = o.hi[turn][i] = 0;
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
  };
  // The row's survivors that `take` accepts, at most kList, into s.list of every CTA.
  auto gather = [&](auto take) {
    for (int i = tid; i < n; i += kThreads) {
      const float v = x[i];
      const uint32_t key = key_of(v);
      if (key == 0u) continue;
      const u64 place = place_of(key, (uint32_t)(i0 + i));
      if (place > cut || !take(v, place)) continue;
      s.shown.items[atomicAdd(&s.shown.n_items, 1)] = {place, weigh(v)};
    }
    cluster.sync();
    int at = 0;
    for (int r = 0; r < ranks; ++r) {
      const Shown* q = cluster.map_shared_rank(&s.shown, r);
      const int m = q->n_items;
      if (tid < m) s.list[at + tid] = q->items[tid];
      at += m;
    }
    if (tid == 0) s.n_list = at;
    cluster.sync();  // the items are read: they may be written again
    if (tid == 0) s.shown.n_items = 0;
    __syncthreads();
  };
  // cut = the place at which the running sum over the order reaches `need`; the level-0 bins are there.
  auto descend = [&](bool weights, u64 need) {
    locate(weights, need);
    int b = s.found_bin;
    u64 before = s.found_before;
    if (s.bin_count[b] <= kList) {
      gather([&](float v, u64) { return bin_of(v) == b; });
    } else {
      // smallest and largest place of the bin's survivors
      u64 lo = ~0ull, hi = 0;
      for (int i = tid; i < n; i += kThreads) {
        const float v = x[i];
        const uint32_t key = key_of(v);
        if (key == 0u || bin_of(v) != b) continue;
        const u64 place = place_of(key, (uint32_t)(i0 + i));
        if (place > cut) continue;
        lo = min(lo, place);
        hi = max(hi, place);
      }
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
      if (tid == 0) {
        for (int w = 0; w < kSampleWarps; ++w) {
          lo = min(lo, s.part[w]);
          hi = max(hi, s.part2[w]);
        }
        s.shown.range[turn][0] = lo;
        s.shown.range[turn][1] = hi;
      }
      cluster.sync();
      for (int r = 0; r < ranks; ++r) {
        const Shown* q = cluster.map_shared_rank(&s.shown, r);
        lo = min(lo, q->range[turn][0]);
        hi = max(hi, q->range[turn][1]);
      }
      for (;;) {  // each turn leaves at most 1/128 of the range
        const int shift = max(0, 56 - __clzll((long long)(hi - lo)));  // (hi - lo) >> shift < 256
        bins(weights, lo, hi, shift);
        locate(weights, need - before);
        const int d = s.found_bin;
        before += s.found_before;
        lo += (u64)d << shift;
        hi = min(hi, lo + ((1ull << shift) - 1));
        const u64 left = s.bin_count[d];
        if (left <= kList) break;
      }
      gather([&](float, u64 place) { return place >= lo && place <= hi; });
    }
    if (tid < s.n_list) {
      const Item me = s.list[tid];
      u64 sum = before;
      for (int j = 0; j < s.n_list; ++j)
        if (s.list[j].place < me.place) sum += weights ? s.list[j].weight : 1ull;
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
    bins(false, 0ull, ~0ull, -1);
    const u64 all = block_sum(tid < kBins ? s.bin_count[tid] : 0ull, s.part);
    if (all > (u64)k) {
      locate(false, (u64)k);
      const int b = s.found_bin;
      if (s.found_before + s.bin_count[b] <= kList) {
        // ---- the first k are on one list: finish on it ----
        gather([&](float v, u64) { return bin_of(v) <= b; });
        const int m = s.n_list;
        Item me = {~0ull, 0ull};
        u64 before = 0;
        int ahead = 0;
        if (tid < m) {
          me = s.list[tid];
          for (int j = 0; j < m; ++j)
            if (s.list[j].place < me.place) {
              before += s.list[j].weight;
              ++ahead;
            }
        }
        bool stays = tid < m && ahead < k;
        const u64 sum = block_sum(stays ? me.weight : 0ull, s.part);
        if (top_p < 1.f) stays = stays && before < needed(sum);
        stays = stays && me.weight >= floor_w;
        __syncthreads();
        if (tid < m) s.list[tid].weight = stays ? me.weight : 0ull;
        const u64 total = block_sum(stays ? me.weight : 0ull, s.part);  // its barriers order the list's writes too
        if (stays && rank == 0) {
          const u64 target = target_of(total);
          u64 run = 0;
          for (int j = 0; j < m; ++j)
            if ((uint32_t)s.list[j].place < (uint32_t)me.place) run += s.list[j].weight;
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
    bins(true, 0ull, cut, -1);
    const u64 sum = block_sum(tid < kBins ? s.bin_weight[tid] : 0ull, s.part);
    const u64 need = needed(sum);
    if (need < sum) descend(true, need);
  }

  // ---- the pick: a thread sums a run of the slice (an odd length: no two lanes in one bank) ----
  const int run = ((n + kThreads - 1) / kThreads) | 1, a0 = min(tid * run, n), a1 = min(a0 + run, n);
  auto stays_weight = [&](int i) {
    const float v = x[i];
    const uint32_t key = key_of(v);
    if (key == 0u || place_of(key, (uint32_t)(i0 + i)) > cut) return 0ull;
    const u64 w = weigh(v);
    return w >= floor_w ? w : 0ull;
  };
  u64 mine = 0;
  for (int i = a0; i < a1; ++i) mine += stays_weight(i);
  u64 here;
  u64 before = block_scan(mine, s.part, &here);
  if (tid == 0) s.shown.sum[0] = here;
  cluster.sync();
  u64 total = 0, ahead = 0;
  for (int r = 0; r < ranks; ++r) {
    const u64 w = cluster.map_shared_rank(&s.shown, r)->sum[0];
    if (r < rank) ahead += w;
    total += w;
  }
  cluster.sync();
  const u64 target = target_of(total);
  before += ahead;
  if (target < before || target >= before + mine) return;
  for (int i = a0; i < a1; ++i) {
    const u64 w = stays_weight(i);
    if (target < before + w) {
      p.ids[row] = i0 + i;
      if (p.prob) p.prob[row] = (float)((double)w / (double)total);
      return;
    }
    before += w;
  }
}

}  // namespace

int sample_prepare_device() {
  return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              kMaxSlice * (int)sizeof(float)) == cudaSuccess
             ? 0
             : -5;
}

cudaError_t sample_launch(const Sample& p, int sm_count, cudaStream_t s) {
  // CTAs per row: while a CTA keeps over 1024 logits and the grid fits the GPU, or the slice does not fit
  // shared memory
  int ranks = 1;
  while (ranks < kMaxCluster && (p.vocab > ranks * kMaxSlice ||
                                 (p.vocab > ranks * 1024 && (long long)p.rows * ranks * 2 <= 3ll * sm_count)))
    ranks *= 2;
  const int slice = ((p.vocab + ranks - 1) / ranks + 3) & ~3;
  const int resident = slice <= kMaxSlice;
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
  return cudaLaunchKernelEx(&cfg, sample_kernel, p, slice, resident);
}

}  // namespace gi
