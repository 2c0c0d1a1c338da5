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
#include "common.cuh"
#include "serve.cuh"

namespace gi {
namespace {

constexpr int kSampleThreads = 1024;
constexpr double kOne = 4398046511104.0;  // 2^42
typedef unsigned long long u64;

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

GI_DEVINL u64 weight_of(uint32_t key, float top, double temperature) {
  if (key == 0u) return 0ull;
  const float x = float_of(key);
  if (top == INFINITY) return x == INFINITY ? (u64)kOne : 0ull;
  return (u64)__double2ll_rn(exp(((double)x - (double)top) / temperature) * kOne);
}

GI_DEVINL u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One block per row, the row read anew for each step.
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(Sample p) {
  constexpr int W = kSampleThreads / 32;
  __shared__ u64 hist[256], part[W], part2[W];
  __shared__ uint32_t s_key;
  __shared__ u64 s_before;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = p.logits + (size_t)row * p.stride;
  const float t = p.temperature ? p.temperature[row] : 1.f;

  auto block_sum = [&](u64 v) {
    v = warp_sum64(v);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = warp_sum64(part[lane]);
    __syncthreads();
    return v;
  };

  // first maximum: the largest (key, lowest index)
  u64 best = 0;
  for (int i = tid; i < p.vocab; i += kSampleThreads) {
    const uint32_t key = key_of(x[i]);
    if (key == 0u) continue;
    const u64 e = (u64)key << 32 | (uint32_t)~i;
    if (e > best) best = e;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 e = __shfl_xor_sync(0xffffffffu, best, o);
    if (e > best) best = e;
  }
  if (lane == 0) part[warp] = best;
  __syncthreads();
  for (int w = 0; w < W; ++w)
    if (part[w] > best) best = part[w];
  __syncthreads();
  if (best == 0ull || !(t > 0.f)) {
    if (tid == 0) {
      p.ids[row] = best ? (int32_t)~(uint32_t)best : -1;
      if (p.prob) p.prob[row] = best ? 1.f : 0.f;
    }
    return;
  }
  const float top = float_of((uint32_t)(best >> 32));
  const double T = (double)t;

  // Survivors: keys above `cut`, and the first `ties` (in index order) of those equal to it.
  uint32_t cut = 0;
  u64 ties = 0;
  // Descends the order until the sum of `what` (1 or the weight) reaches `need` among the present survivors.
  auto descend = [&](bool weights, u64 need, uint32_t old_cut, u64 old_ties) {
    uint32_t prefix = 0, mask = 0;
    u64 before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSampleThreads) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < p.vocab; i += kSampleThreads) {
        const uint32_t key = key_of(x[i]);
        if (key == 0u || (key & mask) != prefix || key <= old_cut) continue;
        atomicAdd(&hist[(key >> shift) & 255], weights ? weight_of(key, top, T) : 1ull);
      }
      if (tid == 0 && old_ties && (old_cut & mask) == prefix)  // the tied survivors
        atomicAdd(&hist[(old_cut >> shift) & 255], weights ? old_ties * weight_of(old_cut, top, T) : old_ties);
      __syncthreads();
      if (tid == 0) {
        u64 sum = before;
        int d = 255;
        for (; d > 0; --d) {
          if (sum + hist[d] >= need) break;
          sum += hist[d];
        }
        s_key = prefix | (uint32_t)d << shift;
        s_before = sum;
      }
      __syncthreads();
      prefix = s_key;
      before = s_before;
      mask |= 255u << shift;
      __syncthreads();
    }
    cut = prefix;
    const u64 each = weights ? weight_of(cut, top, T) : 1ull;
    ties = each ? (need - before + each - 1) / each : 0ull;
  };

  const int k = p.top_k ? p.top_k[row] : 0;
  if (k > 0 && k < p.vocab) {
    u64 n = 0;
    for (int i = tid; i < p.vocab; i += kSampleThreads) n += key_of(x[i]) != 0u;
    if (block_sum(n) > (u64)k) descend(false, (u64)k, 0u, 0ull);
  }
  const float pp = p.top_p ? p.top_p[row] : 1.f;
  if (pp < 1.f) {
    u64 sum = 0;
    for (int i = tid; i < p.vocab; i += kSampleThreads) {
      const uint32_t key = key_of(x[i]);
      if (key > cut) sum += weight_of(key, top, T);
    }
    sum = block_sum(sum) + (ties ? ties * weight_of(cut, top, T) : 0ull);
    const double want = ceil((double)pp * (double)sum);
    const u64 need = want >= 1.0 ? (u64)want : 1ull;
    if (need < sum) descend(true, need, cut, ties);
  }
  const float mp = p.min_p ? p.min_p[row] : 0.f;
  const u64 floor_w = mp > 0.f ? (u64)ceil((double)fminf(mp, 1.f) * kOne) : 0ull;

  // Weights of a warp's run of the row, then the run with the pick, then the pick.
  const int run = (p.vocab + W - 1) / W, r0 = min(warp * run, p.vocab), r1 = min(r0 + run, p.vocab);
  u64 tie_w = ties ? weight_of(cut, top, T) : 0ull;
  if (tie_w < floor_w) tie_w = 0;
  u64 sum = 0, tied = 0;
  for (int i = r0 + lane; i < r1; i += 32) {
    const uint32_t key = key_of(x[i]);
    if (key > cut) {
      const u64 w = weight_of(key, top, T);
      if (w >= floor_w) sum += w;
    } else if (key == cut && key) {
      tied += 1;
    }
  }
  sum = warp_sum64(sum);
  tied = warp_sum64(tied);
  if (lane == 0) {
    part[warp] = sum;
    part2[warp] = tied;
  }
  __syncthreads();
  u64 total = 0, seen_ties = 0, my_before = 0, my_ties = 0, my_sum = 0;
  for (int w = 0; w < W; ++w) {
    const u64 left = ties > seen_ties ? ties - seen_ties : 0ull;
    const u64 s = part[w] + (part2[w] < left ? part2[w] : left) * tie_w;
    if (w == warp) {
      my_before = total;
      my_ties = left;
      my_sum = s;
    }
    total += s;
    seen_ties += part2[w];
  }
  const float u = fminf(fmaxf(p.u[row], 0.f), 1.f - 5.9604644775390625e-8f);
  u64 target = (u64)floor((double)u * (double)total);
  if (target >= total) target = total - 1;
  if (target < my_before || target >= my_before + my_sum) return;
  for (int i0 = r0; i0 < r1; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < r1 ? key_of(x[i]) : 0u;
    const bool tie = key == cut && key;
    const unsigned tb = __ballot_sync(0xffffffffu, tie);
    u64 w = 0;
    if (key > cut) {
      w = weight_of(key, top, T);
      if (w < floor_w) w = 0;
    } else if (tie && (u64)__popc(tb & ((1u << lane) - 1u)) < my_ties) {
      w = tie_w;
    }
    my_ties -= my_ties < (u64)__popc(tb) ? my_ties : (u64)__popc(tb);
    u64 cum = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, cum, o);
      if (lane >= o) cum += y;
    }
    const unsigned over = __ballot_sync(0xffffffffu, my_before + cum > target);
    if (over) {
      if (lane == __ffs(over) - 1) {
        p.ids[row] = i;
        if (p.prob) p.prob[row] = (float)((double)w / (double)total);
      }
      return;
    }
    my_before += __shfl_sync(0xffffffffu, cum, 31);
  }
}

}  // namespace

int sample_prepare_device() { return 0; }

cudaError_t sample_launch(const Sample& p, int, cudaStream_t s) {
  sample_kernel<<<p.rows, kSampleThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace gi
