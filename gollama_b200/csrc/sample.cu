// Drawing the next token: temperature, top-k, top-p, min-p, and the inverse of
// the kept tokens' running sum at a given random number.
//
// A token's weight is exp((l - max) / temperature) to 27 bits, in whole numbers of
// 2^-45 (sample_plan.h), so sums of weights are exact and every order of
// summation gives the same one.  The exponent is reduced in 64 bits and the weight is
// right to 2^-27 of itself and 2^-45 of the largest, so the sum of V tokens to V 2^-45
// and 2^-27 of itself where all errors are of one sign, as in a tail of equal logits,
// and to a small part of that in an ordinary row.  Sums of float32 exponentials are
// off by about 2^-25 of themselves: with tens of thousands of tokens kept that moves
// past a token's edge about once in a thousand rows, and that token is then another.
//
// Tokens are ordered by (logit falling, index rising), a total order; the kept
// ones of top-k and of top-p are each a prefix of it, so each filter is a cut:
// its last kept token.  Nothing is sorted but the few tokens around a cut: a
// histogram finds the bin the cut falls in (of top-k: bins of max - l; of top-p:
// 256 bins per factor of two of the weight), that bin's tokens (or, for a small
// k, all down to it) are gathered and ranked against each other.  A bin of more
// than 512 tokens is first narrowed by the bits of the order itself, 10 at a
// time, which ends for any input, equal logits too.  The draw itself is a sum
// over the kept tokens in index order, taken apart in CTAs, warps and lanes.
//
// A cluster of CTAs holds a row in shared memory, first its logits and then, in
// their place, the weights, so each is read and computed once; the histograms,
// the gathered tokens and the partial sums meet through distributed shared
// memory.  Only what is near a cut reads a logit again.  256 rows of 131075 at
// top_p 0.95 take 237 us, a tenth of a plain copy's rate: a CTA's phases were 3.3 us
// for the logits, 5.1 for weights and histogram, 3.9 for the draw, and the rest of 27
// exchanges between the CTAs of a row and what they wait for (with weights of 2^-31,
// 231 us in all).  128 rows of 32000 with mixed settings take 28 us, one row 9.9.
#include <cfloat>
#include <climits>
#include <cooperative_groups.h>

#include "kv_cache.cuh"
#include "sample_plan.h"

namespace cg = cooperative_groups;

namespace glc {
namespace {

constexpr int NT = 512, NW = NT / 32;
constexpr int BINS = SAMPLE_BINS;
constexpr int CAP = 512;         // tokens that are ranked at once, one per thread
constexpr int POWERS = SAMPLE_POWERS;
constexpr int DIGIT = 10;        // bits of the order per step of narrowing
constexpr int MAX_CLUSTER = 8;
constexpr int SLICE_MAX = 43008; // tokens of a CTA: 168 KB of its shared memory
constexpr int GROUPS = BINS / 32;
static_assert(3 << DIGIT <= BINS, "digits (three sums each) have a bin");
static_assert(CAP <= NT && GROUPS % 32 == 0, "a thread per listed token, a lane per group of bins");
static_assert(BINS <= 16 * NT && GROUPS <= NT && 32 * MAX_CLUSTER <= NT, "a thread per group, and per bin of a group and CTA");
static_assert(SLICE_MAX < (1 << 16), "sums of 16-bit numbers over a slice have 32 bits");
static_assert(SLICE_MAX / NT + 4 <= 127, "a thread's sum of weights");

struct Sample {
  const float* logits;
  size_t ld;
  int vocab, slice;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int64_t* tokens;
  float* logp;
};

using u64 = unsigned long long;

// Position in the order: larger is earlier.
__device__ __forceinline__ u64 order_of(float l, int index) {
  const uint32_t b = __float_as_uint(l + 0.f);  // -0 and 0 are equals
  const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (static_cast<u64>(key) << 32) | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float logit_of(u64 order) {
  const uint32_t key = static_cast<uint32_t>(order >> 32);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ int index_of(u64 order) { return static_cast<int>(~static_cast<uint32_t>(order)); }

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}
__device__ __forceinline__ u64 warp_scan(u64 x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

struct Shared {
  // what the CTAs of the row read of each other
  union {
    uint32_t hist[BINS];
    struct {  // a CTA's own, after the barrier behind which no histogram is read
      u64 pulled[CAP], ranked[CAP];
      uint32_t weights[CAP];
    };
  };
  u64 coarse[GROUPS];  // sums of the histogram over 32 bins
  u64 list[CAP];       // tokens near a cut
  int listed[2];       // how many, by the round's parity: a CTA may still read the last round's
  int first;
  // what they tell each other, by their rank
  float tops[MAX_CLUSTER], sums[MAX_CLUSTER];
  int finites[MAX_CLUSTER];
  u64 totals[2][MAX_CLUSTER], bases[MAX_CLUSTER];
  // a CTA's own
  u64 groups[GROUPS], parts[MAX_CLUSTER][32];
  SamplePower powers[POWERS];
  u64 warp_a[NW], warp_b[NW];
  float warp_f[NW], warp_top[NW];
  int warp_n[NW];
  int bin;           // where a histogram's sum reaches its goal,
  u64 base, in_bin;  // what lies before it and in it
  u64 cut;           // the last kept token of a filter
};
static_assert(MAX_CLUSTER <= 32, "a lane per CTA of a row");

// The sum over the block's threads of x before this thread's, and of all.
__device__ __forceinline__ u64 block_before(u64 x, u64* warps, u64* all, int lane, int warp) {
  const u64 s = warp_scan(x, lane);
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  u64 before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const u64 y = warps[i];
    if (i < warp) before += y;
    sum += y;
  }
  __syncthreads();
  *all = sum;
  return before + s - x;
}

__global__ void __launch_bounds__(NT, 2) sample_kernel(const Sample a) {
  GLC_PDL_ENTRY();
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& s = *reinterpret_cast<Shared*>(raw);
  float* x = reinterpret_cast<float*>(raw + (sizeof(Shared) + 15) / 16 * 16);
  uint32_t* wt = reinterpret_cast<uint32_t*>(x);  // in the logits' place
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  const int row = blockIdx.x / ctas;
  const int first = rank * a.slice;
  const int n = a.vocab - first < a.slice ? (a.vocab - first > 0 ? a.vocab - first : 0) : a.slice;
  const int n4 = (n + 3) >> 2;
  Shared& lead = *cluster.map_shared_rank(&s, 0);
  // A CTA's shared memory may be written to once all of the cluster have started:
  // they say so here and wait for it behind the logits' load.
  cluster.barrier_arrive();

  // ---- the row's settings
  const float temp = a.temperature[row];
  const float u = a.uniform[row];
  const int k_set = a.top_k ? a.top_k[row] : 0;
  const float p_set = a.top_p ? a.top_p[row] : 1.f;
  const float min_set = a.min_p ? a.min_p[row] : 0.f;
  const int k = k_set <= 0 || k_set > a.vocab ? a.vocab : k_set;
  const bool by_p = p_set < 1.f;
  const bool greedy = !(temp > 0.f) || k == 1 || p_set <= 0.f;

  // ---- the logits into shared memory, with their largest, and the mean of some
  const float* src = a.logits + row * a.ld + first;
  float top = -INFINITY, sum = 0.f;
  int finite = 0;
  auto some_of_mean = [&](float l) {
    const bool is = fabsf(l) <= FLT_MAX;
    sum += is ? l : 0.f;
    finite += is;
  };
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int whole4 = n >> 2;
#pragma unroll 8
    for (int i = tid; i < whole4; i += NT) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src) + i);
      top = fmaxf(fmaxf(top, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));  // (a NaN is passed over)
      some_of_mean(v.x);
      reinterpret_cast<float4*>(x)[i] = v;
    }
    for (int i = 4 * whole4 + tid; i < n; i += NT) {
      const float l = src[i];
      top = fmaxf(top, l);
      x[i] = l;
    }
  } else {
#pragma unroll 8
    for (int i = tid; i < n; i += NT) {
      const float l = __ldcs(src + i);
      top = fmaxf(top, l);
      some_of_mean(l);
      x[i] = l;
    }
  }
  if (n + tid < 4 * n4) x[n + tid] = __uint_as_float(0x7fc00000u);  // the last 4 tokens are whole
  if (tid < POWERS) s.powers[tid] = sample_power(tid);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    sum += __shfl_xor_sync(~0u, sum, o);
    finite += __shfl_xor_sync(~0u, finite, o);
  }
  if (lane == 0) s.warp_top[warp] = top, s.warp_f[warp] = sum, s.warp_n[warp] = finite;
  __syncthreads();
  cluster.barrier_wait();
  if (tid < ctas) {  // to each CTA of the row
    top = s.warp_top[0], sum = s.warp_f[0], finite = s.warp_n[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) top = fmaxf(top, s.warp_top[i]), sum += s.warp_f[i], finite += s.warp_n[i];
    Shared& o = *cluster.map_shared_rank(&s, tid);
    o.tops[rank] = top;
    o.sums[rank] = sum;
    o.finites[rank] = finite;
    if (tid == 0) s.first = INT_MAX;
  }
  cluster.sync();
  top = -INFINITY;
  sum = 0.f;
  finite = 0;
  for (int i = 0; i < ctas; ++i) {
    top = fmaxf(top, s.tops[i]);
    sum += s.sums[i];
    finite += s.finites[i];
  }

  auto finish = [&](int64_t token, float logp) {
    a.tokens[row] = token;
    if (a.logp) a.logp[row] = logp;
  };
  if (greedy || top == -INFINITY) {
    // the first of the largest
    int at = INT_MAX;
    if (top > -INFINITY)
      for (int i = tid; i < n4; i += NT) {
        const float4 v = reinterpret_cast<const float4*>(x)[i];
        const int j = v.x == top ? 0 : v.y == top ? 1 : v.z == top ? 2 : v.w == top ? 3 : 4;
        if (j < 4 && first + 4 * i + j < at) at = first + 4 * i + j;
      }
    at = __reduce_min_sync(~0u, at);
    if (lane == 0 && at != INT_MAX) atomicMin(&lead.first, at);
    cluster.sync();
    if (rank == 0 && tid == 0) finish(s.first == INT_MAX ? -1 : s.first, s.first == INT_MAX ? -INFINITY : 0.f);
    return;
  }
  const bool no_end = top > FLT_MAX;  // the infinite ones share all
  auto plain = [&](float l) { return !no_end ? l : l > FLT_MAX ? 0.f : -INFINITY; };
  if (no_end) {
    for (int i = tid; i < n; i += NT) x[i] = plain(x[i]);
    top = 0.f;
    __syncthreads();
    // (src is read again through plain)
  }

  SampleWeights weight;
  weight.top = top;
  const double inv = 1.0 / static_cast<double>(temp);
  weight.scale = inv * (POWERS * 1.4426950408889634);
  weight.powers = s.powers;
  // a token counts from this weight on; min_p >= 1 keeps the largest logit's equals
  const bool only_top = min_set >= 1.f;
  const double least_units = static_cast<double>(min_set) * SAMPLE_UNITS;
  const uint32_t least = only_top ? SAMPLE_ONE : least_units > 1.0 ? sample_code(least_units) : SAMPLE_LEAST;
  auto enough = [&](uint32_t w, auto logit) { return w >= least && (!only_top || logit() == top); };
  // the random number and p as 64-bit fractions; a goal is the high word of a product
  const u64 u64th = !(u > 0.f) ? 0 : u >= 1.f ? ~0ull : static_cast<u64>(static_cast<double>(u) * 18446744073709551616.0);
  const u64 p64 = by_p ? sample_share(p_set) : 0;
  auto p_goal = [&](u64 all) -> u64 { return sample_goal(all, p64); };

  // a token of the order up to `cut` (all but NaN and -infinity where it is 0)
  auto before_cut = [&](float l, int i, u64 cut) {
    if (!cut) return l > -INFINITY;
    const float c = logit_of(cut);
    return l > c || (l == c && first + i <= index_of(cut));
  };
  // bins of top - l for the count, the last one all that is beyond
  const float range = finite > 0 ? top - sum / static_cast<float>(finite) : 0.f;
  const float scale = range > 0.f ? static_cast<float>(BINS) / range : 0.f;
  auto count_bin = [&](float l) {
    // a whole number in the low bits of the sum; beyond 2^23 of them it stays the largest
    const int b = static_cast<int>(__float_as_uint(fmaf(top - l, scale, 8388608.f)) - 0x4b000000u);
    return b < 0 || b >= BINS ? BINS - 1 : b;
  };

  int round = 0;  // of histogram and list
  auto clear = [&] {
    for (int i = tid; i < BINS / 4; i += NT) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) s.listed[round & 1] = 0;
    __syncthreads();
  };
  // The row's histogram, found in each CTA by itself: the bin where its sum,
  // `base` with it, reaches the goal.  value(CTA, bin) is a bin of a CTA's;
  // goal_of(sum of all) the goal.  First in groups of 32 bins, then in one.
  auto locate = [&](int bins, u64 base, auto value, auto goal_of) {
    __syncthreads();
    {  // two threads have the bins of a group
      u64 y = 0;
      if (tid < bins / 16)
#pragma unroll
        for (int i = 0; i < 16; ++i) y += value(s, 16 * tid + ((i + tid) & 15));  // (each lane another bank)
      y += __shfl_xor_sync(~0u, y, 1);
      if (tid < bins / 16 && !(tid & 1)) s.coarse[tid / 2] = y;
    }
    cluster.sync();
    if (tid < GROUPS) {
      u64 y = 0;
      if (tid < bins / 32)
#pragma unroll
        for (int i = 0; i < MAX_CLUSTER; ++i) y += i < ctas ? cluster.map_shared_rank(&s, i)->coarse[tid] : 0;
      s.groups[tid] = y;
    }
    __syncthreads();
    u64 goal = 0;
    if (warp == 0) {
      u64 y[GROUPS / 32], sum_y = 0;
#pragma unroll
      for (int j = 0; j < GROUPS / 32; ++j) sum_y += y[j] = s.groups[GROUPS / 32 * lane + j];
      const u64 upto = warp_scan(sum_y, lane);
      goal = goal_of(__shfl_sync(~0u, upto, 31));
      u64 before = base + upto - sum_y;
      if (lane == 0) s.bin = 0, s.base = base, s.in_bin = 0;  // a goal that no bin reaches finds the first one
      __syncwarp();
#pragma unroll
      for (int j = 0; j < GROUPS / 32; ++j) {
        if (before < goal && goal <= before + y[j]) {
          s.bin = GROUPS / 32 * lane + j;
          s.base = before;
        }
        before += y[j];
      }
    }
    __syncthreads();
    const int group = s.bin;
    if (tid < 32 * MAX_CLUSTER) {
      const int peer = tid / 32;
      s.parts[peer][lane] = peer < ctas ? value(*cluster.map_shared_rank(&s, peer), 32 * group + lane) : 0;
    }
    __syncthreads();
    if (warp == 0) {
      u64 y = 0;
#pragma unroll
      for (int i = 0; i < MAX_CLUSTER; ++i) y += s.parts[i][lane];
      const u64 before = s.base + warp_scan(y, lane) - y;
      __syncwarp();
      if (before < goal && goal <= before + y) {
        s.bin = 32 * group + lane;
        s.base = before;
        s.in_bin = y;
      }
    }
    __syncthreads();
  };
  auto list = [&](float l, int i) {
    const int at = atomicAdd(&s.listed[round & 1], 1);
    if (at < CAP) s.list[at] = order_of(l, first + i);
  };
  auto list_place = [&](int i) {  // its logit is read later, with the others'
    const int at = atomicAdd(&s.listed[round & 1], 1);
    if (at < CAP) s.list[at] = i;
  };
  // after the lists' barrier: how many tokens they have; where that can be ranked
  // and `mine`, all of them in order, with weights
  auto rank_lists = [&](bool mine) {
    int m = lane < ctas ? cluster.map_shared_rank(&s, lane)->listed[round & 1] : 0;
    int upto = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += y;
    }
    m = __shfl_sync(~0u, upto, 31);
    if (m <= CAP && mine) {
      int peer = 0, at = tid;
#pragma unroll
      for (int i = 0; i < MAX_CLUSTER; ++i) {
        const int end = __shfl_sync(~0u, upto, i);
        if (i < ctas && tid >= end) peer = i + 1, at = tid - end;
      }
      const u64 order = tid < m ? cluster.map_shared_rank(&s, peer)->list[at] : 0;
      if (tid < CAP) s.pulled[tid] = order;
      __syncthreads();
      if (tid < m) {
        int r = 0;
#pragma unroll 8
        for (int i = 0; i < m; ++i) r += s.pulled[i] > order;
        s.ranked[r] = order;
        s.weights[r] = weight(logit_of(order));
      }
      __syncthreads();
    }
    return m;
  };
  // of the m ranked tokens, the last with less than the goal before it
  auto cut_of = [&](bool mass, int m, u64 base, u64 goal) {
    if (mass) {
      u64 all;
      const u64 w = tid < m ? sample_weight(s.weights[tid]) : 0;
      const u64 before = base + block_before(w, s.warp_a, &all, lane, warp);
      if (tid < m && before < goal && (tid == m - 1 || before + w >= goal)) s.cut = s.ranked[tid];
      __syncthreads();
      return s.cut;
    }
    const u64 last = s.ranked[goal - base - 1];
    __syncthreads();  // (a histogram may take the list's place)
    return last;
  };
  // A region of the order with more tokens than are ranked at once, narrowed by
  // the order's bits: the logits are read again.  in_region(l, i) says what it has.
  auto narrow = [&](bool mass, u64 base, u64 goal, auto in_region) -> u64 {
    u64 prefix = 0;
    int known = 64, shift = 64 - DIGIT;
    constexpr int DIGITS = 1 << DIGIT;
    for (int step = 0; step < 8; ++step) {  // 7 know all 64 bits, and then a bin has one token at most
      auto digit_of = [&](float l, int i) {
        if (!in_region(l, i)) return -1;
        const u64 o = order_of(l, first + i);
        if (known < 64 && (o >> known) != prefix) return -1;
        return (DIGITS - 1) - static_cast<int>((o >> shift) & (DIGITS - 1));
      };
      ++round;
      clear();
      for (int i = tid; i < n; i += NT) {
        const float l = plain(src[i]);
        const int d = digit_of(l, i);
        if (d < 0) continue;
        const u64 w = mass ? sample_weight(wt[i]) : 1;  // three numbers of 16 bits
        atomicAdd(&s.hist[d], static_cast<uint32_t>(w) & 0xffffu);
        if (w >> 16) {
          atomicAdd(&s.hist[DIGITS + d], static_cast<uint32_t>(w >> 16) & 0xffffu);
          atomicAdd(&s.hist[2 * DIGITS + d], static_cast<uint32_t>(w >> 32));
        }
      }
      locate(DIGITS, base, [](const Shared& o, int i) {
        return o.hist[i] + (static_cast<u64>(o.hist[DIGITS + i]) << 16) + (static_cast<u64>(o.hist[2 * DIGITS + i]) << 32);
      }, [&](u64) { return goal; });
      const int want = s.bin;
      base = s.base;
      for (int i = tid; i < n; i += NT) {
        const float l = plain(src[i]);
        if (digit_of(l, i) == want) list(l, i);
      }
      cluster.sync();
      const int m = rank_lists(true);
      if (m <= CAP) return cut_of(mass, m, base, goal);
      // the digit is known now; the last step's digit repeats bits that are
      const u64 digit = (DIGITS - 1) - want;
      prefix = known < 64 ? (prefix << (known - shift)) | (digit & ((1 << (known - shift)) - 1)) : digit;
      known = shift;
      shift = shift >= DIGIT ? shift - DIGIT : 0;
    }
    return 0;
  };

  // ---- top-k
  u64 cut = 0;  // the last token kept, all if 0
  if (k < a.vocab) {
    clear();
    uint32_t far = 0;  // the last bin, where most tokens are, is counted in registers
#pragma unroll 2
    for (int i = tid; i < n4; i += NT) {
      const float4 v = reinterpret_cast<const float4*>(x)[i];
      const float ls[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = count_bin(ls[j]);
        const bool is = ls[j] > -INFINITY;
        far += is && b == BINS - 1;
        if (is && b < BINS - 1) atomicAdd(&s.hist[b], 1u);
      }
    }
    far = __reduce_add_sync(~0u, far);
    if (lane == 0 && far) atomicAdd(&s.hist[BINS - 1], far);
    u64 goal = k;
    locate(BINS, 0, [](const Shared& o, int i) { return static_cast<u64>(o.hist[i]); }, [&](u64 all) {
      goal = goal < all ? goal : all;  // (the first warp's; below it is the others' too)
      if (lane == 0) s.warp_b[0] = goal;
      return goal;
    });
    goal = s.warp_b[0];
    const int want = s.bin;
    const u64 base = s.base;
    // with a few tokens to keep in all, everything down to the cut is listed
    const bool upto = base + s.in_bin <= CAP;
#pragma unroll 2
    for (int i = tid; i < n4; i += NT) {
      const float4 v = reinterpret_cast<const float4*>(x)[i];
      const float ls[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = count_bin(ls[j]);
        if (ls[j] > -INFINITY && (upto ? b <= want : b == want)) list(ls[j], 4 * i + j);
      }
    }
    cluster.sync();
    if (upto) {
      // the first CTA takes all of the first k and ends the row by itself
      if (rank == 0) rank_lists(true);
      cluster.sync();  // (the others' lists are read)
      if (rank) return;
      const int kept = static_cast<int>(goal);
      u64 all;
      uint32_t w = tid < kept ? s.weights[tid] : 0;
      const u64 before = block_before(sample_weight(w), s.warp_a, &all, lane, warp);
      if (by_p && before >= p_goal(all)) w = 0;
      if (w && !enough(w, [&] { return logit_of(s.ranked[tid]); })) w = 0;
      block_before(sample_weight(w), s.warp_a, &all, lane, warp);
      const int index = tid < kept ? index_of(s.ranked[tid]) : INT_MAX;
      if (tid < kept) s.pulled[tid] = sample_weight(w);
      __syncthreads();
      const u64 at = __umul64hi(all, u64th);
      if (w) {  // in index order: the token whose interval has the goal
        u64 lower = 0;
        for (int i = 0; i < kept; ++i) lower += index_of(s.ranked[i]) < index ? s.pulled[i] : 0;
        if (lower <= at && at < lower + sample_weight(w))
          finish(index, static_cast<float>((static_cast<double>(logit_of(s.ranked[tid])) - weight.top) * inv -
                                           log(static_cast<double>(all) * (1.0 / SAMPLE_UNITS))));
      }
      return;
    }
    const int m = rank_lists(true);
    cut = m <= CAP ? cut_of(false, m, base, goal)
                   : narrow(false, base, goal, [&](float l, int) { return l > -INFINITY && count_bin(l) == want; });
    ++round;
  }

  // ---- the weights, in the logits' place; of top-p, their histogram: sums of
  // their first 16 bits by bin, which is to say nearly where the cut is
  if (by_p) clear();
  SampleSum mine;
#pragma unroll 1
  for (int i = tid; i < n4; i += NT) {
    const float4 v = reinterpret_cast<const float4*>(x)[i];
    const float ls[4] = {v.x, v.y, v.z, v.w};
    uint32_t w[4], lead16[4];
    int bin[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = weight(ls[j], &bin[j], &lead16[j]);
    if (cut) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!before_cut(ls[j], 4 * i + j, cut)) w[j] = lead16[j] = 0;
    }
    if (by_p) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lead16[j]) atomicAdd(&s.hist[bin[j]], lead16[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) mine.add(w[j]);
    }
    reinterpret_cast<uint4*>(wt)[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // the sum of x over this CTA to all of the row, in totals[which]
  auto tell = [&](u64 sum_x, u64* (*place)(Shared&)) {
    sum_x = warp_sum(sum_x);
    if (lane == 0) s.warp_b[warp] = sum_x;
    __syncthreads();
    if (tid < ctas) {
      u64 all = 0;
#pragma unroll
      for (int i = 0; i < NW; ++i) all += s.warp_b[i];
      place(*cluster.map_shared_rank(&s, tid))[rank] = all;
    }
  };
  auto told = [&](const u64* from) {
    u64 all = 0;
    for (int i = 0; i < ctas; ++i) all += from[i];
    return all;
  };
  uint32_t cut_w = SAMPLE_LEAST;
  if (by_p) {
    tell(mine.value(), [](Shared& o) -> u64* { return o.totals[0]; });
    locate(BINS, 0, [](const Shared& o, int i) { return (static_cast<u64>(o.hist[i]) << 15) >> (i / POWERS); },
           [&](u64 all) { return p_goal(all); });
    int bin = s.bin;
    const u64 goal = p_goal(told(s.totals[0]));
    for (;;) {
      // the region of that bin in whole weights: exactly what is before it and in it
      const uint32_t high = sample_bin_top(bin), low = sample_bin_top(bin + 1);
      SampleSum more;
#pragma unroll 2
      for (int i = tid; i < n4; i += NT) {
        const uint4 v = reinterpret_cast<const uint4*>(wt)[i];
        const uint32_t ws[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (ws[j] > high) more.add(ws[j]);
          else if (ws[j] > low) list_place(4 * i + j);
        }
      }
      tell(more.value(), [](Shared& o) -> u64* { return o.bases; });
      if (tid < CAP && tid < s.listed[round & 1]) {  // (tell's barrier: the places are there)
        const int i = static_cast<int>(s.list[tid]);
        s.list[tid] = order_of(plain(src[i]), first + i);
      }
      cluster.sync();
      const u64 base = told(s.bases);
      const int m = rank_lists(true);
      // what the region has; of more tokens than can be ranked, summed in each CTA
      u64 inside = 0;
      if (m <= CAP) {
        block_before(tid < m ? sample_weight(s.weights[tid]) : 0, s.warp_a, &inside, lane, warp);
      } else {
        SampleSum y;
        for (int i = tid; i < n; i += NT)
          if (wt[i] > low && wt[i] <= high) y.add(wt[i]);
        tell(y.value(), [](Shared& o) -> u64* { return o.totals[1]; });
        cluster.sync();
        inside = told(s.totals[1]);
      }
      const int step = goal <= base ? -1 : goal > base + inside ? 1 : 0;
      if (step == 0 || bin + step < 0 || bin + step >= BINS) {
        cut = m <= CAP ? cut_of(true, m, base, goal)
                       : narrow(true, base, goal, [&](float, int i) { return wt[i] > low && wt[i] <= high; });
        break;
      }
      // the first 16 bits said a neighbour: once more.  (Close to 1 the cut is where a few
      // 10^-6 of the sum are many bins: 256 rows of 131075 take 237 us at top_p 0.95, 241 at
      // 0.999, 276 at 0.99999, 663 at 0.9999999.)
      bin += step;
      ++round;
      cluster.sync();
      if (tid == 0) s.listed[round & 1] = 0;
      __syncthreads();
    }
    cut_w = weight(logit_of(cut));
  } else {
    __syncthreads();
  }

  // ---- the draw: warps hold runs of the slice, so sums go in index order.  A
  // token with more than the cut's weight is before it, near that weight its logit
  // says (weights are not monotone to the last unit; those of top-k's dropped
  // tokens are 0)
  const uint32_t near_cut = by_p ? cut_w + SAMPLE_NEAR : 0;
  const uint32_t from_cut = cut_w > SAMPLE_NEAR + SAMPLE_LEAST ? cut_w - SAMPLE_NEAR : SAMPLE_LEAST;
  const uint32_t floor_w = from_cut > least ? from_cut : least;
  auto kept = [&](uint32_t w, int i) -> uint32_t {
    if (w < floor_w) return 0;
    if (w <= near_cut || only_top) {
      const float l = plain(src[i]);
      if ((only_top && l != top) || (by_p && !before_cut(l, i, cut))) return 0;
    }
    return w;
  };
  const int chunk = ((n + NW - 1) / NW + 127) & ~127;
  {
    SampleSum sum_w;
    const int end = (warp + 1) * chunk < n ? (warp + 1) * chunk : n;
#pragma unroll 2
    for (int i = warp * chunk + 4 * lane; i < end; i += 128) {
      const uint4 v = *reinterpret_cast<const uint4*>(wt + i);
      sum_w.add(kept(v.x, i));
      sum_w.add(kept(v.y, i + 1));
      sum_w.add(kept(v.z, i + 2));
      sum_w.add(kept(v.w, i + 3));
    }
    const u64 w = warp_sum(sum_w.value());
    if (lane == 0) s.warp_a[warp] = w;
    tell(lane == 0 ? w : 0, [](Shared& o) -> u64* { return o.totals[1]; });
  }
  cluster.sync();
  u64 all = 0, before = 0;
  for (int i = 0; i < ctas; ++i) {
    if (i < rank) before += s.totals[1][i];
    all += s.totals[1][i];
  }
  u64 goal = __umul64hi(all, u64th);
  if (goal >= before && goal - before < s.totals[1][rank]) {
    // this CTA's: the warp's run it falls in, split over the warps once more
    goal -= before;
    int w0 = 0;
    while (goal >= s.warp_a[w0]) goal -= s.warp_a[w0++];
    const int part = ((chunk + NW - 1) / NW + 31) & ~31;
    const int run0 = w0 * chunk, run1 = run0 + chunk < n ? run0 + chunk : n;
    const int p0 = run0 + warp * part, p1 = p0 + part < run1 ? p0 + part : run1;
    SampleSum sum_w;
    for (int i = p0 + lane; i < p1; i += 32) sum_w.add(kept(wt[i], i));
    const u64 w = warp_sum(sum_w.value());
    if (lane == 0) s.warp_b[warp] = w;
    __syncthreads();
    u64 at = 0;
    for (int i = 0; i < warp; ++i) at += s.warp_b[i];
    if (at <= goal && goal < at + w) {
      for (int i = p0; i < p1; i += 32) {
        const u64 mine = i + lane < p1 ? sample_weight(kept(wt[i + lane], i + lane)) : 0;
        const u64 upto = at + warp_scan(mine, lane);
        if (upto - mine <= goal && goal < upto)
          finish(first + i + lane,
                 static_cast<float>((static_cast<double>(plain(src[i + lane])) - weight.top) * inv -
                                    log(static_cast<double>(all) * (1.0 / SAMPLE_UNITS))));
        at = __shfl_sync(~0u, upto, 31);
        if (goal < at) break;
      }
    }
  }
}

}  // namespace
}  // namespace glc

using glc::Context;

extern "C" int glc_sample(glc_ctx* ctx, const float* logits, int ld, int rows, int vocab, const float* temperature,
                          const int* top_k, const float* top_p, const float* min_p, const float* uniform,
                          int64_t* tokens, float* logp) {
  if (!ctx) return GLC_ERR_INVALID;
  Context* c = reinterpret_cast<Context*>(ctx);
  auto no = [&](const char* why) { return c->fail(GLC_ERR_INVALID, std::string("sample: ") + why); };
  if (rows < 0 || vocab <= 0 || ld < vocab) return no("rows must not be negative, vocab positive, ld at least vocab");
  if (vocab > glc::MAX_CLUSTER * glc::SLICE_MAX)
    return c->fail(GLC_ERR_UNSUPPORTED, "sample: vocab must be at most 344064");
  if (rows == 0) return GLC_OK;
  if (!logits || !temperature || !uniform || !tokens) return no("logits, temperature, uniform and tokens must be given");
  if (((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(temperature) |
        reinterpret_cast<uintptr_t>(top_k) | reinterpret_cast<uintptr_t>(top_p) | reinterpret_cast<uintptr_t>(min_p) |
        reinterpret_cast<uintptr_t>(uniform) | reinterpret_cast<uintptr_t>(logp)) & 3) ||
      (reinterpret_cast<uintptr_t>(tokens) & 7))
    return no("a pointer is not aligned to its elements");
  if (rows > 0x7fffffff / glc::MAX_CLUSTER) return no("too many rows");
  glc::DeviceScope on(c);
  // CTAs of a row: as its slices need, and more while all of them run at once (128 rows
  // of 32000: 27 us with 2, 33 with 4); slices stay small enough for two CTAs on an SM
  // (256 rows of 131075: 231 us with 8, 250 with 4 and slices of 33000).  Above 139000
  // tokens one of 8 leaves no room for a second one: 256 rows of 139000 take 242 us, of
  // 141000 369, of 151936 395 and of 256000 542
  int ctas = 1;
  while (ctas < glc::MAX_CLUSTER && vocab / ctas > 1024 &&
         ((vocab + ctas - 1) / ctas > 16400 || static_cast<long long>(rows) * ctas <= c->num_sms))
    ctas *= 2;
  glc::Sample a{logits, static_cast<size_t>(ld), vocab, ((vocab + ctas - 1) / ctas + 3) & ~3, temperature, top_k,
                top_p, min_p, uniform, tokens, logp};
  const size_t smem = (sizeof(glc::Shared) + 15) / 16 * 16 + sizeof(float) * a.slice;
  static thread_local int ready = -1;
  if (ready != c->device) {
    const cudaError_t e = cudaFuncSetAttribute(
        glc::sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
        static_cast<int>((sizeof(glc::Shared) + 15) / 16 * 16 + sizeof(float) * (glc::SLICE_MAX + 4)));
    if (e != cudaSuccess) return c->fail_cuda(e, "sample: shared memory");
    ready = c->device;
  }
  glc::ProfScope prof(c, glc::PROF_OTHER, 4.0 * rows * vocab, c->stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * ctas);
  cfg.blockDim = dim3(glc::NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c->pdl ? 2 : 1;
  cudaLaunchKernelEx(&cfg, glc::sample_kernel, a);
  GLC_LAUNCH_CHECK(c, "sample");
  return GLC_OK;
}
