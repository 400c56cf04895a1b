// Drawing the next token: temperature, top-k, top-p, min-p, and the inverse of
// the kept tokens' running sum at a given random number.
//
// A token's weight is exp((l - max) / temperature) as a whole number of 2^-42,
// so sums of weights are exact and every order of summation gives the same one.
// The weights themselves are good to 2^-39: with tens of thousands of tokens
// kept, a sum that is off by 2^-25 of itself (float32 exponentials) moves past a
// token's edge about once in a thousand rows, and that token is then another.  Tokens are ordered by (logit falling, index rising), a total order; the
// kept ones of top-k and of top-p are each a prefix of it, so each filter is a
// cut: its last kept token.  Nothing is sorted but the few tokens around a
// cut: a histogram over 1024 bins of max - l finds the bin the cut falls in,
// that bin's tokens (or, for a small k, all down to it) are gathered and
// ranked against each other.  A bin of more than 512 tokens is first narrowed
// by the bits of the order itself, 10 at a time, which ends for any input,
// equal logits too.  The draw itself is a sum over the kept tokens in index
// order, taken apart in CTAs, warps and lanes.
//
// A cluster of 1 to 8 CTAs holds a row in shared memory, so the logits are read
// once; the histograms, the gathered tokens and the partial sums meet in the
// first CTA through distributed shared memory.
#include <cfloat>
#include <climits>
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace cg = cooperative_groups;

namespace glc {
namespace {

constexpr int NT = 512, NW = NT / 32;
constexpr int BINS = 1024;
constexpr int CAP = NT;  // tokens that are ranked at once, one per thread
constexpr int MAX_CLUSTER = 8;
constexpr int SLICE_MAX = 49152;  // tokens of a CTA: 192 KB of its shared memory

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

constexpr int POWERS = 32;

struct Weights {
  float top, c;         // c: 1 / temperature, for what needs no more than 24 bits
  double dtop, inv;     // 1 / temperature
  const double* powers; // 2^(42 - j / 32)
  // round(2^42 exp(-y)), y = (top - l) / temperature = (32 q + j) ln2 / 32 + r with
  // |r| <= ln2 / 64: 2^-q by a shift, 2^(-j/32) from the table, exp(-r) by four
  // terms of its series (r^5 / 120 < 2^-39).
  __device__ __forceinline__ u64 operator()(float l) const {
    const float d = l == top ? 0.f : top - l;
    if (!(d * c < 29.8f)) return 0;  // below 2^-43; and where l is -infinity or not a number
    const double y = (l == top ? 0.0 : dtop - static_cast<double>(l)) * inv;
    const double k = fma(y, 32 * 1.4426950408889634, 6755399441055744.0);  // 1.5 2^52: the whole number in the low bits
    const int n = __double2loint(k);
    const double r = fma(k - 6755399441055744.0, -0.6931471805599453 / 32, y);
    double e = fma(r, 1.0 / 24, -1.0 / 6);
    e = fma(r, e, 0.5);
    e = fma(r, e, -1.0);
    e = fma(r, e, 1.0);
    const double v = fma(powers[n & (POWERS - 1)], e, 4503599627370496.0);  // 2^52: the rounded value in the low bits
    const u64 whole = static_cast<u64>(__double_as_longlong(v)) & 0xfffffffffffffull;
    return whole >> (n >> 5);
  }
};

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
  uint32_t low[BINS], high[BINS];  // a histogram of 64-bit sums, halves apart
  u64 list[CAP], ranked[CAP];
  u64 warp_a[NW], warp_b[NW];
  float warp_f[NW], warp_top[NW];
  int warp_n[NW];
  double powers[POWERS];
  // what the other CTAs read
  float top, sum;
  int first, finite;
  u64 total;
  int gathered[2];  // by the level's parity: a CTA may still read the last level's
  int bin;         // of the last histogram: where the cut falls,
  u64 base, all;   // what lies before that bin, and the whole sum
  uint32_t in_bin; // (of a count) and what is in it
  u64 cut;         // the last kept token of a filter
};

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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  const int row = blockIdx.x / ctas;
  const int first = rank * a.slice;
  const int n = a.vocab - first < a.slice ? (a.vocab - first > 0 ? a.vocab - first : 0) : a.slice;
  Shared& lead = *cluster.map_shared_rank(&s, 0);

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
    if (fabsf(l) <= FLT_MAX) sum += l, ++finite;
  };
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int n4 = n >> 2;
#pragma unroll 8
    for (int i = tid; i < n4; i += NT) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(src) + i);
      top = fmaxf(fmaxf(top, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));  // (a NaN is passed over)
      some_of_mean(v.x);
      reinterpret_cast<float4*>(x)[i] = v;
    }
    for (int i = 4 * n4 + tid; i < n; i += NT) {
      const float l = src[i];
      top = fmaxf(top, l);
      some_of_mean(l);
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
  if (tid < POWERS) s.powers[tid] = exp2(42.0 - tid * (1.0 / POWERS));
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    sum += __shfl_xor_sync(~0u, sum, o);
    finite += __shfl_xor_sync(~0u, finite, o);
  }
  if (lane == 0) s.warp_top[warp] = top, s.warp_f[warp] = sum, s.warp_n[warp] = finite;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < NW; ++i) {
      top = fmaxf(top, s.warp_top[i]);
      sum += s.warp_f[i];
      finite += s.warp_n[i];
    }
    s.top = top;
    s.sum = sum;
    s.finite = finite;
    s.first = INT_MAX;
  }
  cluster.sync();
  top = -INFINITY;
  sum = 0.f;
  finite = 0;
  for (int i = 0; i < ctas; ++i) {
    const Shared& o = *cluster.map_shared_rank(&s, i);
    top = fmaxf(top, o.top);
    sum += o.sum;
    finite += o.finite;
  }

  auto finish = [&](int64_t token, float logp) {
    a.tokens[row] = token;
    if (a.logp) a.logp[row] = logp;
  };
  if (greedy || top == -INFINITY) {
    // the first of the largest; each CTA's own, then the first CTA that has one
    int at = INT_MAX;
    if (top > -INFINITY)
      for (int i = tid; i < n; i += NT)
        if (x[i] == top && first + i < at) at = first + i;
    at = __reduce_min_sync(~0u, at);
    if (lane == 0 && at != INT_MAX) atomicMin(&lead.first, at);
    cluster.sync();
    if (rank == 0 && tid == 0) finish(s.first == INT_MAX ? -1 : s.first, s.first == INT_MAX ? -INFINITY : 0.f);
    return;
  }

  Weights weight;
  weight.top = top;
  weight.dtop = top;
  weight.inv = 1.0 / static_cast<double>(temp);
  weight.c = static_cast<float>(fmin(weight.inv, static_cast<double>(FLT_MAX)));
  weight.powers = s.powers;
  // a token counts from this weight on; min_p >= 1 keeps the largest logit's equals
  const u64 least = min_set > 0.f && min_set < 1.f
                        ? static_cast<u64>(ceil(static_cast<double>(min_set) * 4398046511104.0))
                        : 0;
  const bool only_top = min_set >= 1.f;
  auto enough = [&](float l, u64 w) { return w >= least && (!only_top || l == top); };
  // the random number and p as 64-bit fractions; a goal is the high word of a product
  const u64 u64th = !(u > 0.f) ? 0 : u >= 1.f ? ~0ull : static_cast<u64>(static_cast<double>(u) * 18446744073709551616.0);

  // ---- a filter's cut.  mass: the tokens of the order up to `from` are weighed
  // until p64/2^64 of them all; else they are counted to `target`.  The bins
  // divide [0, range] of top - l evenly, the last one has all that is beyond.
  auto before_cut = [&](float l, int i, u64 from) {  // l is not NaN or -infinity
    if (!from) return l > -INFINITY;
    const float c = logit_of(from);
    return l > c || (l == c && first + i <= index_of(from));
  };
  auto bin_of = [&](float l, float scale) {
    const float d = l == top ? 0.f : top - l;
    // a whole number in the low bits of the sum; beyond 2^23 of them it stays the largest
    const int b = static_cast<int>(__float_as_uint(fmaf(d, scale, 8388608.f)) - 0x4b000000u);
    return b < 0 || b >= BINS ? BINS - 1 : b;
  };
  // tokens the level looks at: of bin `bin0` alone once level > 0, and of them
  // those whose order has the prefix for its bits from `known` on
  auto digit_of = [&](float l, int i, u64 from, float scale, int level, int bin0, int shift, int known, u64 prefix) {
    if (!before_cut(l, i, from)) return -1;
    const int b = bin_of(l, scale);
    if (level == 0) return b;
    if (b != bin0) return -1;
    const u64 o = order_of(l, first + i);
    if (known < 64 && (o >> known) != prefix) return -1;
    return (BINS - 1) - static_cast<int>((o >> shift) & (BINS - 1));
  };
  // one histogram over the cluster; afterwards s.bin, s.base, s.all and
  // s.in_bin of the first CTA hold where `target` (mass: set from its sum at
  // level 0) falls
  auto histogram = [&](bool mass, u64* target, u64 base, u64 p64, u64 from, float scale, int level, int bin0, int shift,
                       int known, u64 prefix) {
    for (int i = tid; i < BINS; i += NT) s.low[i] = s.high[i] = 0;
    if (tid == 0) s.gathered[level & 1] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const float l = x[i];
      const int d = digit_of(l, i, from, scale, level, bin0, shift, known, prefix);
      if (d < 0) continue;
      if (!mass) {
        atomicAdd(&s.low[d], 1u);
      } else {
        const u64 w = weight(l);
        if (w == 0) continue;
        const uint32_t lo = static_cast<uint32_t>(w), hi = static_cast<uint32_t>(w >> 32);
        const uint32_t carry = atomicAdd(&s.low[d], lo) > ~lo ? 1u : 0u;
        if (hi + carry) atomicAdd(&s.high[d], hi + carry);
      }
    }
    cluster.sync();
    if (rank == 0) {
      u64 v[2] = {0, 0};
      for (int i = 0; i < ctas; ++i) {
        const Shared& o = *cluster.map_shared_rank(&s, i);
#pragma unroll
        for (int j = 0; j < 2; ++j) v[j] += (static_cast<u64>(o.high[2 * tid + j]) << 32) + o.low[2 * tid + j];
      }
      u64 all;
      const u64 before = block_before(v[0] + v[1], s.warp_a, &all, lane, warp) + base;
      u64 goal = *target;
      if (level == 0) {  // the least whole number not below p * all; no more tokens than there are
        if (mass) goal = __umul64hi(all, p64) + (all * p64 != 0);
        else if (goal > all) goal = all;
      }
      // the first bin whose sum with all before it reaches the goal
      if (before < goal && goal <= before + v[0] + v[1]) {
        const int j = goal <= before + v[0] ? 0 : 1;
        s.bin = 2 * tid + j;
        s.base = before + (j ? v[0] : 0);
        s.in_bin = static_cast<uint32_t>(v[j]);
      }
      if (tid == 0) s.all = goal;
    }
    cluster.sync();
    *target = lead.all;
  };
  // tokens of the level's bin `want` (level 0 with `upto`: of all bins to it)
  // gathered in the first CTA; how many there are
  auto gather = [&](u64 from, float scale, int level, int bin0, int shift, int known, u64 prefix, int want, bool upto) {
    for (int i = tid; i < n; i += NT) {
      const float l = x[i];
      const int d = digit_of(l, i, from, scale, level, bin0, shift, known, prefix);
      if (d < 0 || (upto ? d > want : d != want)) continue;
      const int at = atomicAdd(&lead.gathered[level & 1], 1);
      if (at < CAP) lead.list[at] = order_of(l, first + i);
    }
    cluster.sync();
    return lead.gathered[level & 1];
  };
  // (first CTA) the list in order
  auto rank_list = [&](int m) {
    if (tid < m) {
      const u64 mine = s.list[tid];
      int r = 0;
      for (int i = 0; i < m; ++i) r += s.list[i] > mine;
      s.ranked[r] = mine;
    }
    __syncthreads();
  };
  auto narrow = [&](bool mass, u64 target, u64 p64, u64 from, float scale, bool all_listed, bool* listed) -> u64 {
    u64 base = 0, prefix = 0;
    int level = 0, bin0 = 0, shift = 54, known = 64;
    *listed = false;
    // 7 steps of 10 bits know all 64, and then a bin holds one token at most
    for (; level < 9; ++level) {
      histogram(mass, &target, base, p64, from, scale, level, bin0, shift, known, prefix);
      const int bin = lead.bin;
      base = lead.base;
      // with a few tokens to keep in all, everything down to the cut is listed
      const bool upto = all_listed && level == 0 && base + lead.in_bin <= CAP;
      const int m = gather(from, scale, level, bin0, shift, known, prefix, bin, upto);
      if (m <= CAP) {
        if (rank == 0) {
          rank_list(m);
          if (upto) base = 0;
          if (mass) {
            const u64 w = tid < m ? weight(logit_of(s.ranked[tid])) : 0;
            u64 all;
            const u64 before = block_before(w, s.warp_a, &all, lane, warp) + base;
            // the last token with less than the goal before it
            if (tid < m && before < target && (tid == m - 1 || before + w >= target)) s.cut = s.ranked[tid];
          } else if (tid == 0) {
            s.cut = s.ranked[target - base - 1];
          }
          __syncthreads();
        }
        *listed = upto;
        if (!upto) cluster.sync();  // the cut is there for the others
        return lead.cut;
      }
      if (level == 0) {
        bin0 = bin;
      } else {  // the digit is known now; the last step's digit repeats bits that are
        prefix = known < 64 ? (prefix << (known - shift)) | (((BINS - 1) - bin) & ((1 << (known - shift)) - 1))
                            : static_cast<u64>((BINS - 1) - bin);
        known = shift;
        shift = shift >= 10 ? shift - 10 : 0;
      }
    }
    return 0;
  };

  u64 cut = 0;  // the last token kept, all if 0
  const float range = top <= FLT_MAX && finite > 0 ? top - sum / static_cast<float>(finite) : 0.f;
  if (k < a.vocab) {
    bool listed;
    const float scale = range > 0.f ? static_cast<float>(BINS) / range : 0.f;
    cut = narrow(false, static_cast<u64>(k), 0, 0, scale, true, &listed);
    if (listed) {
      // ---- the first CTA has all of the first k: it ends the row by itself
      if (rank == 0) {
        const u64 mine = tid < k && tid < CAP ? s.ranked[tid] : 0;
        const bool some = tid < k && tid < s.gathered[0];
        const float l = logit_of(mine);
        u64 w = some ? weight(l) : 0, all;
        u64 before = block_before(w, s.warp_a, &all, lane, warp);
        if (by_p) {
          const u64 p64 = static_cast<u64>(static_cast<double>(p_set) * 18446744073709551616.0);
          const u64 goal = __umul64hi(all, p64) + (all * p64 != 0);
          if (before >= goal && tid > 0) w = 0;
        }
        if (!enough(l, w)) w = 0;
        // in index order: the weight of the kept tokens up to each one
        s.list[tid] = w ? static_cast<u64>(index_of(mine)) : ~0ull;
        s.ranked[tid] = w;
        block_before(w, s.warp_a, &all, lane, warp);  // (its barriers: list and ranked are there)
        if (w) {
          u64 upto = 0;
          const int m = k < CAP ? k : CAP;
          for (int i = 0; i < m; ++i) upto += s.list[i] <= s.list[tid] ? s.ranked[i] : 0;
          const u64 goal = __umul64hi(all, u64th);
          if (upto - w <= goal && goal < upto)
            finish(index_of(mine), static_cast<float>(log(static_cast<double>(w) / static_cast<double>(all))));
        }
      }
      cluster.sync();
      return;
    }
  }
  if (by_p) {
    bool listed;
    // beyond 29.8 / c every weight is 0; half as far behind the mean as before it, few tokens are left
    float r = 29.8f / weight.c;
    if (range > 0.f && 1.5f * range < r) r = 1.5f * range;
    const float scale = r > 0.f && r <= FLT_MAX ? static_cast<float>(BINS) / r : 0.f;
    const u64 p64 = static_cast<u64>(static_cast<double>(p_set) * 18446744073709551616.0);
    const u64 c = narrow(true, 0, p64, cut, scale, false, &listed);
    cut = c > cut ? c : cut;
  }

  // ---- the draw: warps hold runs of the slice, so sums go in index order
  const float cut_l = cut ? logit_of(cut) : -INFINITY;
  const int cut_i = cut ? index_of(cut) : -1;
  auto kept = [&](int i) -> u64 {
    const float l = x[i];
    if (!(l > cut_l || (l == cut_l && first + i <= cut_i))) return 0;
    const u64 w = weight(l);
    return enough(l, w) ? w : 0;
  };
  const int chunk = ((n + NW - 1) / NW + 31) & ~31;
  {
    u64 w = 0;
    const int end = (warp + 1) * chunk < n ? (warp + 1) * chunk : n;
    for (int i = warp * chunk + lane; i < end; i += 32) w += kept(i);
    w = warp_sum(w);
    if (lane == 0) s.warp_a[warp] = w;
    __syncthreads();
    if (tid == 0) {
      u64 all = 0;
      for (int i = 0; i < NW; ++i) all += s.warp_a[i];
      s.total = all;
    }
  }
  cluster.sync();
  u64 all = 0, before = 0;
  for (int i = 0; i < ctas; ++i) {
    const u64 y = cluster.map_shared_rank(&s, i)->total;
    if (i < rank) before += y;
    all += y;
  }
  u64 goal = __umul64hi(all, u64th);
  if (goal >= before && goal - before < s.total) {
    // this CTA's: the warp's run it falls in, split over the warps once more
    goal -= before;
    int w0 = 0;
    while (goal >= s.warp_a[w0]) goal -= s.warp_a[w0++];
    const int part = ((chunk + NW - 1) / NW + 31) & ~31;
    const int run0 = w0 * chunk, run1 = run0 + chunk < n ? run0 + chunk : n;
    const int p0 = run0 + warp * part, p1 = p0 + part < run1 ? p0 + part : run1;
    u64 w = 0;
    for (int i = p0 + lane; i < p1; i += 32) w += kept(i);
    w = warp_sum(w);
    if (lane == 0) s.warp_b[warp] = w;
    __syncthreads();
    u64 at = 0;
    for (int i = 0; i < warp; ++i) at += s.warp_b[i];
    if (at <= goal && goal < at + w) {
      for (int i = p0; i < p1; i += 32) {
        const u64 mine = i + lane < p1 ? kept(i + lane) : 0;
        const u64 upto = at + warp_scan(mine, lane);
        if (upto - mine <= goal && goal < upto)
          finish(first + i + lane, static_cast<float>(log(static_cast<double>(mine) / static_cast<double>(all))));
        at = __shfl_sync(~0u, upto, 31);
        if (goal < at) break;
      }
    }
  }
  cluster.sync();  // the others may still read this CTA's memory
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
    return c->fail(GLC_ERR_UNSUPPORTED, "sample: vocab must be at most 393216");
  if (rows == 0) return GLC_OK;
  if (!logits || !temperature || !uniform || !tokens) return no("logits, temperature, uniform and tokens must be given");
  if (((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(temperature) |
        reinterpret_cast<uintptr_t>(top_k) | reinterpret_cast<uintptr_t>(top_p) | reinterpret_cast<uintptr_t>(min_p) |
        reinterpret_cast<uintptr_t>(uniform) | reinterpret_cast<uintptr_t>(logp)) & 3) ||
      (reinterpret_cast<uintptr_t>(tokens) & 7))
    return no("a pointer is not aligned to its elements");
  if (rows > 0x7fffffff / glc::MAX_CLUSTER) return no("too many rows");
  glc::DeviceScope on(c);
  // CTAs of a row: until the device is full, and as its slice needs
  int ctas = 1;
  while (ctas < glc::MAX_CLUSTER &&
         (static_cast<long long>(rows) * ctas < 2 * c->num_sms || (vocab + ctas - 1) / ctas > 16400) &&
         vocab / ctas > 1024)
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
