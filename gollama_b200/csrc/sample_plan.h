// The whole numbers that sample.cu draws with, for the device and, so that they
// can be checked without one, for the host.
#pragma once
#include <cmath>
#include <cstdint>
#include <cstring>

#if defined(__CUDACC__)
#define SAMPLE_HD __host__ __device__ __forceinline__
#else
#define SAMPLE_HD inline
#endif

namespace glc {

SAMPLE_HD uint32_t sample_bits(float x) {
#if defined(__CUDA_ARCH__)
  return __float_as_uint(x);
#else
  uint32_t y;
  std::memcpy(&y, &x, sizeof y);
  return y;
#endif
}
SAMPLE_HD uint64_t sample_bits(double x) {
#if defined(__CUDA_ARCH__)
  return __double_as_longlong(x);
#else
  uint64_t y;
  std::memcpy(&y, &x, sizeof y);
  return y;
#endif
}
SAMPLE_HD uint64_t sample_high(uint64_t x, uint64_t y) {  // of the product's 128 bits
#if defined(__CUDA_ARCH__)
  return __umul64hi(x, y);
#else
  return static_cast<uint64_t>(static_cast<unsigned __int128>(x) * y >> 64);
#endif
}

// A share p in (0, 1) of a sum as a 64-bit fraction, 2^-64 at least: a smaller one
// asks for the first token as 2^-64 does, and a goal of zero would be reached by no
// token.
SAMPLE_HD uint64_t sample_share(float p) {
  const uint64_t x = static_cast<uint64_t>(static_cast<double>(p) * 18446744073709551616.0);
  return x ? x : 1;
}
// The least whole number not below that share of `all`.
SAMPLE_HD uint64_t sample_goal(uint64_t all, uint64_t share) { return sample_high(all, share) + (all * share != 0); }

// ---------------------------------------------------------------- weights

constexpr int SAMPLE_POWERS = 256;              // bins, and table entries, per factor of two of the weight
constexpr int SAMPLE_BINS = 32 * SAMPLE_POWERS;  // the last one has all that is smaller too
constexpr float SAMPLE_ROUND = 12582912.f;  // 1.5 2^23: added to a number below 2^22, the nearest whole one in the low bits

// A weight has 27 bits and is held as its code, which orders as the weights do: the 26
// bits after its first one, and above them the place of the first one, counted from 1 at
// 2^-UNIT of the largest (0: no weight).  In sums it counts in whole units of 2^-UNIT, cut
// off: sums of up to 344064 weights are then exact below 2^64, and do not depend on their
// order.  Weights in whole numbers of 2^-31, as 32 bits would hold them without a place,
// lose the tail of a row: 131074 equal tokens 22 temperatures below one are 3.7e-5 of the
// sum and came out as 6.1e-5, 22.2 below as nothing.
constexpr int SAMPLE_UNIT = 45;
constexpr double SAMPLE_UNITS = 35184372088832.0;          // 2^UNIT
constexpr uint32_t SAMPLE_ONE = (SAMPLE_UNIT + 1u) << 26;  // the largest
constexpr uint32_t SAMPLE_LEAST = 1u << 26;                // one unit
// Weights of logits next to each other may come out in the wrong order by one in the
// 27th bit.
constexpr uint32_t SAMPLE_NEAR = 4;
SAMPLE_HD uint64_t sample_weight(uint32_t code) {
  const uint64_t m = (code & 0x03ffffffu) | 0x04000000u;
  return (m << (SAMPLE_UNIT - 26)) >> (SAMPLE_UNIT + 1 - (code >> 26));
}
// The code of x units, cut off, x in [1, 2^UNIT]: the number's own first bits.
SAMPLE_HD uint32_t sample_code(double x) { return static_cast<uint32_t>((sample_bits(x) >> 26) - (1022ull << 26)); }
// The weights of bin b are those up to this code and above the next bin's.
SAMPLE_HD uint32_t sample_bin_top(int b) {
  return b < SAMPLE_BINS ? sample_code(exp2(SAMPLE_UNIT - b * (1.0 / SAMPLE_POWERS))) : 0;
}
// A sum of up to 127 weights: whole numbers in the low bits of 2^52 and more, to which a
// code's number is added and cut off (that of code 0 is 1/2); 4 instructions each, the
// weights themselves take 11.
struct SampleSum {
  double x = 4503599627370496.0;
  SAMPLE_HD void add(uint32_t code) {
#if defined(__CUDA_ARCH__)
    x = __dadd_rd(x, __hiloint2double(static_cast<int>((code >> 6) + (1022u << 20)), static_cast<int>(code << 26)));
#else
    x += static_cast<double>(sample_weight(code));
#endif
  }
  SAMPLE_HD uint64_t value() const { return sample_bits(x) & ((1ull << 52) - 1); }
};

// 2^(31 - (j + 1/2) / 256), as the whole number less the bits of ROUND (and 8 more, half
// of the 27th bit), and as a float.
struct SamplePower {
  uint32_t whole;
  float power;
};
SAMPLE_HD SamplePower sample_power(int j) {
  const double y = exp2(31.0 - (j + 0.5) * (1.0 / SAMPLE_POWERS));
  return {static_cast<uint32_t>(y + 0.5) + 8 + sample_bits(SAMPLE_ROUND), static_cast<float>(y)};
}
// The whole number at or below x y, in the low bits of the sum with 1.5 2^52.
SAMPLE_HD double sample_floor(double x, double y) {
#if defined(__CUDA_ARCH__)
  return __fma_rd(x, y, 6755399441055744.0);
#else
  return std::floor(x * y) + 6755399441055744.0;
#endif
}

struct SampleWeights {
  double top, scale;  // scale: 256 log2(e) / temperature
  const SamplePower* powers;
  // (top - l) / temperature = (256 q + j + 1/2 + f) ln2 / 256, |f| <= 1/2, f exact to
  // 2^-25: 2^-q by the code's place, 2^(-(j + 1/2)/256) from the table, 1 - exp(-f ln2 /
  // 256) by three terms of its series (the fourth is below 2^-41), rounded to 2^-31
  // before it is taken off.  *bin: 256 q + j, held to the last one; *lead: of the weight
  // times 2^bin's q, the first 16 bits.  A logit that is -infinity or not a number has
  // weight 0.
  SAMPLE_HD uint32_t operator()(float l, int* bin, uint32_t* lead) const {
    const double d = top - static_cast<double>(l);
    const double k = sample_floor(d, scale);
    const float f = static_cast<float>(fma(d, scale, 6755399441055744.0 - k)) - 0.5f;
    // the bin itself is compared, since 1 / temperature may pass what a float holds, and a
    // difference of logits that is next to nothing is then many bins away all the same;
    // after UNIT places weights are below a unit
    const bool some = k < 6755399441055744.0 + SAMPLE_UNIT * SAMPLE_POWERS;
    const int n = some ? static_cast<int>(sample_bits(k)) : 0;
    constexpr float L = static_cast<float>(0.6931471805599453 / SAMPLE_POWERS);
    const float y = f * fmaf(f, fmaf(f, L * L * L / 6, -L * L / 2), L);
    const SamplePower p = powers[n & (SAMPLE_POWERS - 1)];
    const uint32_t w = p.whole - sample_bits(fmaf(p.power, y, SAMPLE_ROUND));  // [2^30, 2^31] + 8, off by 2 at most
    const int q = n / SAMPLE_POWERS;
    *bin = n < SAMPLE_BINS ? n : SAMPLE_BINS - 1;
    *lead = some ? w >> (q > 31 ? q - 16 : 15) : 0;
    return some ? (w >> 4) + (static_cast<uint32_t>(SAMPLE_UNIT - 1 - q) << 26) : 0;
  }
  SAMPLE_HD uint32_t operator()(float l) const {
    int bin;
    uint32_t lead;
    return (*this)(l, &bin, &lead);
  }
};

}  // namespace glc
