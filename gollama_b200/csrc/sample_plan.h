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
SAMPLE_HD int sample_low_bits(double x) {
#if defined(__CUDA_ARCH__)
  return __double2loint(x);
#else
  uint64_t y;
  std::memcpy(&y, &x, sizeof y);
  return static_cast<int>(static_cast<uint32_t>(y));
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
constexpr int SAMPLE_BINS = 32 * SAMPLE_POWERS;
constexpr float SAMPLE_ROUND = 12582912.f;  // 1.5 2^23: added to a number below 2^22, the nearest whole one in the low bits

// 2^(31 - j / 256), as the whole number less the bits of ROUND, and as a float.
struct SamplePower {
  uint32_t whole;
  float power;
};
SAMPLE_HD SamplePower sample_power(int j) {
  const double y = exp2(31.0 - j * (1.0 / SAMPLE_POWERS));
  return {static_cast<uint32_t>(y + 0.5) + sample_bits(SAMPLE_ROUND), static_cast<float>(y)};
}

struct SampleWeights {
  double top, scale;  // scale: 256 log2(e) / temperature
  const SamplePower* powers;
  // (top - l) / temperature = (256 q + j + f) ln2 / 256, |f| <= 1/2, f exact to 2^-40:
  // 2^-q by a shift, 2^(-j/256) from the table, 1 - exp(-f ln2 / 256) by three terms
  // of its series (the fourth is below 2^-41), rounded to units before it is taken
  // off.  *bin: 256 q + j; *lead: the weight's first 16 bits, before the shift.
  // A logit that is -infinity or not a number has weight 0.
  SAMPLE_HD uint32_t operator()(float l, int* bin, uint32_t* lead) const {
    const double d = top - static_cast<double>(l);
    const double k = fma(d, scale, 6755399441055744.0);  // 1.5 2^52: the whole number in the low bits
    const float f = static_cast<float>(fma(d, scale, 6755399441055744.0 - k));
    // the bin itself is held below the last one, beyond which weights round to 0 or 1:
    // 1 / temperature may pass what a float holds, and a difference of logits that is
    // next to nothing is then many bins away all the same
    const bool some = k < 6755399441055744.0 + (SAMPLE_BINS - 1);
    const int n = some ? sample_low_bits(k) : SAMPLE_BINS - 1;
    constexpr float L = static_cast<float>(0.6931471805599453 / SAMPLE_POWERS);
    const float y = f * fmaf(f, fmaf(f, L * L * L / 6, -L * L / 2), L);
    const SamplePower p = powers[n & (SAMPLE_POWERS - 1)];
    const uint32_t w = p.whole - sample_bits(fmaf(p.power, y, SAMPLE_ROUND));
    const int q = n / SAMPLE_POWERS;
    *bin = n;
    *lead = some ? w >> 15 : 0;
    return some ? (w + ((1u << q) >> 1)) >> q : 0;
  }
  SAMPLE_HD uint32_t operator()(float l) const {
    int bin;
    uint32_t lead;
    return (*this)(l, &bin, &lead);
  }
};

}  // namespace glc
