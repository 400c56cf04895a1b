// The whole numbers that sample.cu draws with, for the device and, so that they
// can be checked without one, for the host.
#pragma once
#include <cstdint>

#if defined(__CUDACC__)
#define SAMPLE_HD __host__ __device__ __forceinline__
#else
#define SAMPLE_HD inline
#endif

namespace glc {

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

}  // namespace glc
