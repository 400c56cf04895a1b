// Test harness: the arithmetic of sampling (gollama_b200/csrc/sample_plan.h) on the
// host.  Built by tests/test_sample_plan.py; never linked into the library.
#include "../../gollama_b200/csrc/sample_plan.h"

extern "C" uint64_t sample_goal_of(uint64_t all, float p) { return glc::sample_goal(all, glc::sample_share(p)); }

// Weights, bins and leading bits of n logits below `top`.
extern "C" void sample_weights_of(float top, float temperature, const float* l, int n, uint32_t* w, int* bin, uint32_t* lead) {
  glc::SamplePower powers[glc::SAMPLE_POWERS];
  for (int j = 0; j < glc::SAMPLE_POWERS; ++j) powers[j] = glc::sample_power(j);
  const glc::SampleWeights weight{top, 1.0 / static_cast<double>(temperature) * (glc::SAMPLE_POWERS * 1.4426950408889634), powers};
  for (int i = 0; i < n; ++i) w[i] = weight(l[i], &bin[i], &lead[i]);
}
extern "C" int sample_bins() { return glc::SAMPLE_BINS; }
