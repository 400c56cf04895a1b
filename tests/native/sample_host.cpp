// Test harness: the arithmetic of sampling (gollama_b200/csrc/sample_plan.h) on the
// host.  Built by tests/test_sample_plan.py; never linked into the library.
#include "../../gollama_b200/csrc/sample_plan.h"

extern "C" uint64_t sample_goal_of(uint64_t all, float p) { return glc::sample_goal(all, glc::sample_share(p)); }

// Weights (in units of 2^-SAMPLE_UNIT), bins, leading bits and codes of n logits below `top`.
extern "C" void sample_weights_of(float top, float temperature, const float* l, int n, uint64_t* w, int* bin, uint32_t* lead,
                                  uint32_t* code) {
  glc::SamplePower powers[glc::SAMPLE_POWERS];
  for (int j = 0; j < glc::SAMPLE_POWERS; ++j) powers[j] = glc::sample_power(j);
  const glc::SampleWeights weight{top, 1.0 / static_cast<double>(temperature) * (glc::SAMPLE_POWERS * 1.4426950408889634), powers};
  for (int i = 0; i < n; ++i) {
    code[i] = weight(l[i], &bin[i], &lead[i]);
    w[i] = glc::sample_weight(code[i]);
  }
}
extern "C" int sample_bins() { return glc::SAMPLE_BINS; }
extern "C" int sample_unit() { return glc::SAMPLE_UNIT; }
extern "C" uint32_t sample_code_of(double x) { return glc::sample_code(x); }
extern "C" uint64_t sample_weight_of(uint32_t code) { return glc::sample_weight(code); }
extern "C" uint32_t sample_near() { return glc::SAMPLE_NEAR; }
extern "C" uint32_t sample_bin_top_of(int bin) { return glc::sample_bin_top(bin); }
