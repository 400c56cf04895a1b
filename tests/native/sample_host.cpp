// Test harness: the arithmetic of sampling (gollama_b200/csrc/sample_plan.h) on the
// host.  Built by tests/test_sample_plan.py; never linked into the library.
#include "../../gollama_b200/csrc/sample_plan.h"

extern "C" uint64_t sample_goal_of(uint64_t all, float p) { return glc::sample_goal(all, glc::sample_share(p)); }
