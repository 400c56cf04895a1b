// Test harness: the look at all sequences of a call that glc_kv_append and glc_kv_read
// take (gollama_b200/csrc/kv_plan.h), as `threads` threads do.  Built by
// tests/test_kv_starts.py; never linked into the library.
#include "../../gollama_b200/csrc/kv_plan.h"

extern "C" int kv_look_of(const glc_kv_cache* cache, const glc_kv_batch* batch, int threads) {
  int err = 0;
  for (int i = 0; i < threads; ++i) glc::kv_look(glc::kv_seqs(*batch), cache->page_size, i, threads, &err);
  return err;
}
