// Test harness: the kernel that the attention over the 4-bit cache takes for a call
// and how it cuts the work, from gollama_b200/csrc/kv_plan.h on the host.  Built by
// tests/test_kv_variants.py; never linked into the library.
#include <algorithm>

#include "../../gollama_b200/csrc/kv_plan.h"

using namespace glc;

// out: query tiles, warps, whether each CTA has one piece of one item, the most units
// that a CTA has of one item, items cut between CTAs, items
extern "C" int kv_shape(const glc_kv_cache* cache, const glc_kv_batch* batch, int group, int sms, int* out) {
  const KvPools c = kv_pools(*cache);
  const KvSeqs s = kv_seqs(*batch);
  int err = 0;
  const KvVariant v = kv_variant(c.head_dim, s.rows, s.seqs, group, c.kv_heads, sms);
  const int rt = v.tiles ? 8 * v.tiles : 4, unit = v.warps * KV_WK;
  const int toks = group < rt ? rt / group : 1, parts = (group + rt - 1) / rt;
  const int grid = sms * kv_per_sm(c.head_dim, v.tiles, v.warps);
  auto pieces = [&](int per) {
    int sum = 0;
    for (int b = 0; b < s.seqs; ++b) sum += kv_head_pieces(kv_rows(s, c.page, toks, parts, b, &err), unit, per) * c.kv_heads;
    return sum;
  };
  const int total = pieces(1), ctas = std::min(total, grid), least = (total + ctas - 1) / ctas;
  int per = 1, alone = 0;
  for (int i = least; i <= kv_most_per(least) && !alone; i += least < 16 ? 1 : least / 16)
    if (pieces(i) <= grid) per = i, alone = 1;
  int at = 0, most = 0, cut = 0, items = 0;
  for (int b = 0; b < s.seqs; ++b) {
    const KvRows w = kv_rows(s, c.page, toks, parts, b, &err);
    for (int h = 0; h < c.kv_heads; ++h)
      for (int tile = 0; tile < w.tiles; ++tile, ++items) {
        const int units = kv_run_units(w, tile / w.parts, unit);
        if (alone) {
          most = std::max(most, std::min(per, units));
          cut += units > per;
        } else {
          int first = kv_cta_of(at, total, ctas), last = kv_cta_of(at + units - 1, total, ctas);
          cut += first != last;
          for (int x = first; x <= last; ++x)
            most = std::max(most, std::min(at + units, kv_cta_begin(x + 1, total, ctas)) - std::max(at, kv_cta_begin(x, total, ctas)));
        }
        at += units;
      }
  }
  const int r[] = {v.tiles, v.warps, alone, most, cut, items};
  std::copy(r, r + 6, out);
  return err;
}
