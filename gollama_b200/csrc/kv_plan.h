// Where a token of the paged 4-bit key/value cache lies, which position of which
// sequence a row of the operands is, and how the attention over the cache cuts
// its work: the index arithmetic of kv_cache.cu and attention_kv.cu, for the
// device and, so that it can be checked without one, for the host.
#pragma once
#include <cstddef>
#include <cstdint>

#include "../../include/gollama_cuda.h"

#if defined(__CUDACC__)
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace glc {

constexpr int KV_GROUP = 32;         // elements that share a scale
constexpr int KV_BAD_ARGUMENT = 110; // GLC_DEV_BAD_ARGUMENT

// glc_kv_cache with the sizes that follow from it.
struct KvPools {
  uint8_t* k;
  uint8_t* v;
  int num_pages, page, kv_heads, head_dim;
  size_t chunk;   // bytes of one page of one head
  int scales_at;  // of them, where the scales begin
};
struct KvSeqs {
  const int* table;
  const int* lens;
  const int* starts;
  int seqs, max_pages, rows;
};

inline KvPools kv_pools(const glc_kv_cache& c) {
  KvPools p;
  p.k = static_cast<uint8_t*>(c.k);
  p.v = static_cast<uint8_t*>(c.v);
  p.num_pages = c.num_pages;
  p.page = c.page_size;
  p.kv_heads = c.num_kv_heads;
  p.head_dim = c.head_dim;
  p.chunk = static_cast<size_t>(c.page_size) * (c.head_dim / 16) * 9;
  p.scales_at = c.page_size * (c.head_dim / 2);
  return p;
}
inline KvSeqs kv_seqs(const glc_kv_batch& b) {
  return {b.page_table, b.lens, b.starts, b.num_seqs, b.max_pages, b.num_rows};
}

KV_HD void kv_bad(int* err) {
#if defined(__CUDA_ARCH__)
  atomicCAS(err, 0, KV_BAD_ARGUMENT);
#else
  if (*err == 0) *err = KV_BAD_ARGUMENT;
#endif
}

// The rows [first, first + n) of sequence b that hold its new tokens, and its
// length.  Where the length is not within the table or the rows are not within the
// operands the error word is set and there are no rows: a length cut to the table's
// would put the new tokens on the slots of its last ones.
struct KvSpan {
  int first, n, len;
  bool bad;  // its starts do not ascend within the operands' rows
};
KV_HD KvSpan kv_span(const KvSeqs& s, int page, int b, int* err) {
  KvSpan r;
  r.len = s.lens[b];
  const int most = s.max_pages * page;  // at most 2^30, checked by the host
  const bool fits = r.len >= 0 && r.len <= most;
  if (!fits) {
    kv_bad(err);
    r.len = 0;
  }
  r.first = b;
  r.n = 1;
  r.bad = false;
  if (s.starts) {
    r.first = s.starts[b];
    const int end = s.starts[b + 1];
    if (r.first < 0 || end < r.first || end > s.rows) {
      kv_bad(err);
      r.first = 0;
      r.n = 0;
      r.bad = true;
    } else {
      r.n = end - r.first;
    }
  }
  if (!fits) r.n = 0;
  return r;
}

// Sequence and position of row t: false where the row belongs to no sequence
// or its position is negative.  With starts, the last sequence that begins at
// or before t.
KV_HD bool kv_row(const KvSeqs& s, int page, int t, int* err, int* seq, int* pos) {
  int b = t;
  if (s.starts) {
    int lo = 0, hi = s.seqs;  // starts[lo] <= t < starts[hi], when it holds at all
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s.starts[mid] <= t) lo = mid;
      else hi = mid;
    }
    b = lo;
  } else if (t >= s.seqs) {
    return false;
  }
  const KvSpan r = kv_span(s, page, b, err);
  const int i = t - r.first;
  if (i < 0 || i >= r.n) return false;
  *seq = b;
  *pos = r.len - r.n + i;
  return *pos >= 0;
}

// Every step-th sequence from `first` on is looked at for its rows and length alone:
// where starts do not ascend, a row's search may pass by the pair that is wrong.
KV_HD void kv_look(const KvSeqs& s, int page, long long first, long long step, int* err) {
  if (!s.starts) return;  // a row is a sequence
  for (long long b = first; b < s.seqs; b += step) kv_span(s, page, static_cast<int>(b), err);
}

// Page `index` of sequence b; -1 (and the error word) where the table has none.
KV_HD int kv_page(const KvSeqs& s, int num_pages, int b, int index, int* err) {
  const int p = s.table[static_cast<size_t>(b) * s.max_pages + index];
  if (p < 0 || p >= num_pages) {
    kv_bad(err);
    return -1;
  }
  return p;
}

// ---------------------------------------------------------------- attention

constexpr int KV_WK = 32;  // keys of a warp's tile

// The sequences' rows are disjoint only if every one's starts ascend: only then is the
// sum of their units what the host allowed for, so one bad pair ends the whole call.

// The items of one KV head of a sequence.  A tile of `rt` query rows holds the
// heads of `toks` whole tokens, or, where a group has more heads than that, up to
// rt heads of one token (`parts` tiles per token).  Tile i sees the keys of its
// last token, in units of `unit` keys, one at least (an item without keys still
// writes its rows).
struct KvRows {
  int first, n, len, toks, parts, tiles;
  bool bad;
};
KV_HD KvRows kv_rows(const KvSeqs& s, int page, int toks, int parts, int b, int* err) {
  const KvSpan r = kv_span(s, page, b, err);
  KvRows w;
  w.first = r.first;
  w.n = r.n;
  w.len = r.len;
  w.bad = r.bad;
  w.toks = toks;
  w.parts = parts;
  w.tiles = r.n <= toks ? (r.n ? parts : 0) : (r.n + toks - 1) / toks * parts;
  return w;
}
// Keys seen by the last token of the run of tokens `run`.
KV_HD int kv_run_keys(const KvRows& w, int run) {
  const int last = (run + 1) * w.toks < w.n ? (run + 1) * w.toks : w.n;
  const int keys = w.len - w.n + last;
  return keys < 0 ? 0 : keys;
}
KV_HD int kv_run_units(const KvRows& w, int run, int unit) {
  const int u = (kv_run_keys(w, run) + unit - 1) / unit;
  return u < 1 ? 1 : u;
}
// One past the last run with as many units as `run` has: the runs' keys grow by
// `toks` each, so equals are counted by a division, not one by one.
KV_HD int kv_run_equals(const KvRows& w, int run, int units, int unit) {
  const long long room = static_cast<long long>(units) * unit - (w.len - w.n);  // new tokens that fit
  if (room >= w.n) return w.tiles / w.parts;
  const int end = static_cast<int>(room) / w.toks;
  return end > run ? end : run + 1;
}
// The sum over the tiles of a head of their units, in pieces of `per` units
// (per = 1: the units).
KV_HD int kv_head_pieces(const KvRows& w, int unit, int per) {
  if (w.tiles == w.parts) {  // one run of tokens
    const int u = kv_run_units(w, 0, unit);
    return (per == 1 ? u : (u + per - 1) / per) * w.parts;
  }
  const int runs = w.tiles / w.parts;
  int sum = 0;
  for (int i = 0; i < runs;) {
    const int u = kv_run_units(w, i, unit), next = kv_run_equals(w, i, u, unit);
    sum += (per == 1 ? u : (u + per - 1) / per) * (next - i) * w.parts;
    i = next;
  }
  return sum;
}
// The tile in which piece `at` of a head lies: its first piece and its units.
KV_HD int kv_find_tile(const KvRows& w, int unit, int per, int at, int* first, int* units) {
  const int runs = w.tiles / w.parts;
  int sum = 0;
  for (int i = 0; i < runs;) {
    const int u = kv_run_units(w, i, unit), next = kv_run_equals(w, i, u, unit);
    const int pieces = (u + per - 1) / per, all = pieces * (next - i) * w.parts;
    if (at < sum + all) {
      const int skip = (at - sum) / pieces;
      *first = sum + skip * pieces;
      *units = u;
      return i * w.parts + skip;
    }
    sum += all;
    i = next;
  }
  *first = sum;
  *units = 1;
  return 0;
}

// The kernel that a call takes: query tiles of 8 rows of an item (0: one tile of 4 rows)
// and warps of a CTA.  By the rows that share a KV head of a sequence, on average: as many
// query tiles in an item as they fill, since an item unpacks its keys and values once.
//   up to 4 rows: hi and lo as neighbouring columns of one product, 145 -> 123 us (64
//     x 8192 tokens, 32/8 heads of 128);
//   narrow heads, more than 24 rows: four tiles (items of 8 rows took 522 us for a
//     512-token chunk on 4096, 32/4 heads of 64, items of up to 32 take 409);
//   wide heads, 17 to 24 rows: three tiles, 60.5 -> 53.8 us (5 tokens each, 32/8 heads
//     of 128).  For longer chunks two (785 us, three 845), and for 24 rows of narrow
//     heads two (23.4 us, three 25.0): fewer registers, more warps.
// Few items are cut between many CTAs, and few large CTAs leave fewer parts to
// join: one sequence of 131072 tokens (32/4 heads of 64) 23.6 us against 39.5 with
// CTAs of 4 warps, of 16384 11.0 against 22.2.  Of many items a CTA has several, and
// small CTAs overlap one's joins with another's copies: 32 sequences of 2048 take
// 14.4 and 14.5 us.
struct KvVariant {
  int tiles, warps;
};
inline KvVariant kv_variant(int head_dim, long long rows, int seqs, int group, int kv_heads, int sms) {
  const long long shared = rows * group / seqs;
  if (head_dim <= 64 && shared > 24) return {4, 4};
  if (head_dim >= 96 && shared > 16 && shared <= 24) return {3, 4};
  if (shared > 8) return {2, 4};
  const bool many = rows * ((group + 7) / 8) * kv_heads >= sms / 2;
  return {shared <= 4 ? 0 : 1, many ? 4 : 16};
}
// Its CTAs of an SM: 12 warps of 168 registers, of narrow heads 16 of 128.  More warps
// with fewer registers compute addresses again and again (measured before tiles took
// their own maximum, 12 instructions more): at 128 a tile of 128
// elements takes 757 instructions, at 168 680 (64 x 8192 tokens, 32/8 heads of
// 128: 114.5 and 111.7 us); a tile of 64 at 96, 128 and 168 takes 560, 513 and 464
// (128 x 4096 tokens, 32/4 heads of 64: 49.2, 45.8 and 48.0 us).
constexpr int kv_per_sm(int head_dim, int tiles, int warps) {
  return warps >= 12 ? 1 : (tiles > 2 && head_dim >= 96 ? 8 : tiles > 1 || head_dim >= 96 ? 12 : 16) / warps;
}

// Units that a call may have, at most: they are counted in 32 bits.  Of all variants
// the tiles of 4 rows and the units of 128 keys make the most.
inline double kv_most_units(double rows, double seqs, double group, double kv_heads, double max_pages, double page) {
  const double parts = static_cast<double>((static_cast<long long>(group) + 3) / 4);
  return (rows * parts + seqs) * kv_heads * (max_pages * page / (4 * KV_WK) + 1);
}

// Of `total` units, CTA c of `ctas` (at most total) has a run of total / ctas, the
// first total % ctas of them one more: where its run begins, and the CTA of a unit.
KV_HD int kv_cta_begin(int cta, int total, int ctas) {
  const int base = total / ctas, more = total - base * ctas;
  return base * cta + (cta < more ? cta : more);
}
KV_HD int kv_cta_of(int unit, int total, int ctas) {
  const int base = total / ctas, more = total - base * ctas, head = (base + 1) * more;
  return unit < head ? unit / (base + 1) : more + (unit - head) / base;
}
// Items cut into even pieces of at most `per` units, one for each CTA, beat runs
// of units that pass from item to item, as long as `per` is near the average:
// how far it may go from the least that could do (32 sequences of up to 2048 tokens:
// 16.4 us in runs, 14.3 in pieces).
KV_HD int kv_most_per(int least) { return least + (least < 8 ? 1 : least / 8); }

// Where a CTA is in its share of the work: units [at, end) of all, in the item
// [item_at, item_at + units).  alone: the share is one piece of one item, which the
// CTAs first to last share.
struct KvPlace {
  int at, end, item_at, units, total, ctas;
  int alone, first, last;
  int b, h, tile;
  KvRows w;
};
// The CTAs that share the item.
KV_HD int kv_first_cta(const KvPlace& p) { return p.alone ? p.first : kv_cta_of(p.item_at, p.total, p.ctas); }
KV_HD int kv_last_cta(const KvPlace& p) { return p.alone ? p.last : kv_cta_of(p.item_at + p.units - 1, p.total, p.ctas); }
// The place of the CTA whose share begins at piece `at` of sequence b's (in pieces
// of `per` units where `alone`, else in units), all before b being `before`.
KV_HD void kv_place(KvPlace* p, const KvRows& w, int b, int unit, int per, int alone, int cta, int at, int before) {
  const int per_head = kv_head_pieces(w, unit, per);
  p->h = at / per_head;
  p->b = b;
  p->w = w;
  p->alone = alone;
  int first = 0;
  if (w.tiles == 1) {
    p->tile = 0;
    p->units = kv_run_units(w, 0, unit);
  } else {
    p->tile = kv_find_tile(w, unit, per, at - p->h * per_head, &first, &p->units);
  }
  const int piece = at - p->h * per_head - first;  // of the tile
  if (alone) {
    p->item_at = 0;
    p->at = piece * per;
    p->end = p->at + per < p->units ? p->at + per : p->units;
    p->first = cta - piece;
    p->last = p->first + (p->units + per - 1) / per - 1;
  } else {
    p->item_at = before + at - piece;
    p->at = before + at;
    p->end = kv_cta_begin(cta + 1, p->total, p->ctas);
  }
}

// A tile of KV_WK keys in shared memory: codes of the keys, codes of the
// values, scales of the keys, scales of the values.
template <int HD>
struct KvTile {
  static constexpr int NB = HD / KV_GROUP;       // scales of a token, and 16-byte pieces of its codes
  static constexpr int ROW = HD / 2;             // bytes of its codes
  static constexpr int CODES = KV_WK * ROW;
  static constexpr int SCALES = KV_WK * NB * 2;
  static constexpr int BYTES = 2 * (CODES + SCALES);
  // 8 lanes copy one side of one group of 16 tokens, in 16-byte pieces: lane i
  // the pieces i + 8 j of the codes, and piece i of the scales if there is one.
  static constexpr int LANE_PIECES = 2 * NB;
  static constexpr int GROUP_SCALES = 2 * NB;
  static_assert(16 * ROW == 8 * LANE_PIECES * 16, "a group's codes");

  // Byte of piece `ch` of a token.  The pieces are swizzled so that a piece of 8
  // tokens falls in 8 different quads of banks.
  static KV_HD int code_at(int token, int ch) {
    return token * ROW + 16 * (HD == 128 ? ch ^ ((token >> 1) & 3) : HD == 64 ? ch ^ ((token >> 2) & 1) : ch);
  }
  // Where piece i + 8 j of the codes goes, relative to piece i's unswizzled
  // place: the tokens of 8 pieces in a row share their swizzle.
  static KV_HD int swizzle(int j) { return HD == 128 ? (j & 3) << 4 : HD == 64 ? (j & 1) << 4 : 0; }
  // The first byte of a side of a group in the tile: of its codes and scales.
  static KV_HD int codes_of(int side, int grp) { return side * CODES + grp * 16 * ROW; }
  static KV_HD int scales_of(int side, int grp) { return 2 * CODES + side * SCALES + grp * 32 * NB; }
};

// The page (index in the sequence) and the slot in it, both in groups of 16
// tokens, of a group that walks a sequence in equal steps.
struct KvWalk {
  int index, slot;
  KV_HD void start(int key, int page16) {
    index = (key >> 4) / page16;
    slot = (key >> 4) - index * page16;
  }
  KV_HD void advance(int step_index, int step_slot, int page16) {
    index += step_index;
    slot += step_slot;
    if (slot >= page16) slot -= page16, ++index;
  }
};

}  // namespace glc
