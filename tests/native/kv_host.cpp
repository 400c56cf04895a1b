// Test harness: the index arithmetic of the paged 4-bit cache and of the
// attention over it (gollama_b200/csrc/kv_plan.h) walked on the host as the
// kernels walk it, and a context without a device for the tests of refused
// arguments.  Built by tests/test_kv_plan.py; never linked into the library.
#include <algorithm>
#include <cstring>
#include <map>
#include <set>
#include <vector>

#include "../../gollama_b200/csrc/glc_internal.h"
#include "../../gollama_b200/csrc/kv_plan.h"

using namespace glc;

// A context whose calls can be refused (they return before they touch a
// device); it is never destroyed through the library.
extern "C" void* test_context() {
  auto* c = new Context();
  c->num_sms = 148;
  return c;
}
extern "C" void test_context_free(void* c) { delete static_cast<Context*>(c); }

namespace {

// 0, or a number that names what went wrong
template <int HD>
int walk(const KvPools& c, const KvSeqs& s, int group, int rt, int warps, int grid, int* err) {
  using Tile = KvTile<HD>;
  const int unit = warps * KV_WK;
  const int toks = group < rt ? rt / group : 1, parts_of = (group + rt - 1) / rt;
  auto rows_of = [&](int b) { return kv_rows(s, c.page, toks, parts_of, b, err); };
  for (int b = 0; b < s.seqs; ++b)
    if (rows_of(b).bad) {  // the kernel's CTAs all return
      for (int i = b; i < s.seqs; ++i) rows_of(i);
      return 0;
    }
  long long all = 0;
  for (int b = 0; b < s.seqs; ++b) all += static_cast<long long>(kv_head_pieces(rows_of(b), unit, 1)) * c.kv_heads;
  if (all > kv_most_units(s.rows, s.seqs, group, c.kv_heads, s.max_pages, c.page)) return 100;
  auto pieces_of = [&](int per) {
    int sum = 0;
    for (int b = 0; b < s.seqs; ++b) sum += kv_head_pieces(rows_of(b), unit, per) * c.kv_heads;
    return sum;
  };
  const int total = pieces_of(1);
  const int ctas = std::min(total, grid);
  const size_t pool = static_cast<size_t>(c.num_pages) * c.kv_heads * c.chunk;
  // the shares as the kernel finds them
  int per = 1, alone = 0, used = ctas;
  if (ctas > 0) {
    const int least = (total + ctas - 1) / ctas;
    for (int i = least; i <= kv_most_per(least); i += least < 16 ? 1 : least / 16)
      if (pieces_of(i) <= grid) {
        per = i;
        alone = 1;
        used = pieces_of(i);
        break;
      }
  }
  // (sequence, head, tile) -> per key how often it was read; and who wrote it
  std::map<std::vector<int>, std::vector<int>> seen;
  std::map<std::vector<int>, std::vector<std::pair<int, int>>> parts;  // (cta, slot) of an item's parts
  std::map<int, int> arrivals, needed;
  std::set<std::vector<int>> whole;
  for (int cta = 0; cta < used; ++cta) {
    const int begin = alone ? cta : kv_cta_begin(cta, total, ctas);
    if (!alone) {
      if (begin >= kv_cta_begin(cta + 1, total, ctas)) return 1;
      for (int x = begin; x < kv_cta_begin(cta + 1, total, ctas); ++x)
        if (kv_cta_of(x, total, ctas) != cta) return 2;
    }
    KvPlace p = {};
    p.total = total;
    p.ctas = ctas;
    int before = 0, b = 0;
    for (; b < s.seqs; ++b) {
      const int y = kv_head_pieces(rows_of(b), unit, per) * c.kv_heads;
      if (begin < before + y) break;
      before += y;
    }
    if (b == s.seqs) return 3;
    kv_place(&p, rows_of(b), b, unit, per, alone, cta, begin - before, before);
    const int page16 = c.page >> 4, step_pages = (unit / 16) / page16, step_slot = (unit / 16) % page16;
    for (;;) {
      const KvRows& w = p.w;
      const int item_end = p.item_at + p.units, seg_end = std::min(item_end, p.end), at = p.at, tile = p.tile, h = p.h;
      b = p.b;
      if (at < p.item_at || at >= seg_end) return 4;
      const int run_at = tile / w.parts, part_at = tile - run_at * w.parts;
      const int keys = kv_run_keys(w, run_at);
      const int key0 = (at - p.item_at) * unit;
      const int key1 = std::min((seg_end - p.item_at) * unit, keys);
      const int tok0 = run_at * w.toks, head0 = part_at * rt;
      const int width = group < rt ? group : std::min(group - head0, rt);
      const int rows = std::min(w.n - tok0, w.toks) * width;
      if (rows < 1 || rows > rt || head0 + width > group) return 5;
      auto& count = seen[{b, h, tile}];
      count.resize(keys);
      for (int warp = 0; warp < warps; ++warp) {
        KvWalk g[2];
        int next = key0 + warp * KV_WK;
        for (int i = 0; i < 2; ++i) g[i].start(next + 16 * i, page16);
        for (int key = next; key < key1; key += unit) {
          std::set<int> to_all;
          size_t base[2] = {0, 0};
          bool ok[2];
          for (int i = 0; i < 2; ++i) {
            const int k = key + 16 * i;
            ok[i] = false;
            if (k < key1) {
              if (g[i].index != k / c.page || g[i].slot != k % c.page / 16) return 6;
              if (g[i].index >= s.max_pages) return 7;
              const int p = kv_page(s, c.num_pages, b, g[i].index, err);
              ok[i] = p >= 0;
              base[i] = (ok[i] ? static_cast<size_t>(p) * c.kv_heads * c.chunk : 0) + h * c.chunk;
            }
          }
          for (int lane = 0; lane < 32; ++lane) {
            const int lane8 = lane & 7, side = lane >> 4, i = (lane >> 3) & 1;
            for (int j = 0; j < Tile::LANE_PIECES; ++j) {
              const int to = Tile::codes_of(side, i) + ((lane8 * 16) ^ Tile::swizzle(j & 3)) + 128 * j;
              const int token = (lane8 + 8 * j) * 16 / Tile::ROW, ch = (lane8 + 8 * j) % Tile::NB;
              if (to % 16 || !to_all.insert(to).second) return 8;
              if (to != side * Tile::CODES + Tile::code_at(16 * i + token, ch)) return 9;
              if (!ok[i]) continue;
              const size_t src = base[i] + static_cast<size_t>(g[i].slot) * 16 * Tile::ROW + lane8 * 16 + 128 * j;
              if (src + 16 > pool || src % 16) return 10;
              if (src - base[i] != static_cast<size_t>((key + 16 * i) % c.page + token) * Tile::ROW + 16 * ch) return 11;
              if (src - base[i] + 16 > static_cast<size_t>(c.scales_at)) return 11;
              if (side == 0 && ch == 0 && key + 16 * i + token < key1) ++count[key + 16 * i + token];
            }
            if (lane8 < Tile::GROUP_SCALES) {
              const int to = Tile::scales_of(side, i) + lane8 * 16;
              if (to < 2 * Tile::CODES || to + 16 > Tile::BYTES || !to_all.insert(to).second) return 12;
              if (!ok[i]) continue;
              const size_t src = base[i] + c.scales_at + static_cast<size_t>(g[i].slot) * 32 * Tile::NB + lane8 * 16;
              if (src + 16 > base[i] + c.chunk || src + 16 > pool || src % 16) return 13;
            }
          }
          if (to_all.size() * 16 != Tile::BYTES) return 23;
          for (int i = 0; i < 2; ++i) g[i].advance(step_pages, step_slot, page16);
        }
      }
      if (at == p.item_at && seg_end == item_end) {
        if (!whole.insert({b, h, tile}).second) return 14;
      } else {
        const int first = kv_first_cta(p), last = kv_last_cta(p);
        parts[{b, h, tile}].push_back({cta, at == p.item_at ? 1 : 0});
        if ((cta == first) != (at == p.item_at) || cta < first || cta > last) return 15;
        ++arrivals[first];
        needed[first] = last - first + 1;
      }
      if (p.alone || item_end >= p.end) break;
      p.at = p.item_at = item_end;
      if (++p.tile == p.w.tiles) {
        p.tile = 0;
        if (++p.h == c.kv_heads) {
          p.h = 0;
          do {
            if (++p.b >= s.seqs) return 16;
            p.w = rows_of(p.b);
          } while (p.w.tiles == 0);
        }
      }
      p.units = kv_run_units(p.w, p.tile / p.w.parts, unit);
    }
  }
  for (auto& a : arrivals)
    if (a.second != needed[a.first]) return 17;
  for (auto& p : parts) {
    if (whole.count(p.first)) return 18;
    std::set<std::pair<int, int>> distinct(p.second.begin(), p.second.end());
    if (distinct.size() != p.second.size()) return 19;
  }
  // every item once, every key of it that has a page once
  for (int b = 0; b < s.seqs; ++b) {
    const KvRows w = rows_of(b);
    int covered = 0;
    for (int h = 0; h < c.kv_heads; ++h)
      for (int tile = 0; tile < w.tiles; ++tile) {
        const std::vector<int> id{b, h, tile};
        if (!whole.count(id) && !parts.count(id)) return 20;
        const auto& count = seen[id];
        for (size_t k = 0; k < count.size(); ++k) {
          const int p = s.table[static_cast<size_t>(b) * s.max_pages + k / c.page];
          if (count[k] != (p >= 0 && p < c.num_pages ? 1 : 0)) return 21;
        }
      }
    for (int i = 0; i < w.tiles; i += w.parts) covered += std::min(w.toks, w.n - i / w.parts * w.toks);
    if (covered != w.n) return 22;
  }
  return 0;
}

}  // namespace

extern "C" int kv_walk(const glc_kv_cache* cache, const glc_kv_batch* batch, int group, int rt, int warps, int grid,
                       int* err) {
  const KvPools c = kv_pools(*cache);
  const KvSeqs s = kv_seqs(*batch);
  switch (c.head_dim) {
    case 32: return walk<32>(c, s, group, rt, warps, grid, err);
    case 64: return walk<64>(c, s, group, rt, warps, grid, err);
    case 96: return walk<96>(c, s, group, rt, warps, grid, err);
    case 128: return walk<128>(c, s, group, rt, warps, grid, err);
  }
  return -1;
}

// Rows of kv_append and kv_read: sequence and position of each (-1: none).
extern "C" void kv_rows_of(const glc_kv_cache* cache, const glc_kv_batch* batch, int* seq, int* pos, int* err) {
  const KvSeqs s = kv_seqs(*batch);
  for (int t = 0; t < s.rows; ++t) {
    seq[t] = -1;
    pos[t] = -1;
    int b, p;
    if (kv_row(s, cache->page_size, t, err, &b, &p)) {
      seq[t] = b;
      pos[t] = p;
    }
  }
}

// Quads of banks that a piece of 8 tokens falls in (8: no conflict).
extern "C" int kv_bank_quads(int hd, int token0, int ch) {
  std::set<int> quads;
  for (int i = 0; i < 8; ++i) {
    const int at = hd == 32 ? KvTile<32>::code_at(token0 + i, ch) : hd == 64 ? KvTile<64>::code_at(token0 + i, ch)
                   : hd == 96 ? KvTile<96>::code_at(token0 + i, ch) : KvTile<128>::code_at(token0 + i, ch);
    quads.insert(at / 16 % 8);
  }
  return static_cast<int>(quads.size());
}
