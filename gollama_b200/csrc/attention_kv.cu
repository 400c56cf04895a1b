// Attention of new tokens over the paged 4-bit key/value cache.
//
// For a query row q and the keys k_j = d_j (n_j - 8) it sees (n the 4-bit
// codes, d one scale per 32 elements), the running form of the softmax over
// tiles of keys:
//   s_j = q . k_j * log2(e) / sqrt(hd),  m' = max(m, max s_j),
//   p_j = 2^(s_j - max s_j),  w = 2^(max s_j - m'),
//   l = l 2^(m - m') + w sum p_j,  o = o 2^(m - m') + w sum p_j v_j.
//
// Codes become matrix operands without being scaled: two of them OR'ed into the
// mantissas of two halves are 1024 + n (or 1024 + 16 n), and one packed addition
// (or fused multiply-add) makes n - 8 of them, exactly.  (The bare bits would be
// the subnormal half n 2^-24, one instruction less, but the products align
// subnormal operands by their exponent field and lose 7 bits of the sum: errors
// of 1e-5 instead of 5e-7 were measured.)  Keys and values are the 16-row
// operand of m16n8k16 products, 8 query rows the other, which is float32 split
// into two halves (hi + lo, 22 bits) and goes through in two products with one
// accumulator.  The scales enter outside the products: a key's in float32 after
// the product over its 32 elements, a value's before it, on the probabilities'
// halves (hi' = hi d, lo' = lo d + the exact rest fma(hi, d, -hi')).  Each tile's
// probabilities are relative to its own maximum, so that what lies beside a key
// with nearly all of the weight keeps its bits.
//
// A work item is a sequence, a KV head and 4 to 32 query rows ((new token, head of
// the KV head's group) pairs); its keys are cut into units, the units of all
// items laid end to end and dealt out evenly over the CTAs, so that lengths
// may differ and a single long sequence fills the device.  Each warp walks its
// own tiles of 32 keys with its own ring of asynchronous copies; the warps of
// a CTA join at the end of an item.  Items cut between CTAs leave partial
// (m, l, o); the CTA that arrives last joins them in the order of their keys.
//
// It is bound by instructions: a tile of 32 keys of 128 elements takes a warp 692 for
// 4 query rows (issue slots 0.57 used, the matrix pipe 19 %).  64 sequences of up to
// 8192 tokens, 32/8 heads of 128, take 117 to 123 us, 0.57 to 0.60 of a plain copy's
// rate for the 455 MB of cache; 512 new tokens on 4096, 32/4 heads of 64: 0.36 of the
// matrix pipe.  Small batches are bound by latency: the share of the work, the page
// table, the copy, the join.
#include <cfloat>

#include "kv_cache.cuh"

namespace glc {
namespace {

constexpr int WK = KV_WK;

struct AttnKv {
  KvPools c;
  KvSeqs s;
  const float* q;
  size_t q_ld;
  float* o;
  size_t o_ld;
  float* lse;
  int group;     // query heads per KV head
  int toks, parts;  // of a tile of query rows: tokens, or tiles of a token
  float scale2;  // log2(e) / sqrt(head_dim)
  float* part;   // [2 * CTAs][RT * (HD + 2)]
  int* count;    // arrivals, by the CTA in which the item starts; zero between calls
  int* err;
  uint32_t k1024, less72;  // pairs of halves: 1024, -72
};

// NQ: query tiles of 8 rows of an item, or 0: one tile of 4 rows, whose hi and lo
// are its 8 columns; W: warps.
template <int HD, int NQ, int W>
struct Shape {
  using Tile = KvTile<HD>;
  static constexpr int NB = Tile::NB;
  static constexpr int RT = NQ ? 8 * NQ : 4;  // query rows of an item
  static constexpr int STAGES = HD >= 96 ? 2 : 3;
  static constexpr int PER_SM = kv_per_sm(HD, NQ, W);
  static constexpr int SCALES = WK * NB * 6;  // a tile's scales as the products take them
  static constexpr int WARP = STAGES * Tile::BYTES + SCALES;
  static constexpr int QUERIES = NQ ? NQ * NB * 1024 : NB * 512;  // the queries as operands
  static constexpr int JOIN = W * RT * (HD + 2) * 4;  // the warps' (o, m, l), in the place of all this
  static constexpr int SMEM = QUERIES + W * WARP > JOIN ? QUERIES + W * WARP : JOIN;
  static_assert(WARP % 16 == 0, "rings start on 16 bytes");
};

// 16 bytes, `size` of them from src and zeros after
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// d = a b + c
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, const float* c) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Pairs of halves as 32-bit words throughout.
__device__ __forceinline__ uint32_t add2(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}
__device__ __forceinline__ uint32_t mul2(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}
__device__ __forceinline__ uint32_t fma2(uint32_t x, uint32_t y, uint32_t w) {
  uint32_t z;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(z) : "r"(x), "r"(y), "r"(w));
  return z;
}
__device__ __forceinline__ uint32_t neg2(uint32_t x) {
  uint32_t z;
  asm("neg.f16x2 %0, %1;" : "=r"(z) : "r"(x));
  return z;
}
// (x0, x1) as halves hi + lo: 22 bits where lo is a normal half
__device__ __forceinline__ void split2(float x0, float x1, uint32_t* hi, uint32_t* lo) {
  float f0, f1;
  asm("{\n\t.reg .b16 a, b;\n\t"
      "cvt.rn.f16x2.f32 %0, %4, %3;\n\t"
      "mov.b32 {a, b}, %0;\n\t"
      "cvt.f32.f16 %1, a;\n\t"
      "cvt.f32.f16 %2, b;\n\t}"
      : "=r"(*hi), "=f"(f0), "=f"(f1)
      : "f"(x0), "f"(x1));
  asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(*lo) : "f"(x0 - f0), "f"(x1 - f1));
}
// Codes less 8 of the low nibbles of x's halves, and of the next ones.  The
// constants that an instruction has no second immediate for are kernel
// parameters, so that they stay in registers.
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t mask, uint32_t y) {
  uint32_t z;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(z) : "r"(x), "r"(mask), "r"(y));  // (x & mask) | y
  return z;
}
__device__ __forceinline__ float half_float(uint32_t x) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(x)));
}
// N halves of shared memory, in pairs
template <int N>
__device__ __forceinline__ void load_halves(uint32_t at, uint32_t* x) {
  if constexpr (N == 4) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at));
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x[0]) : "r"(at));
  } else {
#pragma unroll
    for (int i = 0; i < (N + 1) / 2; ++i) {
      unsigned short a, b = 0;
      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(a) : "r"(at + 4 * i));
      if (2 * i + 1 < N) asm volatile("ld.shared.b16 %0, [%1];" : "=h"(b) : "r"(at + 4 * i + 2));
      x[i] = a | static_cast<uint32_t>(b) << 16;
    }
  }
}
struct Unpack {
  uint32_t k1024, less72;
  __device__ __forceinline__ uint32_t low(uint32_t x) const {
    return add2(masked_or(x, 0x000f000fu, k1024), 0xe408e408u);  // - 1032
  }
  __device__ __forceinline__ uint32_t next(uint32_t x) const {
    return fma2(masked_or(x, 0x00f000f0u, k1024), 0x2c002c00u, less72);  // / 16 - 72
  }
};

__device__ __forceinline__ int arrive(int* count) {
  int before;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
  return before;
}
// (M, L, o) += the part (m, l, y)
__device__ __forceinline__ void add_part(float m, float l, float4 y, float* M, float* L, float4* o) {
  const float now = fmaxf(*M, m), ns = now == -INFINITY ? 0.f : now;
  const float old = exp2_fast(*M - ns), by = exp2_fast(m - ns);
  *M = now;
  *L = fmaf(l, by, *L * old);
  o->x = fmaf(y.x, by, o->x * old);
  o->y = fmaf(y.y, by, o->y * old);
  o->z = fmaf(y.z, by, o->z * old);
  o->w = fmaf(y.w, by, o->w * old);
}

template <int HD, int NQ, int W>
__global__ void __launch_bounds__(W * 32, Shape<HD, NQ, W>::PER_SM) attention_kv_kernel(const AttnKv a) {
  GLC_PDL_ENTRY();
  using S = Shape<HD, NQ, W>;
  using Tile = KvTile<HD>;
  constexpr int NB = S::NB, RT = S::RT, STAGES = S::STAGES, UNIT = W * WK;
  constexpr bool PAIRED = NQ == 0;        // columns 2r and 2r + 1 are hi and lo of row r
  constexpr int TILES = NQ ? NQ : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ KvPlace place;
  __shared__ int sum_s[2][W];
  __shared__ int last_s;
  __shared__ __align__(16) float rs_s[RT];  // what a row's products are short of its scores
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // ---- the share of this CTA: thread i counts the units of its run of
  // sequences, a scan over the threads finds the run that the share begins in; of
  // up to 32 sequences each warp counts by itself, without barriers
  {
    if (tid == 0) place.b = -1;
    const bool few = a.s.seqs <= 32;
    const int me = few ? lane : tid;
    const int run = a.s.seqs <= W * 32 ? 1 : (a.s.seqs + W * 32 - 1) / (W * 32);
    const int b0 = me * run < a.s.seqs ? me * run : a.s.seqs;
    const int b1 = b0 + run < a.s.seqs ? b0 + run : a.s.seqs;
    KvRows w = {};
    if (b0 < b1) w = kv_rows(a.s, a.c.page, a.toks, a.parts, b0, a.err);
    // pieces of `per` units of the run, those of all before it, and of all
    int calls = 0;
    bool bad = false;  // starts that do not ascend: nothing is done
    auto count = [&](int per, int* mine, int* before, int* total) {
      int y = 0;
      for (int b = b0; b < b1; ++b) {
        if (run > 1) w = kv_rows(a.s, a.c.page, a.toks, a.parts, b, a.err);
        bad |= w.bad;
        y += kv_head_pieces(w, UNIT, per) * a.c.kv_heads;
      }
      int upto = y;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, upto, o);
        if (lane >= o) upto += v;
      }
      *mine = y;
      *before = upto - y;
      if (few) {
        *total = __shfl_sync(~0u, upto, 31);
        bad = __any_sync(~0u, bad);
        return;
      }
      int* sums = sum_s[calls++ & 1];
      if (lane == 31) sums[warp] = upto;
      bad = __syncthreads_or(bad);
      *total = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if (i < warp) *before += sums[i];
        *total += sums[i];
      }
    };
    int mine, before, total;
    count(1, &mine, &before, &total);
    if (bad) return;  // the same for the whole CTA, and for all of them
    const int ctas = total < static_cast<int>(gridDim.x) ? total : static_cast<int>(gridDim.x);
    if (static_cast<int>(blockIdx.x) >= ctas) return;
    // one piece of one item for each CTA, where pieces come out even enough
    const int least = (total + ctas - 1) / ctas;
    int per = 1, alone = 0, begin = kv_cta_begin(blockIdx.x, total, ctas);
    for (int i = least; i <= kv_most_per(least); i += least < 16 ? 1 : least / 16) {
      int m, f, pieces;
      count(i, &m, &f, &pieces);
      if (pieces <= static_cast<int>(gridDim.x)) {
        if (static_cast<int>(blockIdx.x) >= pieces) return;
        per = i, alone = 1, begin = blockIdx.x, mine = m, before = f;
        break;
      }
    }
    if (few && warp) mine = 0;  // the first warp says
    __syncwarp();               // (place.b is -1)
    if (before <= begin && begin < before + mine) {
      place.total = total;
      place.ctas = ctas;
      for (int b = b0; b < b1; ++b) {
        if (run > 1) w = kv_rows(a.s, a.c.page, a.toks, a.parts, b, a.err);
        const int y = kv_head_pieces(w, UNIT, per) * a.c.kv_heads;
        if (begin < before + y) {
          kv_place(&place, w, b, UNIT, per, alone, blockIdx.x, begin - before, before);
          break;
        }
        before += y;
      }
    }
    __syncthreads();
    if (place.b < 0) return;  // not reached, were the lengths left alone meanwhile
  }

  uint4* queries = reinterpret_cast<uint4*>(smem);  // [query tile][block][half of it][lane]: hi, hi, lo, lo; paired: [block][lane]: the halves' column
  uint8_t* ring = smem + S::QUERIES + warp * S::WARP;
  float* kscale = reinterpret_cast<float*>(ring + STAGES * Tile::BYTES);                   // [block][key % 8][key / 8]
  __half* vscale = reinterpret_cast<__half*>(ring + STAGES * Tile::BYTES + WK * NB * 4);  // [block][pair % 4][key / 8][2]
  const uint32_t ring_u = smem_u32(ring);
  const int page16 = a.c.page >> 4;
  const uint32_t page_bytes = static_cast<uint32_t>(a.c.chunk * a.c.kv_heads);
  // 8 lanes each copy a side of a group of 16 tokens of a tile
  const int lane8 = lane & 7, side = lane >> 4, grp = (lane >> 3) & 1;
  const uint32_t codes_to = ring_u + Tile::codes_of(side, grp), scales_to = ring_u + Tile::scales_of(side, grp) + lane8 * 16;
  uint32_t swizzled[4];  // piece lane8 as the pieces lane8 + 8 j of the group's codes are swizzled
#pragma unroll
  for (int j = 0; j < 4; ++j) swizzled[j] = codes_to + ((lane8 * 16) ^ Tile::swizzle(j));
  // a warp's tiles lie UNIT keys apart
  const uint32_t scales_from = a.c.scales_at;
  const int step_pages = (UNIT / 16) / page16, step_slot = (UNIT / 16) % page16;

  const Unpack unpack{a.k1024, a.less72};
  for (;;) {
    // ---- one item, or the part of it that lies in this share
    int key0, key1, edge_key, rows, width, tok0, head0;
    const int* table;
    const uint8_t* head;  // piece lane8 of the item's head in page 0 of the lane's side
    {
      const KvPlace& p = place;
      const int run_at = p.w.parts == 1 ? p.tile : p.tile / p.w.parts, part_at = p.tile - run_at * p.w.parts;
      const int seg_end = p.item_at + p.units < p.end ? p.item_at + p.units : p.end;
      key0 = (p.at - p.item_at) * UNIT;
      key1 = (seg_end - p.item_at) * UNIT;
      const int keys = kv_run_keys(p.w, run_at);
      if (key1 > keys) key1 = keys;
      table = a.s.table + static_cast<size_t>(p.b) * a.s.max_pages;
      head = (side ? a.c.v : a.c.k) + static_cast<size_t>(p.h) * a.c.chunk + lane8 * 16;
      // the tile's first token and head, and its rows (those past the last repeat
      // row 0 and are not written)
      tok0 = run_at * p.w.toks, head0 = part_at * RT;
      width = a.group < RT ? a.group : a.group - head0 < RT ? a.group - head0 : RT;  // heads of a token
      rows = (p.w.n - tok0 < p.w.toks ? p.w.n - tok0 : p.w.toks) * width;
      edge_key = p.w.len - p.w.n + tok0;  // the last key that all rows see
    }
    // the last key that row r sees
    auto row_last = [&](int r) { return edge_key + (r < rows ? r : 0) / width; };

    // the queries' values are on their way while the table's are looked up
    static_assert(TILES <= W, "a warp per query tile");
    float x[NB][8];
    if (warp < TILES) {
      const int mine = PAIRED ? g >> 1 : 8 * warp + g, r = mine < rows ? mine : 0, token = tok0 + r / width, hh = head0 + r % width;
      const float* qp =
          a.q + static_cast<size_t>(place.w.first + token) * a.q_ld + static_cast<size_t>(place.h * a.group + hh) * HD;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float4 u = *reinterpret_cast<const float4*>(qp + 32 * i + 8 * t);
        const float4 v = *reinterpret_cast<const float4*>(qp + 32 * i + 8 * t + 4);
        x[i][0] = u.x, x[i][1] = u.y, x[i][2] = u.z, x[i][3] = u.w;
        x[i][4] = v.x, x[i][5] = v.y, x[i][6] = v.z, x[i][7] = v.w;
      }
    }
    // The lane's group of 16 tokens in the warp's next tile: its page (-1: none), and
    // where its codes and scales are in that.  An index that is no page is noted, and
    // said at the end.
    int next = key0 + warp * WK;
    KvWalk walk;
    walk.start(next + 16 * grp, page16);
    bool bad = false;
    auto table_page = [&] {
      int p = -1;
      if (next + 16 * grp < key1) {
        p = table[walk.index];
        bad |= static_cast<unsigned>(p) >= static_cast<unsigned>(a.c.num_pages);
      }
      return static_cast<unsigned>(p) < static_cast<unsigned>(a.c.num_pages) ? p : -1;
    };
    int page = table_page();

    // copies the tile at `next` to the stage at `to` and looks the following one's
    // page up.  A group has whole pages of 16 slots, so the slots behind the last key
    // are copied too: their codes are numbers, their scales are not used.
    uint32_t to = 0;
    auto fetch = [&] {
      if (next < key1) {
        const uint8_t* from = head + static_cast<uint64_t>(page < 0 ? 0 : page) * page_bytes;
        const uint8_t* codes = from + static_cast<uint32_t>(walk.slot) * (16 * Tile::ROW);
        const uint8_t* scales = from + (static_cast<uint32_t>(walk.slot) * (32 * NB) + scales_from);
        const int size = page < 0 ? 0 : 16;  // 0: zeros are stored, nothing is read
#pragma unroll
        for (int j = 0; j < Tile::LANE_PIECES; ++j) copy16(swizzled[j & 3] + to + 128 * j, codes + 128 * j, size);
        if (lane8 < Tile::GROUP_SCALES) copy16(scales_to + to, scales, size);
        to = to == (STAGES - 1) * Tile::BYTES ? 0 : to + Tile::BYTES;
        next += UNIT;
        walk.advance(step_pages, step_slot, page16);
        page = table_page();
      }
      copies_close();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch();

    // ---- the queries as operands, a tile of 8 rows per warp: lane (g, t) has
    // elements 8t .. 8t + 7 of each block of row g, in the order in which the codes
    // of 8 elements come apart: (0,4), (1,5); (2,6), (3,7)
    if (warp < TILES) {
      const int n = warp;
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i][j]));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      // the row's largest magnitude goes to [2^13, 2^14)
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = e < -100 ? -100 : e > 126 ? 126 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
      if (t == 0) rs_s[PAIRED ? g >> 1 : 8 * n + g] = a.scale2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * 0.0001220703125f;  // 2^(e - 13)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] *= up;
        uint4 q[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          split2(x[i][2 * j], x[i][2 * j + 4], &q[j].x, &q[j].z);
          split2(x[i][2 * j + 1], x[i][2 * j + 5], &q[j].y, &q[j].w);
          if (!PAIRED) queries[((n * NB + i) * 2 + j) * 32 + lane] = q[j];
        }
        if (PAIRED)
          queries[i * 32 + lane] = g & 1 ? make_uint4(q[0].z, q[0].w, q[1].z, q[1].w) : make_uint4(q[0].x, q[0].y, q[1].x, q[1].y);
      }
    }
    __syncthreads();
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};

    // rows: elements 4g + e of a block, columns: queries; [..][j][0..1] is e = 2j, [2..3] e = 2j + 1
    float acc[TILES][NB][2][4];
    constexpr float NONE = -FLT_MAX;  // the maximum of no score: differences of two are numbers
    float m[TILES][2], l[TILES][2];  // of queries 8n + 2t and 8n + 2t + 1; paired: [0][0], of query t
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      m[n][0] = m[n][1] = NONE;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[n][i][j][x] = 0.f;
    }
    // A tile's probabilities are taken relative to its own largest score and held at
    // 2^pexp times their size, value scales at 2^vexp times theirs: products stay below
    // 2^15, and hi and lo are normal halves for all probabilities down to 2^-15 of the
    // tile's largest (2^4 times, relative to the running maximum, gave errors of 3e-5 in
    // keys beside one that has nearly all of the weight and a small value).  The tile's
    // sum is then added at 2^(its maximum - m - pexp).  m is raised only when a score
    // passes it by more than 2^SLACK, so that the sums are seldom rescaled.
    constexpr float SLACK = 4.f;
    float pexp = 12.f;
    int vexp = 0;
    uint32_t vtop = 0;  // largest scale (bits) that they allow
    uint32_t up = 0x3c003c00u;  // 2^vexp, in pairs of halves

    uint32_t stage = 0;  // bytes
    for (int key = key0 + warp * WK; key < key1; key += UNIT) {
      copies_wait<STAGES - 2>();
      __syncwarp();  // the tile is there for all lanes, and all are done with the last one's stage
      fetch();
      const uint32_t from = ring_u + stage;
      bool odd_scale;  // some value scale is infinite or not a number
      {
        // lane = key: its scales, zero behind the last key
        const uint32_t at = from + 2 * Tile::CODES + lane * (2 * NB);
        uint32_t kd[(NB + 1) / 2], vd[(NB + 1) / 2];  // pairs of blocks
        load_halves<NB>(at, kd);
        load_halves<NB>(at + Tile::SCALES, vd);
        if (key + WK > key1 && key + lane >= key1) {
#pragma unroll
          for (int i = 0; i < (NB + 1) / 2; ++i) kd[i] = vd[i] = 0;
        }
        uint32_t big = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          kscale[(i * 8 + lane8) * 4 + (lane >> 3)] = half_float(i & 1 ? kd[i / 2] >> 16 : kd[i / 2]);
          const uint32_t mag = (i & 1 ? vd[i / 2] >> 16 : vd[i / 2]) & 0x7fffu;
          big = big > mag ? big : mag;
        }
        big = __reduce_max_sync(~0u, big);
        odd_scale = big > 0x7bffu;
        if (odd_scale) {  // (the finite ones' sizes count)
          big = 0;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const uint32_t mag = (i & 1 ? vd[i / 2] >> 16 : vd[i / 2]) & 0x7fffu;
            if (mag <= 0x7bffu) big = big > mag ? big : mag;
          }
          big = __reduce_max_sync(~0u, big);
        }
        if (big > vtop) {  // the same for the whole warp
          // the largest scale to [1, 2): room for scales four times as large.  Scales made
          // larger lose nothing; made smaller, by 2^-6 at most, those below 2^-8 lose bits,
          // so beyond that the probabilities make way: to 2^3 for the largest scales.
          const int e = big < 0x400u ? -15 : static_cast<int>(big >> 10) - 15;
          const int now = e > 6 ? -6 : -e;
          pexp = static_cast<float>(12 - (e + now));
          const float by = vtop ? __uint_as_float(static_cast<uint32_t>(127 + now - vexp) << 23) : 0.f;
#pragma unroll
          for (int n = 0; n < TILES; ++n)
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[n][i][j][x] *= by;
          vexp = now;
          vtop = e + 3 > 15 ? 0x7fffu : (static_cast<uint32_t>(e + 3 + 15) << 10) - 1;
          up = static_cast<uint32_t>(15 + vexp) * 0x04000400u;
        }
#pragma unroll
        for (int i = 0; i < (NB + 1) / 2; ++i) {
          const uint32_t d = mul2(vd[i], up);
          __half* to = vscale + (((lane >> 1) & 3) * 4 + (lane >> 3)) * 2 + (lane & 1);
          to[(2 * i) * 32] = __ushort_as_half(static_cast<unsigned short>(d));
          if (2 * i + 1 < NB) to[(2 * i + 1) * 32] = __ushort_as_half(static_cast<unsigned short>(d >> 16));
        }
      }
      __syncwarp();

      // ---- s of keys 16 j + g (x = 0, 1: queries 2t, 2t + 1) and 16 j + 8 + g (x = 2, 3);
      // paired: x = 0 and 1, of query t
      float s[TILES][2][4];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        uint32_t kw[4];  // codes of elements 8t .. 8t + 7 of the block, keys 8x + g
        ldsm4(kw, from + Tile::code_at(lane, i));
        const float4 d = *reinterpret_cast<const float4*>(kscale + (i * 8 + g) * 4);
        uint32_t ka[2][8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t x = kw[2 * j], y = kw[2 * j + 1], xs = x >> 8, ys = y >> 8;
          ka[j][0] = unpack.low(x), ka[j][1] = unpack.low(y), ka[j][2] = unpack.next(x), ka[j][3] = unpack.next(y);
          ka[j][4] = unpack.low(xs), ka[j][5] = unpack.low(ys), ka[j][6] = unpack.next(xs), ka[j][7] = unpack.next(ys);
        }
        if constexpr (PAIRED) {
          const uint4 q = queries[i * 32 + lane];
          float c[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) mma16816(c[j], ka[j][0], ka[j][1], ka[j][2], ka[j][3], q.x, q.y, zero);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma16816(c[j], ka[j][4], ka[j][5], ka[j][6], ka[j][7], q.z, q.w, c[j]);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const float dd = j ? (z ? d.w : d.z) : (z ? d.y : d.x), y = c[j][2 * z] + c[j][2 * z + 1];
              s[0][j][z] = i ? fmaf(dd, y, s[0][j][z]) : dd * y;
            }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const uint4 q0 = queries[((n * NB + i) * 2) * 32 + lane], q1 = queries[((n * NB + i) * 2 + 1) * 32 + lane];
          float c[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) mma16816(c[j], ka[j][0], ka[j][1], ka[j][2], ka[j][3], q0.x, q0.y, zero);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma16816(c[j], ka[j][4], ka[j][5], ka[j][6], ka[j][7], q1.x, q1.y, c[j]);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma16816(c[j], ka[j][0], ka[j][1], ka[j][2], ka[j][3], q0.z, q0.w, c[j]);
#pragma unroll
          for (int j = 0; j < 2; ++j) mma16816(c[j], ka[j][4], ka[j][5], ka[j][6], ka[j][7], q1.z, q1.w, c[j]);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float dd = j ? (z < 2 ? d.z : d.w) : (z < 2 ? d.x : d.y);
              s[n][j][z] = i ? fmaf(dd, c[j][z], s[n][j][z]) : dd * c[j][z];
            }
        }
      }

      // ---- the running softmax of queries 8n + 2t and 8n + 2t + 1
      const bool edge = key + WK > key1 || key + WK - 1 > edge_key;
      // probabilities as halves, turned so that lane (g, t) has column g and keys 2t, 2t + 1 of each 8
      uint32_t hi[TILES][4], lo[TILES][4];
      float by_tile[TILES][2];  // what the tile's sums count
      uint32_t own[4];  // paired: what the lane's column is, hi or lo; hi is 0 where it is hi
      if constexpr (PAIRED) {
        const float rs = rs_s[t];
        if (edge) {
          __syncwarp();  // (a branch, not selects)
          const int last = row_last(t);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int k = key + 16 * j + 8 * z + g;
              if (k > last || k >= key1) s[0][j][z] = -INFINITY;
            }
        }
        float top = fmaxf(fmaxf(s[0][0][0], s[0][0][1]), fmaxf(s[0][1][0], s[0][1][1]));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
        top = fmaxf(top, __shfl_xor_sync(~0u, top, 16)) * rs;
        if (__any_sync(~0u, top > m[0][0] + SLACK)) {
          const float now = fmaxf(m[0][0], top), by = exp2_fast(m[0][0] - now);
          m[0][0] = now;
          l[0][0] *= by;
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[0][i][j][x] *= by;
        }
        const float ts = fmaxf(top - pexp, NONE);
        by_tile[0][0] = exp2_fast(ts - m[0][0]);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p = exp2_fast(fmaf(s[0][j][i], rs, -ts));
            sum += p;
            uint32_t ph, pl;
            split2(p, p, &ph, &pl);
            ph = transposed(ph);
            pl = transposed(pl);
            own[2 * j + i] = g & 1 ? pl : ph;
            hi[0][2 * j + i] = g & 1 ? ph : 0u;
          }
        l[0][0] = fmaf(sum, by_tile[0][0], l[0][0]);
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float2 rs = *reinterpret_cast<const float2*>(rs_s + 8 * n + 2 * t);
        if (edge) {
          __syncwarp();  // (a branch, not selects)
          const int last0 = row_last(8 * n + 2 * t), last1 = row_last(8 * n + 2 * t + 1);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const int k = key + 16 * j + (z >> 1) * 8 + g;
              if (k > (z & 1 ? last1 : last0) || k >= key1) s[n][j][z] = -INFINITY;
            }
        }
        float top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[i] = fmaxf(fmaxf(s[n][0][i], s[n][0][i + 2]), fmaxf(s[n][1][i], s[n][1][i + 2]));
          top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 4));
          top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 8));
          top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 16)) * (i ? rs.y : rs.x);
        }
        if (__any_sync(~0u, top[0] > m[n][0] + SLACK || top[1] > m[n][1] + SLACK)) {
          float by[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float now = fmaxf(m[n][i], top[i]);
            by[i] = exp2_fast(m[n][i] - now);
            m[n][i] = now;
            l[n][i] *= by[i];
          }
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[n][i][j][x] *= by[x & 1];
        }
        float ts[2], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ts[i] = fmaxf(top[i] - pexp, NONE);
          by_tile[n][i] = exp2_fast(ts[i] - m[n][i]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = exp2_fast(fmaf(s[n][j][2 * i], rs.x, -ts[0]));
            const float p1 = exp2_fast(fmaf(s[n][j][2 * i + 1], rs.y, -ts[1]));
            sum[0] += p0;
            sum[1] += p1;
            uint32_t ph, pl;
            split2(p0, p1, &ph, &pl);
            hi[n][2 * j + i] = transposed(ph);
            lo[n][2 * j + i] = transposed(pl);
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) l[n][i] = fmaf(sum[i], by_tile[n][i], l[n][i]);
      }
      const bool fix = odd_scale && edge;

      // ---- o: a tile's sum from zero, then added.  (The products cut their sums
      // off, each by up to 2^-24 of what is there: a long row summed in them alone
      // came out 2e-6 too small after 4096 keys.)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        uint32_t vw[4];  // codes of elements 4g .. 4g + 3, keys 8x + 2t and 8x + 2t + 1
        ldsm4t(vw, from + Tile::CODES + Tile::code_at(lane, i));
        const uint4 d4 = *reinterpret_cast<const uint4*>(vscale + (i * 4 + t) * 8);
        const uint32_t dw[4] = {d4.x, d4.y, d4.z, d4.w};
        uint32_t va[2][8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u = vw[2 * j], v = vw[2 * j + 1], us = u >> 8, vs = v >> 8;
          va[j][0] = unpack.low(u), va[j][1] = unpack.next(u), va[j][2] = unpack.low(v), va[j][3] = unpack.next(v);
          va[j][4] = unpack.low(us), va[j][5] = unpack.next(us), va[j][6] = unpack.low(vs), va[j][7] = unpack.next(vs);
        }
        if constexpr (PAIRED) {
          uint32_t p[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) p[x] = fma2(own[x], dw[x], fma2(hi[0][x], dw[x], neg2(mul2(hi[0][x], dw[x]))));
          if (fix) {  // a key that a row does not see counts nothing, whatever its scale is
            const int last = row_last(g >> 1);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int k = key + 8 * x + 2 * t;
              p[x] &= (k <= last ? 0x0000ffffu : 0u) | (k + 1 <= last ? 0xffff0000u : 0u);
            }
          }
          float y[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              mma16816(y[e], va[j][4 * e], va[j][4 * e + 1], va[j][4 * e + 2], va[j][4 * e + 3], p[2 * j], p[2 * j + 1],
                       j ? y[e] : zero);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int z = 0; z < 4; ++z) acc[0][i][e][z] = fmaf(y[e][z], by_tile[0][0], acc[0][i][e][z]);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            ph[x] = mul2(hi[n][x], dw[x]);
            pl[x] = fma2(lo[n][x], dw[x], fma2(hi[n][x], dw[x], neg2(ph[x])));
          }
          if (fix) {  // a key that a row does not see counts nothing, whatever its scale is
            const int last = row_last(8 * n + g);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int k = key + 8 * x + 2 * t;
              const uint32_t keep = (k <= last ? 0x0000ffffu : 0u) | (k + 1 <= last ? 0xffff0000u : 0u);
              ph[x] &= keep;
              pl[x] &= keep;
            }
          }
          float y[2][4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              mma16816(y[e], va[j][4 * e], va[j][4 * e + 1], va[j][4 * e + 2], va[j][4 * e + 3], ph[2 * j], ph[2 * j + 1],
                       j ? y[e] : zero);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              mma16816(y[e], va[j][4 * e], va[j][4 * e + 1], va[j][4 * e + 2], va[j][4 * e + 3], pl[2 * j], pl[2 * j + 1], y[e]);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int z = 0; z < 4; ++z) acc[n][i][e][z] = fmaf(y[e][z], by_tile[n][z & 1], acc[n][i][e][z]);
        }
      }
      stage = stage == (STAGES - 1) * Tile::BYTES ? 0 : stage + Tile::BYTES;
    }
    copies_wait<0>();
    if (bad) kv_bad(a.err);

    // ---- the warps' parts of the segment joined through shared memory
    const float down = __uint_as_float(static_cast<uint32_t>(127 - vexp) << 23);
    __syncthreads();  // the rings are free
    float* jo = reinterpret_cast<float*>(smem) + warp * RT * HD;
    float* jm = reinterpret_cast<float*>(smem) + W * RT * HD;  // [W][RT] m, then l
    if constexpr (PAIRED) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float(*y)[4] = acc[0][i];
        *reinterpret_cast<float4*>(jo + t * HD + 32 * i + 4 * g) = make_float4(
            (y[0][0] + y[0][1]) * down, (y[0][2] + y[0][3]) * down, (y[1][0] + y[1][1]) * down, (y[1][2] + y[1][3]) * down);
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[0][0] += __shfl_xor_sync(~0u, l[0][0], o);
      if (g == 0) {
        jm[warp * RT + t] = m[0][0] == NONE ? -INFINITY : m[0][0];
        jm[W * RT + warp * RT + t] = l[0][0];
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<float4*>(jo + (8 * n + 2 * t + x) * HD + 32 * i + 4 * g) =
              make_float4(acc[n][i][0][x] * down, acc[n][i][0][2 + x] * down, acc[n][i][1][x] * down,
                          acc[n][i][1][2 + x] * down);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][x] += __shfl_xor_sync(~0u, l[n][x], o);
        if (g == 0) {
          jm[warp * RT + 8 * n + 2 * t + x] = m[n][x] == NONE ? -INFINITY : m[n][x];
          jm[W * RT + warp * RT + 8 * n + 2 * t + x] = l[n][x];
        }
      }
    }
    __syncthreads();
    const KvPlace p = place;
    const int item_end = p.item_at + p.units;
    const bool whole = p.at == p.item_at && item_end <= p.end;
    float* part = a.part + static_cast<size_t>(2 * blockIdx.x + (p.at == p.item_at ? 1 : 0)) * RT * (HD + 2);
    auto write = [&](int r, int c4, float M, float L, float4 o) {
      const int tk = p.w.first + tok0 + r / width, hh = p.h * a.group + head0 + r % width;
      const float inv = M == -INFINITY ? 0.f : 1.f / L;
      reinterpret_cast<float4*>(a.o + static_cast<size_t>(tk) * a.o_ld + static_cast<size_t>(hh) * HD)[c4] =
          make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      if (a.lse && c4 == 0)
        a.lse[static_cast<size_t>(tk) * a.c.kv_heads * a.group + hh] =
            M == -INFINITY ? (L == 0.f ? -INFINITY : L) : M * 0.69314718055994531f + logf(L);  // (L: or NaN)
    };
    for (int i = tid; i < RT * HD / 4; i += W * 32) {
      const int r = i / (HD / 4), c4 = i - r * (HD / 4);
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x) M = fmaxf(M, jm[x * RT + r]);
      const float Ms = M == -INFINITY ? 0.f : M;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float by = exp2_fast(jm[x * RT + r] - Ms);
        const float4 y = reinterpret_cast<const float4*>(smem)[(x * RT + r) * (HD / 4) + c4];
        L = fmaf(jm[W * RT + x * RT + r], by, L);
        o.x = fmaf(y.x, by, o.x);
        o.y = fmaf(y.y, by, o.y);
        o.z = fmaf(y.z, by, o.z);
        o.w = fmaf(y.w, by, o.w);
      }
      if (whole) {
        if (r < rows) write(r, c4, M, L, o);
      } else {
        reinterpret_cast<float4*>(part)[i] = o;
        if (c4 == 0) {
          part[RT * HD + r] = M;
          part[RT * HD + RT + r] = L;
        }
      }
    }
    if (!whole) {
      // ---- the last of the item's CTAs to arrive joins the parts
      const int first_cta = kv_first_cta(p), last_cta = kv_last_cta(p);
      __syncthreads();
      if (tid == 0) {
        // releases the CTA's part (its writes are before the barrier) and acquires the others'
        last_s = arrive(a.count + first_cta) == last_cta - first_cta;
        if (last_s) a.count[first_cta] = 0;
      }
      __syncthreads();
      if (last_s) {
        // a thread has PER elements of every part; where there are more threads than
        // elements, groups of them take every GROUPSth part and join in shared memory
        constexpr int ELEMS = RT * HD / 4, GROUPS = ELEMS < W * 32 ? W * 32 / ELEMS : 1;
        constexpr int PER = (ELEMS + W * 32 - 1) / (W * 32);
        const int group = GROUPS > 1 ? tid / ELEMS : 0, i0 = GROUPS > 1 ? tid - group * ELEMS : tid;
        float M[PER], L[PER];
        float4 o[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) M[k] = -INFINITY, L[k] = 0.f, o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (group < GROUPS) {
#pragma unroll(PER > 2 ? 2 : 8 / PER)
          for (int x = first_cta + group; x <= last_cta; x += GROUPS) {
            const float* y = a.part + static_cast<size_t>(2 * x + (x == first_cta ? 1 : 0)) * RT * (HD + 2);
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              const int i = i0 + k * W * 32, r = i / (HD / 4);
              if (i < ELEMS)
                add_part(__ldcg(y + RT * HD + r), __ldcg(y + RT * HD + RT + r), __ldcg(reinterpret_cast<const float4*>(y) + i),
                         &M[k], &L[k], &o[k]);
            }
          }
        }
        if constexpr (GROUPS > 1) {
          float4* so = reinterpret_cast<float4*>(smem);
          float2* sm = reinterpret_cast<float2*>(smem + GROUPS * ELEMS * 16);
          if (group < GROUPS) {
            so[group * ELEMS + i0] = o[0];
            if (i0 % (HD / 4) == 0) sm[group * RT + i0 / (HD / 4)] = make_float2(M[0], L[0]);
          }
          __syncthreads();
          if (group == 0) {
#pragma unroll
            for (int x = 1; x < GROUPS; ++x) {
              const float2 ml = sm[x * RT + i0 / (HD / 4)];
              add_part(ml.x, ml.y, so[x * ELEMS + i0], &M[0], &L[0], &o[0]);
            }
          }
        }
        if (group == 0) {
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const int i = i0 + k * W * 32, r = i / (HD / 4);
            if (i < ELEMS && r < rows) write(r, i - r * (HD / 4), M[k], L[k], o[k]);
          }
        }
      }
    }
    // ---- the next item: the next tile of rows, head, sequence that has any
    if (p.alone || item_end >= p.end) return;
    __syncthreads();  // all have read the place, and the shared memory is the rings again
    if (tid == 0) {
      KvPlace& n = place;
      n.at = n.item_at = item_end;
      if (++n.tile == n.w.tiles) {
        n.tile = 0;
        if (++n.h == a.c.kv_heads) {
          n.h = 0;
          do {  // units remain, so a sequence with rows does (were the lengths left alone meanwhile)
            if (++n.b >= a.s.seqs) {
              n.b = -1;
              break;
            }
            n.w = kv_rows(a.s, a.c.page, a.toks, a.parts, n.b, a.err);
          } while (n.w.tiles == 0);
        }
      }
      if (n.b >= 0) n.units = kv_run_units(n.w, n.tile / n.w.parts, UNIT);
    }
    __syncthreads();
    if (place.b < 0) return;
  }
}

template <int HD, int NQ, int W>
int launch(Context* ctx, const AttnKv& a, cudaStream_t s) {
  using S = Shape<HD, NQ, W>;
  static thread_local int ready = -1;  // device on which the attribute is set
  if (ready != ctx->device) {
    const cudaError_t e =
        cudaFuncSetAttribute(attention_kv_kernel<HD, NQ, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return ctx->fail_cuda(e, "attention_kv: shared memory");
    ready = ctx->device;
  }
  const int ctas = ctx->num_sms * S::PER_SM;
  if (ctas > Context::kKvCounters) return ctx->fail(GLC_ERR_UNSUPPORTED, "attention_kv: more SMs than counters");
  void* ws = nullptr;
  const int rc = ctx->workspace(sizeof(float) * 2 * ctas * S::RT * (HD + 2), &ws);
  if (rc) return rc;
  AttnKv b = a;
  b.part = static_cast<float*>(ws);
  b.toks = a.group < S::RT ? S::RT / a.group : 1;
  b.parts = (a.group + S::RT - 1) / S::RT;
  glc::launch_pdl(ctx, attention_kv_kernel<HD, NQ, W>, dim3(ctas), dim3(W * 32), S::SMEM, s, b);
  GLC_LAUNCH_CHECK(ctx, "attention_kv");
  return GLC_OK;
}

template <int HD>
int launch_for(Context* ctx, const AttnKv& a, cudaStream_t s) {
  const KvVariant v = kv_variant(HD, a.s.rows, a.s.seqs, a.group, a.c.kv_heads, ctx->num_sms);
  if constexpr (HD <= 64) {
    if (v.tiles == 4) return launch<HD, 4, 4>(ctx, a, s);
  } else {
    if (v.tiles == 3) return launch<HD, 3, 4>(ctx, a, s);
  }
  if (v.tiles == 2) return launch<HD, 2, 4>(ctx, a, s);
  if (v.tiles == 0) return v.warps == 4 ? launch<HD, 0, 4>(ctx, a, s) : launch<HD, 0, 16>(ctx, a, s);
  return v.warps == 4 ? launch<HD, 1, 4>(ctx, a, s) : launch<HD, 1, 16>(ctx, a, s);
}

}  // namespace
}  // namespace glc

using glc::Context;

extern "C" int glc_attention_kv(glc_ctx* ctx, const glc_kv_cache* cache, const glc_kv_batch* batch, const float* q,
                                int q_ld, int num_heads, float* o, int o_ld, float* lse) {
  if (!ctx) return GLC_ERR_INVALID;
  Context* c = reinterpret_cast<Context*>(ctx);
  int rc = glc::kv_check(c, "attention_kv", cache, batch);
  if (rc) return rc;
  auto no = [&](const char* why) { return c->fail(GLC_ERR_INVALID, std::string("attention_kv: ") + why); };
  if (!q || !o) return no("q and o must be given");
  if (num_heads <= 0 || num_heads % cache->num_kv_heads) return no("num_heads must be a multiple of num_kv_heads");
  const long long width = static_cast<long long>(num_heads) * cache->head_dim;
  if (q_ld < width || o_ld < width || ((q_ld | o_ld) & 3))
    return no("row strides must be multiples of 4 and at least num_heads * head_dim");
  if (q == o && q_ld != o_ld) return no("o may be q where their strides are equal");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) return no("q and o must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(lse) & 3) return no("lse must be 4-byte aligned");
  const int group = num_heads / cache->num_kv_heads;
  if (static_cast<long long>(batch->num_rows) * group > 0x40000000) return no("too many query rows");
  if (glc::kv_pools(*cache).chunk * cache->num_kv_heads > 0xffffffffu) return no("a page must stay below 4 GB");
  if (glc::kv_most_units(batch->num_rows, batch->num_seqs, group, cache->num_kv_heads, batch->max_pages, cache->page_size) >
      2147483647.0) return no("num_rows, num_kv_heads and max_pages are too large together");
  if (batch->num_rows == 0 || batch->num_seqs == 0) return GLC_OK;
  glc::DeviceScope on(c);
  glc::AttnKv a;
  a.c = glc::kv_pools(*cache);
  a.s = glc::kv_seqs(*batch);
  a.q = q;
  a.q_ld = q_ld;
  a.o = o;
  a.o_ld = o_ld;
  a.lse = lse;
  a.group = group;
  a.scale2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(cache->head_dim)));
  a.part = nullptr;
  a.count = c->kv_count;
  a.err = c->d_err;
  a.k1024 = 0x64006400u;
  a.less72 = 0xd480d480u;
  // the cache's share of the traffic depends on lengths that the host does not have
  glc::ProfScope prof(c, glc::PROF_OTHER, 8.0 * batch->num_rows * width, c->stream);
  switch (cache->head_dim) {
    case 32: return glc::launch_for<32>(c, a, c->stream);
    case 64: return glc::launch_for<64>(c, a, c->stream);
    case 96: return glc::launch_for<96>(c, a, c->stream);
    default: return glc::launch_for<128>(c, a, c->stream);
  }
}
