// Attention of new tokens over the paged 4-bit key/value cache.
//
// For a query row q and the keys k_j = d_j (n_j - 8) it sees (n the 4-bit
// codes, d one scale per 32 elements), the running form of the softmax over
// tiles of keys:
//   s_j = q . k_j * log2(e) / sqrt(hd),  m' = max(m, max s_j),
//   p_j = 2^(s_j - m'),  l = l 2^(m - m') + sum p_j,  o = o 2^(m - m') + sum p_j v_j.
//
// A code of the cache is a whole number below 16, so as the low mantissa bits
// of a half it is exact (n 2^-24; in the next nibble n 2^-20), and one AND
// makes two matrix operands of it: nothing is dequantized.  The other operand
// is float32 split into two halves (hi + lo, 22 bits), which share the 16 rows
// of one m16n8k16 product: rows 0-7 hold hi and rows 8-15 lo of 8 query rows.
// The scales enter in float32: a key's after the product over its 32 elements
// (one product pair per block of 32), a value's before it, on the
// probabilities.  The "- 8" is a constant per query and block (the initial
// value of q . n) and a sum of the scaled probabilities per block of values.
//
// Query rows are (new token, head of the KV head's group), RT = 8 at a time.
// A work item is a sequence, a KV head and such a tile of rows; its keys are
// cut into units, the units of all items laid end to end and dealt out evenly
// to one CTA per SM, so that lengths may differ and a single long sequence
// fills the device.  Items cut between CTAs leave partial (m, l, o); the CTA
// that arrives last joins them in the order of their keys.
#include <cfloat>

#include "kv_cache.cuh"

namespace glc {
namespace {

constexpr int RT = KV_RT, WK = KV_WK;
constexpr int STAGES = 3; // tiles of a warp's ring

struct AttnKv {
  KvPools c;
  KvSeqs s;
  const float* q;
  size_t q_ld;
  float* o;
  size_t o_ld;
  float* lse;
  int group;     // query heads per KV head
  float scale2;  // log2(e) / sqrt(head_dim)
  float* part;   // [2 * CTAs][RT * (HD + 2)]
  int* count;    // arrivals, by the CTA in which the item starts; zero between calls
  int* err;
};

template <int HD>
struct Shape {
  using Tile = KvTile<HD>;
  static constexpr int NB = Tile::NB;
  static constexpr int WARPS = HD >= 96 ? 12 : 16;
  static constexpr int FSCALES = 2 * NB * WK * 4;  // a tile's scales as floats
  static constexpr int RING = WARPS * (STAGES * Tile::BYTES + FSCALES);
  // the warps' (o, m, l) at the end of an item, in the ring's place
  static constexpr int JOIN = WARPS * RT * (HD + 2) * 4;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16 : 0) : "memory");
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
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (x0, x1) as halves hi + lo: 22 bits where lo is a normal half
__device__ __forceinline__ void split2(float x0, float x1, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(x0, x1);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x0 - f.x, x1 - f.y);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = *reinterpret_cast<const uint32_t*>(&l);
}

template <int HD>
__global__ void __launch_bounds__(Shape<HD>::WARPS * 32, 1) attention_kv_kernel(const AttnKv a) {
  GLC_PDL_ENTRY();
  using S = Shape<HD>;
  using Tile = KvTile<HD>;
  constexpr int NB = S::NB, W = S::WARPS, UNIT = W * WK;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long sum_s[W];
  __shared__ long long at_s[2];
  __shared__ int seq_s, last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // ---- the share of this CTA: thread i counts the units of its run of
  // sequences, a scan over the threads finds the run that the share begins in
  if (tid == 0) seq_s = -1;
  const int run = (a.s.seqs + W * 32 - 1) / (W * 32);
  const int b0 = tid * run < a.s.seqs ? tid * run : a.s.seqs;
  const int b1 = b0 + run < a.s.seqs ? b0 + run : a.s.seqs;
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += kv_head_units(kv_rows(a.s, a.c.page, a.group, b, a.err), UNIT) * a.c.kv_heads;
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(~0u, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sum_s[warp] = upto;
  __syncthreads();
  long long total = 0, before = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (i < warp) before += sum_s[i];
    total += sum_s[i];
  }
  upto += before;
  const long long ctas = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= ctas) return;
  const long long begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
  if (upto - mine <= begin && begin < upto) {
    long long at = upto - mine;
    for (int b = b0; b < b1; ++b) {
      const long long u = kv_head_units(kv_rows(a.s, a.c.page, a.group, b, a.err), UNIT) * a.c.kv_heads;
      if (begin < at + u) {
        seq_s = b;
        at_s[0] = at;
        at_s[1] = u;
        break;
      }
      at += u;
    }
  }
  __syncthreads();
  int b = seq_s;
  if (b < 0) return;
  KvRows w = kv_rows(a.s, a.c.page, a.group, b, a.err);
  long long per_head = at_s[1] / a.c.kv_heads;
  int h = static_cast<int>((begin - at_s[0]) / per_head);
  int units = 1;
  long long item_at;  // first unit of the item
  int tile = kv_find_tile(w, UNIT, begin - at_s[0] - h * per_head, &item_at, &units);
  item_at += at_s[0] + h * per_head;

  uint8_t* ring = smem + warp * (STAGES * Tile::BYTES);
  float* fsc = reinterpret_cast<float*>(smem + W * STAGES * Tile::BYTES + warp * S::FSCALES);
  const uint32_t ring_u = smem_u32(ring);
  const int page16 = a.c.page >> 4;
  // a warp's tiles lie UNIT keys apart
  const int step_pages = (UNIT / 16) / page16, step_slot = (UNIT / 16) % page16;

  for (long long at = begin; at < end;) {
    // ---- one item, or the part of it that lies in this share
    const long long item_end = item_at + units;
    const long long seg_end = item_end < end ? item_end : end;
    const int run_at = tile / w.parts, part_at = tile - run_at * w.parts;
    const int keys = kv_run_keys(w, run_at);
    const int key0 = static_cast<int>(at - item_at) * UNIT;
    int key1 = static_cast<int>(seg_end - item_at) * UNIT;
    if (key1 > keys) key1 = keys;

    // the tile's first token and head, its rows, and this thread's row g (the
    // rows past the last repeat row 0 and are not written)
    const int tok0 = run_at * w.toks, head0 = part_at * RT;
    const int width = a.group < RT ? a.group : a.group - head0 < RT ? a.group - head0 : RT;  // heads of a token
    const int rows = (w.n - tok0 < w.toks ? w.n - tok0 : w.toks) * width;
    const int my_row = g < rows ? g : 0, my_tok = tok0 + my_row / width, my_head = head0 + my_row % width;
    const int last_key = w.len - w.n + my_tok;  // the last key this row sees
    const float* qp =
        a.q + static_cast<size_t>(w.first + my_tok) * a.q_ld + static_cast<size_t>(h * a.group + my_head) * HD;
    uint32_t qf[NB][2][4];
    float base[NB][2];  // -8 times the sum of q over a block, of hi and of lo
    float rs;           // what a product is short of s: the row's power of two, units of the codes, scale2
    {
      float x[NB][8], top = 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float4 u = *reinterpret_cast<const float4*>(qp + 32 * i + 8 * t);
        const float4 v = *reinterpret_cast<const float4*>(qp + 32 * i + 8 * t + 4);
        x[i][0] = u.x, x[i][1] = u.y, x[i][2] = u.z, x[i][3] = u.w;
        x[i][4] = v.x, x[i][5] = v.y, x[i][6] = v.z, x[i][7] = v.w;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[i][j]));
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      // the row's largest magnitude goes to [2^13, 2^14); subnormal rows stay as they are
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = e < -100 ? -100 : e > 126 ? 126 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
      rs = a.scale2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * 2048.f;  // 2^(e - 13 + 24)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        // code pairs (0,4), (2,6) of 8 count n 2^-24, pairs (1,5), (3,7) n 2^-20
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] *= up * (j & 1 ? 0.0625f : 1.f);
        split2(x[i][0], x[i][4], &qf[i][0][0], &qf[i][0][1]);
        split2(x[i][1], x[i][5], &qf[i][0][2], &qf[i][0][3]);
        split2(x[i][2], x[i][6], &qf[i][1][0], &qf[i][1][1]);
        split2(x[i][3], x[i][7], &qf[i][1][2], &qf[i][1][3]);
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma16816(d, qf[i][0], 0x80088008u, 0x80808080u);
        mma16816(d, qf[i][1], 0x80088008u, 0x80808080u);
        base[i][0] = d[0];
        base[i][1] = d[2];
      }
    }

    float acc[NB][4][4];
    float vsum[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      vsum[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    // probabilities times value scales are held at 2^vexp times their size, so
    // that the largest lies in the halves' range and lo is a normal half
    int vexp = 0;
    uint32_t vtop = 0;  // largest scale (bits) that vexp allows

    // the two groups of 16 tokens of the warp's next tile, and their pages
    KvWalk walk[2];
    int page[2];
    int next = key0 + warp * WK;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      walk[i].start(next + 16 * i, page16);
      page[i] = next + 16 * i < key1 ? kv_page(a.s, a.c.num_pages, b, walk[i].index, a.err) : -1;
    }
    const size_t head_at = static_cast<size_t>(h) * a.c.chunk;
    const size_t page_bytes = a.c.chunk * a.c.kv_heads;

    // copies the tile at `next` to a stage and looks the following one's pages up
    auto fetch = [&](int stage) {
      if (next < key1) {
        const uint32_t to = ring_u + stage * Tile::BYTES;
        const bool ok0 = page[0] >= 0, ok1 = page[1] >= 0;
        const size_t f0 = (ok0 ? page[0] * page_bytes : 0) + head_at;
        const size_t f1 = (ok1 ? page[1] * page_bytes : 0) + head_at;
#pragma unroll
        for (int j = 0; j < Tile::CODE_PIECES / 32; ++j) {
          int token, from, at;
          Tile::code_piece(lane + 32 * j, &token, &from, &at);
          const bool hi = token >= 16;
          const size_t src =
              (hi ? f1 : f0) + static_cast<size_t>((hi ? walk[1].slot : walk[0].slot) * 16 + (token & 15)) * Tile::ROW + from;
          const bool some = (hi ? ok1 : ok0) && next + token < key1;
          copy16(to + at, a.c.k + src, some);
          copy16(to + Tile::CODES + at, a.c.v + src, some);
        }
        if (lane < Tile::SCALE_PIECES) {
          int side, grp, from, at;
          Tile::scale_piece(lane, &side, &grp, &from, &at);
          const size_t src = (grp ? f1 : f0) + a.c.scales_at +
                             static_cast<size_t>(grp ? walk[1].slot : walk[0].slot) * (32 * NB) + from;
          copy16(to + at, (side ? a.c.v : a.c.k) + src, grp ? ok1 : ok0);
        }
        next += UNIT;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          walk[i].advance(step_pages, step_slot, page16);
          page[i] = next + 16 * i < key1 ? kv_page(a.s, a.c.num_pages, b, walk[i].index, a.err) : -1;
        }
      }
      copies_close();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);

    int stage = 0;
    for (int key = key0 + warp * WK; key < key1; key += UNIT) {
      copies_wait<STAGES - 2>();
      __syncwarp();  // the tile is there for all lanes, and all are done with the last one's stage
      fetch(stage == 0 ? STAGES - 1 : stage - 1);
      const uint32_t from = ring_u + stage * Tile::BYTES;
      {
        // lane = key: its scales as floats, zero behind the last key
        const __half* ks = reinterpret_cast<const __half*>(ring + stage * Tile::BYTES + 2 * Tile::CODES) + lane * NB;
        const __half* vs = ks + WK * NB;
        const bool some = key + lane < key1;
        uint32_t big = 0;
        float kf[NB], vf[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const uint32_t vb = some ? __half_as_ushort(vs[i]) : 0u;
          kf[i] = some ? __half2float(ks[i]) : 0.f;
          vf[i] = __half2float(__ushort_as_half(static_cast<unsigned short>(vb)));
          const uint32_t mag = vb & 0x7fffu;
          big = big > mag ? big : mag;
        }
        big = __reduce_max_sync(~0u, big);
        if (big > vtop) {  // the same for the whole warp
          if (big > 0x7bffu) big = 0x7bffu;
          // the largest scale to [2^12, 2^13): room for scales four times as large
          const int e = big < 0x400u ? -15 : static_cast<int>(big >> 10) - 15;
          const int now = 12 - e;
          const float by = vtop ? __uint_as_float(static_cast<uint32_t>(127 + now - vexp) << 23) : 0.f;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            vsum[i] *= by;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[i][j][x] *= by;
          }
          vexp = now;
          vtop = e + 3 > 15 ? 0x7fffu : (static_cast<uint32_t>(e + 3 + 15) << 10) - 1;
        }
        const float up = __uint_as_float(static_cast<uint32_t>(127 + vexp) << 23);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          fsc[i * WK + lane] = kf[i];
          fsc[(NB + i) * WK + lane] = vf[i] * up;
        }
      }
      __syncwarp();

      // ---- s: tiles of 8 keys; column pair t of tiles 2j and 2j + 1 is keys 16 j + 4 t .. + 3
      float s[4][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) s[2 * j + i][0] = s[2 * j + i][1] = 0.f;
        constexpr int PAIRS = (NB * 2 + 3) / 4;  // ldmatrix x4 per 16 keys
        uint32_t kw[PAIRS][4];
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
          // matrix mi: tile (of 8 keys) and block of 32 elements
          const int mi = p * 4 + (lane >> 3);
          const int tl = mi / NB < 2 ? mi / NB : 0, bl = mi / NB < 2 ? mi % NB : 0;
          const int row = 16 * j + 8 * tl + (lane & 7);
          ldsm4(kw[p], from + Tile::code_at(row, bl));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const float4 d = *reinterpret_cast<const float4*>(fsc + i * WK + 16 * j + 4 * t);
#pragma unroll
          for (int tl = 0; tl < 2; ++tl) {
            const int mi = tl * NB + i;
            const uint32_t x = kw[mi >> 2][mi & 3], y = x >> 8;
            float c[4] = {base[i][0], base[i][0], base[i][1], base[i][1]};
            mma16816(c, qf[i][0], x & 0x000f000fu, x & 0x00f000f0u);
            mma16816(c, qf[i][1], y & 0x000f000fu, y & 0x00f000f0u);
            s[2 * j + tl][0] = fmaf(tl ? d.z : d.x, c[0] + c[2], s[2 * j + tl][0]);
            s[2 * j + tl][1] = fmaf(tl ? d.w : d.y, c[1] + c[3], s[2 * j + tl][1]);
          }
        }
      }

      // ---- the running softmax of row g
      const bool edge = key + WK > key1 || key + WK - 1 > w.len - w.n + tok0;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[i][x] *= rs;
          if (edge) {
            const int k = key + 16 * (i >> 1) + 4 * t + 2 * (i & 1) + x;
            if (k > last_key || k >= key1) s[i][x] = -INFINITY;
          }
          top = fmaxf(top, s[i][x]);
        }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      if (__any_sync(~0u, top > m)) {
        const float now = fmaxf(m, top);
        const float by = now == -INFINITY ? 0.f : exp2_fast(m - now);
        m = now;
        l *= by;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          vsum[i] *= by;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[i][j][x] *= by;
        }
      }
      const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          s[i][x] = exp2_fast(s[i][x] - ms);
          l += s[i][x];
        }

      // ---- o: 16 keys at a time
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
          uint32_t vw[4];
          {
            const int mi = lane >> 3, bl = NB == 1 ? 0 : (i + (mi >> 1) < NB ? i + (mi >> 1) : i);
            const int row = 16 * j + 8 * (mi & 1) + (lane & 7);
            ldsm4t(vw, from + Tile::CODES + Tile::code_at(row, bl));
          }
#pragma unroll
          for (int ii = 0; ii < 2; ++ii) {
            if (i + ii >= NB) break;
            const float4 d = *reinterpret_cast<const float4*>(fsc + (NB + i + ii) * WK + 16 * j + 4 * t);
            float x0 = s[2 * j][0] * d.x, x1 = s[2 * j][1] * d.y;
            float x2 = s[2 * j + 1][0] * d.z, x3 = s[2 * j + 1][1] * d.w;
            if (edge) {  // a key that this row does not see counts nothing, whatever its scale is
              const int k = key + 16 * j + 4 * t;
              if (k > last_key) x0 = 0.f;
              if (k + 1 > last_key) x1 = 0.f;
              if (k + 2 > last_key) x2 = 0.f;
              if (k + 3 > last_key) x3 = 0.f;
            }
            vsum[i + ii] += (x0 + x1) + (x2 + x3);
            uint32_t pf[4];
            split2(x0, x1, &pf[0], &pf[1]);
            split2(x2, x3, &pf[2], &pf[3]);
            const uint32_t u = vw[2 * ii], v = vw[2 * ii + 1], uy = u >> 8, vy = v >> 8;
            mma16816(acc[i + ii][0], pf, u & 0x000f000fu, v & 0x000f000fu);
            mma16816(acc[i + ii][1], pf, u & 0x00f000f0u, v & 0x00f000f0u);
            mma16816(acc[i + ii][2], pf, uy & 0x000f000fu, vy & 0x000f000fu);
            mma16816(acc[i + ii][3], pf, uy & 0x00f000f0u, vy & 0x00f000f0u);
          }
        }
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    copies_wait<0>();

    // ---- the warps' parts of the segment joined through shared memory
    l += __shfl_xor_sync(~0u, l, 1);
    l += __shfl_xor_sync(~0u, l, 2);
    const float down = __uint_as_float(static_cast<uint32_t>(127 - vexp) << 23);
    __syncthreads();  // the ring is free
    float* jo = reinterpret_cast<float*>(smem) + warp * RT * HD;
    float* jm = reinterpret_cast<float*>(smem) + W * RT * HD;  // [W][RT] m, then l
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      vsum[i] += __shfl_xor_sync(~0u, vsum[i], 1);
      vsum[i] += __shfl_xor_sync(~0u, vsum[i], 2);
      // columns 4 (2t) + j and 4 (2t + 1) + j of the block
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float unit = j & 1 ? 1048576.f : 16777216.f;
        x[j] = ((acc[i][j][0] + acc[i][j][2]) * unit - 8.f * vsum[i]) * down;
        x[4 + j] = ((acc[i][j][1] + acc[i][j][3]) * unit - 8.f * vsum[i]) * down;
      }
      float4* to = reinterpret_cast<float4*>(jo + g * HD + 32 * i + 8 * t);
      to[0] = make_float4(x[0], x[1], x[2], x[3]);
      to[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
    if (t == 0) {
      jm[warp * RT + g] = m;
      jm[W * RT + warp * RT + g] = l;
    }
    __syncthreads();
    const bool whole = at == item_at && seg_end == item_end;
    const int first_cta = kv_cta_of(item_at, total, ctas);
    const int last_cta = kv_cta_of(item_end - 1, total, ctas);
    float* part = a.part + static_cast<size_t>(2 * blockIdx.x + (at == item_at ? 1 : 0)) * RT * (HD + 2);
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
        if (r < rows) {
          const int tk = tok0 + r / width, hh = h * a.group + head0 + r % width;
          const float inv = M == -INFINITY ? 0.f : 1.f / L;
          reinterpret_cast<float4*>(a.o + static_cast<size_t>(w.first + tk) * a.o_ld + static_cast<size_t>(hh) * HD)[c4] =
              make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
          if (a.lse && c4 == 0)
            a.lse[static_cast<size_t>(w.first + tk) * a.c.kv_heads * a.group + hh] =
                M == -INFINITY ? -INFINITY : M * 0.69314718055994531f + logf(L);
        }
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
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int need = last_cta - first_cta + 1;
        last_s = atomicAdd(a.count + first_cta, 1) == need - 1;
        if (last_s) a.count[first_cta] = 0;
      }
      __syncthreads();
      if (last_s) {
        __threadfence();
        for (int i = tid; i < RT * HD / 4; i += W * 32) {
          const int r = i / (HD / 4), c4 = i - r * (HD / 4);
          if (r >= rows) continue;
          float M = -INFINITY, L = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int x = first_cta; x <= last_cta; ++x) {
            const float* p = a.part + static_cast<size_t>(2 * x + (x == first_cta ? 1 : 0)) * RT * (HD + 2);
            const float pm = __ldcg(p + RT * HD + r), pl = __ldcg(p + RT * HD + RT + r);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(p) + i);
            const float now = fmaxf(M, pm), ns = now == -INFINITY ? 0.f : now;
            const float old = exp2_fast(M - ns), by = exp2_fast(pm - ns);
            M = now;
            L = fmaf(pl, by, L * old);
            o.x = fmaf(y.x, by, o.x * old);
            o.y = fmaf(y.y, by, o.y * old);
            o.z = fmaf(y.z, by, o.z * old);
            o.w = fmaf(y.w, by, o.w * old);
          }
          const int tk = tok0 + r / width, hh = h * a.group + head0 + r % width;
          const float inv = M == -INFINITY ? 0.f : 1.f / L;
          reinterpret_cast<float4*>(a.o + static_cast<size_t>(w.first + tk) * a.o_ld + static_cast<size_t>(hh) * HD)[c4] =
              make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
          if (a.lse && c4 == 0)
            a.lse[static_cast<size_t>(w.first + tk) * a.c.kv_heads * a.group + hh] =
                M == -INFINITY ? -INFINITY : M * 0.69314718055994531f + logf(L);
        }
      }
    }
    __syncthreads();  // the shared memory is the ring again

    // ---- the next item: the next tile of rows, head, sequence that has any
    at = seg_end;
    if (at < end) {
      item_at = item_end;
      if (++tile == w.tiles) {
        tile = 0;
        if (++h == a.c.kv_heads) {
          h = 0;
          do {  // units remain, so a sequence with rows does (were the lengths left alone meanwhile)
            if (++b >= a.s.seqs) return;
            w = kv_rows(a.s, a.c.page, a.group, b, a.err);
          } while (w.tiles == 0);
        }
      }
      units = kv_run_units(w, tile / w.parts, UNIT);
    }
  }
}

template <int HD>
int launch(Context* ctx, const AttnKv& a, int ctas, cudaStream_t s) {
  static thread_local int ready = -1;  // device on which the attribute is set
  if (ready != ctx->device) {
    const cudaError_t e = cudaFuncSetAttribute(attention_kv_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               Shape<HD>::SMEM);
    if (e != cudaSuccess) return ctx->fail_cuda(e, "attention_kv: shared memory");
    ready = ctx->device;
  }
  glc::launch_pdl(ctx, attention_kv_kernel<HD>, dim3(ctas), dim3(Shape<HD>::WARPS * 32), Shape<HD>::SMEM, s, a);
  GLC_LAUNCH_CHECK(ctx, "attention_kv");
  return GLC_OK;
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
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) return no("q and o must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(lse) & 3) return no("lse must be 4-byte aligned");
  const int group = num_heads / cache->num_kv_heads;
  if (static_cast<long long>(batch->num_rows) * group > 0x40000000) return no("too many query rows");
  if (batch->num_rows == 0 || batch->num_seqs == 0) return GLC_OK;
  glc::DeviceScope on(c);
  const int ctas = c->num_sms;
  const int hd = cache->head_dim;
  void* ws = nullptr;
  rc = c->workspace(sizeof(float) * 2 * ctas * glc::RT * (hd + 2), &ws);
  if (rc) return rc;
  glc::AttnKv a;
  a.c = glc::kv_pools(*cache);
  a.s = glc::kv_seqs(*batch);
  a.q = q;
  a.q_ld = q_ld;
  a.o = o;
  a.o_ld = o_ld;
  a.lse = lse;
  a.group = group;
  a.scale2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(hd)));
  a.part = static_cast<float*>(ws);
  a.count = c->kv_count;
  a.err = c->d_err;
  // the cache's share of the traffic depends on lengths that the host does not have
  glc::ProfScope prof(c, glc::PROF_OTHER, 8.0 * batch->num_rows * width, c->stream);
  switch (hd) {
    case 32: return glc::launch<32>(c, a, ctas, c->stream);
    case 64: return glc::launch<64>(c, a, ctas, c->stream);
    case 96: return glc::launch<96>(c, a, ctas, c->stream);
    default: return glc::launch<128>(c, a, ctas, c->stream);
  }
}
