// Attention of new tokens over the paged 4-bit key/value cache.
//
// For a query row q and the keys k_j = d_j (n_j - 8) it sees (n the 4-bit
// codes, d one scale per 32 elements), the running form of the softmax over
// tiles of keys:
//   s_j = q . k_j * log2(e) / sqrt(hd),  m' = max(m, max s_j),
//   p_j = 2^(s_j - m'),  l = l 2^(m - m') + sum p_j,  o = o 2^(m - m') + sum p_j v_j.
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
// halves (hi' = hi d, lo' = lo d + the exact rest fma(hi, d, -hi')).
//
// A work item is a sequence, a KV head and 8 query rows ((new token, head of
// the KV head's group) pairs); its keys are cut into units, the units of all
// items laid end to end and dealt out evenly over the CTAs, so that lengths
// may differ and a single long sequence fills the device.  Each warp walks its
// own tiles of 32 keys with its own ring of asynchronous copies; the warps of
// a CTA join at the end of an item.  Items cut between CTAs leave partial
// (m, l, o); the CTA that arrives last joins them in the order of their keys.
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
  float scale2;  // log2(e) / sqrt(head_dim)
  float* part;   // [2 * CTAs][RT * (HD + 2)]
  int* count;    // arrivals, by the CTA in which the item starts; zero between calls
  int* err;
};

template <int HD, int W>
struct Shape {
  using Tile = KvTile<HD>;
  static constexpr int NB = Tile::NB;
  static constexpr int RT = 8;  // query rows of an item
  static constexpr int STAGES = HD >= 96 ? 2 : 3;
  static constexpr int PER_SM = 16 / W;  // CTAs: 16 warps of 128 registers
  static constexpr int KS = NB == 3 ? 4 : NB;  // floats of a key's scales
  static constexpr int SCALES = WK * KS * 4 + NB * WK * 2;  // a tile's scales as the products take them
  static constexpr int WARP = STAGES * Tile::BYTES + SCALES;
  static constexpr int JOIN = W * RT * (HD + 2) * 4;  // the warps' (o, m, l), in the rings' place
  static constexpr int SMEM = W * WARP > JOIN ? W * WARP : JOIN;
  static_assert(WARP % 16 == 0, "rings start on 16 bytes");
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
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
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// d = a b + c
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, const float* c) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 halves(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
// (x0, x1) as halves hi + lo: 22 bits where lo is a normal half
__device__ __forceinline__ void split2(float x0, float x1, __half2* hi, __half2* lo) {
  *hi = __floats2half2_rn(x0, x1);
  const float2 f = __half22float2(*hi);
  *lo = __floats2half2_rn(x0 - f.x, x1 - f.y);
}
// codes less 8 of the low nibbles of x's halves, and of the next ones
__device__ __forceinline__ uint32_t codes0(uint32_t x) {
  return bits(__hadd2(halves((x & 0x000f000fu) | 0x64006400u), halves(0xe408e408u)));  // - 1032
}
__device__ __forceinline__ uint32_t codes1(uint32_t x) {
  return bits(__hfma2(halves((x & 0x00f000f0u) | 0x64006400u), halves(0x2c002c00u), halves(0xd480d480u)));  // / 16 - 72
}

template <int HD, int W>
__global__ void __launch_bounds__(W * 32, Shape<HD, W>::PER_SM) attention_kv_kernel(const AttnKv a) {
  GLC_PDL_ENTRY();
  using S = Shape<HD, W>;
  using Tile = KvTile<HD>;
  constexpr int NB = S::NB, RT = S::RT, STAGES = S::STAGES, UNIT = W * WK;
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
  for (int b = b0; b < b1; ++b) mine += kv_head_units(kv_rows(a.s, a.c.page, a.group, RT, b, a.err), UNIT) * a.c.kv_heads;
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
      const long long u = kv_head_units(kv_rows(a.s, a.c.page, a.group, RT, b, a.err), UNIT) * a.c.kv_heads;
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
  KvRows w = kv_rows(a.s, a.c.page, a.group, RT, b, a.err);
  long long per_head = at_s[1] / a.c.kv_heads;
  int h = static_cast<int>((begin - at_s[0]) / per_head);
  int units = 1;
  long long item_at;  // first unit of the item
  int tile = kv_find_tile(w, UNIT, begin - at_s[0] - h * per_head, &item_at, &units);
  item_at += at_s[0] + h * per_head;

  uint8_t* ring = smem + warp * S::WARP;
  float* kscale = reinterpret_cast<float*>(ring + STAGES * Tile::BYTES);            // [key][KS]
  __half* vscale = reinterpret_cast<__half*>(ring + STAGES * Tile::BYTES + WK * S::KS * 4);  // [block][t][8 keys][pair]
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

    // the tile's first token and head, and its rows (those past the last repeat
    // row 0 and are not written)
    const int tok0 = run_at * w.toks, head0 = part_at * RT;
    const int width = a.group < RT ? a.group : a.group - head0 < RT ? a.group - head0 : RT;  // heads of a token
    const int rows = (w.n - tok0 < w.toks ? w.n - tok0 : w.toks) * width;
    auto row_token = [&](int r) { return tok0 + (r < rows ? r : 0) / width; };

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
        const bool full = next + WK <= key1 && ok0 && ok1;
#pragma unroll
        for (int j = 0; j < Tile::CODE_PIECES / 32; ++j) {
          int token, from, at_;
          Tile::code_piece(lane + 32 * j, &token, &from, &at_);
          const bool hi = token >= 16;
          const size_t src =
              (hi ? f1 : f0) + static_cast<size_t>((hi ? walk[1].slot : walk[0].slot) * 16 + (token & 15)) * Tile::ROW + from;
          if (full) {
            copy16(to + at_, a.c.k + src);
            copy16(to + Tile::CODES + at_, a.c.v + src);
          } else {
            const bool some = (hi ? ok1 : ok0) && next + token < key1;
            copy16(to + at_, a.c.k + src, some);
            copy16(to + Tile::CODES + at_, a.c.v + src, some);
          }
        }
        if (lane < Tile::SCALE_PIECES) {
          int side, grp, from, at_;
          Tile::scale_piece(lane, &side, &grp, &from, &at_);
          const size_t src = (grp ? f1 : f0) + a.c.scales_at +
                             static_cast<size_t>(grp ? walk[1].slot : walk[0].slot) * (32 * NB) + from;
          copy16(to + at_, (side ? a.c.v : a.c.k) + src, grp ? ok1 : ok0);
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

    // ---- the queries as operands: lane (g, t) holds elements 8t .. 8t + 7 of
    // each block of row g, and of columns 2t and 2t + 1 what goes by query
    uint32_t qf[NB][2][4];  // per block and half of it: hi, hi, lo, lo
    float rs[2];            // what a product is short of s: the row's power of two and scale2
    int last_key[2];        // the last key the row sees
    {
      const int my_row = g < rows ? g : 0, my_tok = tok0 + my_row / width, my_head = head0 + my_row % width;
      const float* qp =
          a.q + static_cast<size_t>(w.first + my_tok) * a.q_ld + static_cast<size_t>(h * a.group + my_head) * HD;
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
      // the row's largest magnitude goes to [2^13, 2^14)
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
      e = e < -100 ? -100 : e > 126 ? 126 : e;
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - e) << 23);
      const float my_rs = a.scale2 * __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * 0.0001220703125f;  // 2^(e - 13)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        rs[i] = __shfl_sync(~0u, my_rs, 4 * (2 * t + i));
        last_key[i] = w.len - w.n + row_token(2 * t + i);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] *= up;
        // in the order in which the codes of 8 elements come apart: (0,4), (1,5); (2,6), (3,7)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          __half2 h0, l0, h1, l1;
          split2(x[i][2 * j], x[i][2 * j + 4], &h0, &l0);
          split2(x[i][2 * j + 1], x[i][2 * j + 5], &h1, &l1);
          qf[i][j][0] = bits(h0), qf[i][j][1] = bits(h1), qf[i][j][2] = bits(l0), qf[i][j][3] = bits(l1);
        }
      }
    }
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};

    // rows: elements 4g + e of a block, columns: queries; [..][j][0..1] is e = 2j, [2..3] e = 2j + 1
    float acc[NB][2][4];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[i][j][x] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    // probabilities are held at 2^PEXP and value scales at 2^vexp times their
    // size: their products stay below 2^15, and lo and lo' are normal halves
    // where they matter
    constexpr int PEXP = 8;
    int vexp = 0;
    uint32_t vtop = 0;  // largest scale (bits) that vexp allows

    int stage = 0;
    for (int key = key0 + warp * WK; key < key1; key += UNIT) {
      copies_wait<STAGES - 2>();
      __syncwarp();  // the tile is there for all lanes, and all are done with the last one's stage
      fetch(stage == 0 ? STAGES - 1 : stage - 1);
      const uint32_t from = ring_u + stage * Tile::BYTES;
      bool odd_scale;  // some value scale is infinite or not a number
      {
        // lane = key: its scales, zero behind the last key
        const __half* ks = reinterpret_cast<const __half*>(ring + stage * Tile::BYTES + 2 * Tile::CODES) + lane * NB;
        const __half* vs = ks + WK * NB;
        const bool some = key + lane < key1;
        uint32_t big = 0;
        __half vh[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          kscale[lane * S::KS + i] = some ? __half2float(ks[i]) : 0.f;
          vh[i] = some ? vs[i] : __ushort_as_half(0);
          const uint32_t mag = __half_as_ushort(vh[i]) & 0x7fffu;
          big = big > mag ? big : mag;
        }
        big = __reduce_max_sync(~0u, big);
        odd_scale = big > 0x7bffu;
        if (big > vtop) {  // the same for the whole warp
          if (odd_scale) big = 0x7bffu;
          // the largest scale to [2^4, 2^5): room for scales four times as large
          const int e = big < 0x400u ? -15 : static_cast<int>(big >> 10) - 15;
          const int now = 4 - e;
          const float by = vtop ? __uint_as_float(static_cast<uint32_t>(127 + now - vexp) << 23) : 0.f;
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int x = 0; x < 4; ++x) acc[i][j][x] *= by;
          vexp = now;
          vtop = e + 3 > 15 ? 0x7fffu : (static_cast<uint32_t>(e + 3 + 15) << 10) - 1;
        }
        const float up = __uint_as_float(static_cast<uint32_t>(127 + vexp) << 23);
#pragma unroll
        for (int i = 0; i < NB; ++i)
          vscale[((i * 4 + ((lane >> 1) & 3)) * 4 + (lane >> 3)) * 2 + (lane & 1)] =
              __float2half_rn(__half2float(vh[i]) * up);
      }
      __syncwarp();

      // ---- s of keys 16 j + g (x = 0, 1: queries 2t, 2t + 1) and 16 j + 8 + g (x = 2, 3)
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        constexpr int PAIRS = (NB * 2 + 3) / 4;  // ldmatrix x4 per 16 keys: (8 keys, block) matrices
        uint32_t kw[PAIRS][4];
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
          const int mi = p * 4 + (lane >> 3);
          const int tl = mi / NB < 2 ? mi / NB : 0, bl = mi / NB < 2 ? mi % NB : 0;
          ldsm4(kw[p], from + Tile::code_at(16 * j + 8 * tl + (lane & 7), bl));
        }
        float d0[4], d1[4];
        if constexpr (NB >= 3) {
          *reinterpret_cast<float4*>(d0) = *reinterpret_cast<const float4*>(kscale + (16 * j + g) * 4);
          *reinterpret_cast<float4*>(d1) = *reinterpret_cast<const float4*>(kscale + (16 * j + 8 + g) * 4);
        } else if constexpr (NB == 2) {
          *reinterpret_cast<float2*>(d0) = *reinterpret_cast<const float2*>(kscale + (16 * j + g) * 2);
          *reinterpret_cast<float2*>(d1) = *reinterpret_cast<const float2*>(kscale + (16 * j + 8 + g) * 2);
        } else {
          d0[0] = kscale[16 * j + g];
          d1[0] = kscale[16 * j + 8 + g];
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const uint32_t x = kw[i >> 2][i & 3], y = kw[(NB + i) >> 2][(NB + i) & 3], xs = x >> 8, ys = y >> 8;
          const uint32_t a0 = codes0(x), a1 = codes0(y), a2 = codes1(x), a3 = codes1(y);
          const uint32_t e0 = codes0(xs), e1 = codes0(ys), e2 = codes1(xs), e3 = codes1(ys);
          float c[4];
          mma16816(c, a0, a1, a2, a3, qf[i][0][0], qf[i][0][1], zero);
          mma16816(c, a0, a1, a2, a3, qf[i][0][2], qf[i][0][3], c);
          mma16816(c, e0, e1, e2, e3, qf[i][1][0], qf[i][1][1], c);
          mma16816(c, e0, e1, e2, e3, qf[i][1][2], qf[i][1][3], c);
#pragma unroll
          for (int z = 0; z < 4; ++z) s[j][z] = i ? fmaf(z < 2 ? d0[i] : d1[i], c[z], s[j][z]) : (z < 2 ? d0[0] : d1[0]) * c[z];
        }
      }

      // ---- the running softmax of queries 2t and 2t + 1
      const bool edge = key + WK > key1 || key + WK - 1 > w.len - w.n + tok0;
      if (edge) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const int k = key + 16 * j + (z >> 1) * 8 + g;
            if (k > last_key[z & 1] || k >= key1) s[j][z] = -INFINITY;
          }
      }
      float top[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(fmaxf(s[0][i], s[0][i + 2]), fmaxf(s[1][i], s[1][i + 2]));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 4));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 8));
        top[i] = fmaxf(top[i], __shfl_xor_sync(~0u, top[i], 16)) * rs[i];
      }
      if (__any_sync(~0u, top[0] > m[0] || top[1] > m[1])) {
        float by[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float now = fmaxf(m[i], top[i]);
          by[i] = now == -INFINITY ? 0.f : exp2_fast(m[i] - now);
          m[i] = now;
          l[i] *= by[i];
        }
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[i][j][x] *= by[x & 1];
      }
      const float ms[2] = {m[0] == -INFINITY ? 0.f : m[0] - PEXP, m[1] == -INFINITY ? 0.f : m[1] - PEXP};
      // probabilities as halves, turned so that lane (g, t) has query g and keys 2t, 2t + 1 of each 8
      __half2 hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = exp2_fast(fmaf(s[j][2 * i], rs[0], -ms[0]));
          const float p1 = exp2_fast(fmaf(s[j][2 * i + 1], rs[1], -ms[1]));
          l[0] += p0;
          l[1] += p1;
          __half2 ph, pl;
          split2(p0, p1, &ph, &pl);
          hi[2 * j + i] = halves(transposed(bits(ph)));
          lo[2 * j + i] = halves(transposed(bits(pl)));
        }
      uint32_t seen = 0xffu;  // bit 2i + x: key 8i + 2t + x counts for query g
      if (odd_scale && edge) {
        const int last = w.len - w.n + row_token(g);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key + 8 * (i >> 1) + 2 * t + (i & 1) > last) seen &= ~(1u << i);
      }

      // ---- o
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        uint32_t vw[4];  // codes of element pairs, 8 keys each
        ldsm4t(vw, from + Tile::CODES + Tile::code_at(lane, i));
        const uint4 d4 = *reinterpret_cast<const uint4*>(vscale + (i * 4 + t) * 8);
        const uint32_t dw[4] = {d4.x, d4.y, d4.z, d4.w};
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const __half2 d = halves(dw[x]);
          const __half2 big = __hmul2(hi[x], d);
          const __half2 rest = __hfma2(lo[x], d, __hfma2(hi[x], d, __hneg2(big)));
          ph[x] = bits(big);
          pl[x] = bits(rest);
        }
        if (seen != 0xffu) {  // a key that a row does not see counts nothing, whatever its scale is
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t keep = ((seen >> (2 * x)) & 1u ? 0x0000ffffu : 0u) | ((seen >> (2 * x + 1)) & 1u ? 0xffff0000u : 0u);
            ph[x] &= keep;
            pl[x] &= keep;
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u = vw[2 * j], v = vw[2 * j + 1], us = u >> 8, vs = v >> 8;
          const uint32_t a0 = codes0(u), a1 = codes1(u), a2 = codes0(v), a3 = codes1(v);
          mma16816(acc[i][0], a0, a1, a2, a3, ph[2 * j], ph[2 * j + 1], acc[i][0]);
          mma16816(acc[i][0], a0, a1, a2, a3, pl[2 * j], pl[2 * j + 1], acc[i][0]);
          const uint32_t c0 = codes0(us), c1 = codes1(us), c2 = codes0(vs), c3 = codes1(vs);
          mma16816(acc[i][1], c0, c1, c2, c3, ph[2 * j], ph[2 * j + 1], acc[i][1]);
          mma16816(acc[i][1], c0, c1, c2, c3, pl[2 * j], pl[2 * j + 1], acc[i][1]);
        }
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    copies_wait<0>();

    // ---- the warps' parts of the segment joined through shared memory
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[i] += __shfl_xor_sync(~0u, l[i], o);
      l[i] *= 1.f / (1 << PEXP);
    }
    const float down = __uint_as_float(static_cast<uint32_t>(127 - PEXP - vexp) << 23);
    __syncthreads();  // the rings are free
    float* jo = reinterpret_cast<float*>(smem) + warp * RT * HD;
    float* jm = reinterpret_cast<float*>(smem) + W * RT * HD;  // [W][RT] m, then l
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float4*>(jo + (2 * t + x) * HD + 32 * i + 4 * g) =
            make_float4(acc[i][0][x] * down, acc[i][0][2 + x] * down, acc[i][1][x] * down,
                        acc[i][1][2 + x] * down);
    if (g == 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        jm[warp * RT + 2 * t + x] = m[x];
        jm[W * RT + warp * RT + 2 * t + x] = l[x];
      }
    }
    __syncthreads();
    const bool whole = at == item_at && seg_end == item_end;
    float* part = a.part + static_cast<size_t>(2 * blockIdx.x + (at == item_at ? 1 : 0)) * RT * (HD + 2);
    auto write = [&](int r, int c4, float M, float L, float4 o) {
      const int tk = tok0 + r / width, hh = h * a.group + head0 + r % width;
      const float inv = M == -INFINITY ? 0.f : 1.f / L;
      reinterpret_cast<float4*>(a.o + static_cast<size_t>(w.first + tk) * a.o_ld + static_cast<size_t>(hh) * HD)[c4] =
          make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      if (a.lse && c4 == 0)
        a.lse[static_cast<size_t>(w.first + tk) * a.c.kv_heads * a.group + hh] =
            M == -INFINITY ? -INFINITY : M * 0.69314718055994531f + logf(L);
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
      const int first_cta = kv_cta_of(item_at, total, ctas), last_cta = kv_cta_of(item_end - 1, total, ctas);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        last_s = atomicAdd(a.count + first_cta, 1) == last_cta - first_cta;
        if (last_s) a.count[first_cta] = 0;
      }
      __syncthreads();
      if (last_s) {
        __threadfence();
        for (int i = tid; i < rows * HD / 4; i += W * 32) {
          const int r = i / (HD / 4), c4 = i - r * (HD / 4);
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
          write(r, c4, M, L, o);
        }
      }
    }
    __syncthreads();  // the shared memory is the rings again

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
            w = kv_rows(a.s, a.c.page, a.group, RT, b, a.err);
          } while (w.tiles == 0);
        }
      }
      units = kv_run_units(w, tile / w.parts, UNIT);
    }
  }
}

template <int HD, int W>
int launch(Context* ctx, const AttnKv& a, cudaStream_t s) {
  using S = Shape<HD, W>;
  static thread_local int ready = -1;  // device on which the attribute is set
  if (ready != ctx->device) {
    const cudaError_t e =
        cudaFuncSetAttribute(attention_kv_kernel<HD, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
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
  glc::launch_pdl(ctx, attention_kv_kernel<HD, W>, dim3(ctas), dim3(W * 32), S::SMEM, s, b);
  GLC_LAUNCH_CHECK(ctx, "attention_kv");
  return GLC_OK;
}

template <int HD>
int launch_for(Context* ctx, const AttnKv& a, cudaStream_t s) {
  // Few items are cut between many CTAs, and few large CTAs leave fewer parts to
  // join; of many items a CTA has several, and small CTAs overlap one's joins
  // with another's copies.
  const long long items = static_cast<long long>(a.s.rows) * ((a.group + 7) / 8) * a.c.kv_heads;
  return items >= ctx->num_sms / 2 ? launch<HD, 4>(ctx, a, s) : launch<HD, 16>(ctx, a, s);
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
  // the cache's share of the traffic depends on lengths that the host does not have
  glc::ProfScope prof(c, glc::PROF_OTHER, 8.0 * batch->num_rows * width, c->stream);
  switch (cache->head_dim) {
    case 32: return glc::launch_for<32>(c, a, c->stream);
    case 64: return glc::launch_for<64>(c, a, c->stream);
    case 96: return glc::launch_for<96>(c, a, c->stream);
    default: return glc::launch_for<128>(c, a, c->stream);
  }
}
