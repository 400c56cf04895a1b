// The paged 4-bit key/value cache: storing new tokens (with the rotation of
// keys and queries) and reading tokens back.
//
// Both are one pass over their operands: a stored token moves (num_heads + 2
// num_kv_heads) * head_dim floats in, num_heads * head_dim floats and
// 2 num_kv_heads * head_dim * 9/16 bytes out.  13916 tokens of 32/8 heads of 128
// with their read-back take 164 to 168 us, 0.66 to 0.68 of a plain copy's rate; looking each
// row up on its own and reading none ahead took 281.
#include <cfloat>
#include <climits>

#include "kv_cache.cuh"

namespace glc {
namespace {

constexpr int ROWS = 256;  // rows that a block looks up at once, a thread each
constexpr int AHEAD = 4;   // of them, read before the first is used
constexpr int MOST = 8;    // rows of a block

// Where a row lies.  The lookup is four or five reads deep: done for all of a
// block's rows at once, the rows' own reads then wait for none of it.
struct RowAt {
  int pos;   // -1: no token
  int page;  // -1: none
  int slot;
};
__device__ __forceinline__ RowAt row_at(const KvPools& c, const KvSeqs& s, int t, int limit, int* err) {
  RowAt r = {-1, -1, 0};
  int seq, pos;
  if (t < s.rows && kv_row(s, c.page, t, err, &seq, &pos)) {
    if (pos >= limit) {
      kv_bad(err);
    } else {
      const int index = pos / c.page;
      r.pos = pos;
      r.slot = pos - index * c.page;
      r.page = kv_page(s, c.num_pages, seq, index, err);
    }
  }
  return r;
}

// Codes of 4 elements where x (1 / d) may lie to the wrong side of a half: the
// residual x - n d is exact (n d has 15 bits, and the difference lies on x's grid
// and below d), and is held against d / 2.
__device__ __noinline__ unsigned nearest_codes(const float* x, float d, float rd) {
  const float edge = 0.5f * fabsf(d);
  unsigned bits = 0;
  for (int i = 0; i < 4; ++i) {
    float n = rintf(__fmul_rn(x[i], rd));
    n = fminf(fmaxf(n, -16.f), 16.f);
    const float rest = fmaf(-n, d, x[i]);
    const float by = (rest < 0.f) == (d < 0.f) ? 1.f : -1.f;
    if (fabsf(rest) > edge || (fabsf(rest) == edge && (static_cast<int>(n) & 1))) n += by;
    n = fminf(fmaxf(n, -8.f), 7.f);
    bits |= static_cast<unsigned>(static_cast<int>(n) + 8) << (4 * i);
  }
  return bits;
}

// The call's sequences, dealt out over the threads of the first `lookers` rows of blocks.
// The last thing of a kernel: as the first it took the append to 74 registers, and the
// ragged batch above 179 us for 165.
__device__ __forceinline__ void look_at_all(const KvPools& c, const KvSeqs& s, int lookers, int* err) {
  if (blockIdx.y >= lookers) return;
  const long long block = static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x;
  kv_look(s, c.page, block * blockDim.x + threadIdx.x, static_cast<long long>(lookers) * gridDim.x * blockDim.x, err);
}

// A thread holds 4 consecutive elements (two rotation pairs) of one head of
// one row; 8 neighbouring lanes hold the 32 that share a scale, so the largest
// magnitude is three shuffles.  blockIdx.x covers the heads of a row (queries,
// keys, values, in that order), blockIdx.y the rows, `step` in a row for a block.
__global__ void __launch_bounds__(256)
    kv_append_kernel(KvPools c, KvSeqs s, const float* q, size_t q_ld, float* q_out, size_t q_out_ld, int heads,
                     const float* k, size_t k_ld, const float* v, size_t v_ld, const float* __restrict__ cos_t,
                     const float* __restrict__ sin_t, int table_rows, int step, int lookers,
                     int* __restrict__ err) {
  GLC_PDL_ENTRY();
  __shared__ RowAt at_s[ROWS];
  const int quads = c.head_dim >> 2;
  const int u = blockIdx.x * blockDim.x + threadIdx.x;
  const int head = u / quads, at = u - head * quads;
  const bool is_q = head < heads, is_k = !is_q && head < heads + c.kv_heads;
  // units come in whole groups of 8 lanes; those past the row stay for the shuffles
  const bool some = head < heads + 2 * c.kv_heads;
  const int h = is_q ? head : is_k ? head - heads : head - heads - c.kv_heads;
  const int half = c.head_dim >> 1;
  const int lane = threadIdx.x & 31;
  const float* src = (is_q ? q : is_k ? k : v) + static_cast<size_t>(h) * c.head_dim + 4 * at;
  const size_t ld = is_q ? q_ld : is_k ? k_ld : v_ld;
  const bool turn = cos_t && (is_q || is_k);
  const int end = min(s.rows, (static_cast<int>(blockIdx.y) + 1) * step);
  for (int t0 = blockIdx.y * step; t0 < end; t0 += ROWS) {
    const int rows = min(ROWS, end - t0);
    __syncthreads();
    if (threadIdx.x < rows) at_s[threadIdx.x] = row_at(c, s, t0 + threadIdx.x, cos_t ? table_rows : INT_MAX, err);
    __syncthreads();
    for (int r0 = 0; r0 < rows; r0 += AHEAD) {
      float4 x4[AHEAD];
      float2 co[AHEAD], si[AHEAD];
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) {
        x4[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        co[r] = si[r] = make_float2(0.f, 0.f);
        if (r0 + r < rows && some && at_s[r0 + r].pos >= 0) {
          const int pos = at_s[r0 + r].pos;
          x4[r] = *reinterpret_cast<const float4*>(src + (t0 + r0 + r) * ld);
          if (turn) {
            co[r] = reinterpret_cast<const float2*>(cos_t + static_cast<size_t>(pos) * half)[at];
            si[r] = reinterpret_cast<const float2*>(sin_t + static_cast<size_t>(pos) * half)[at];
          }
        }
      }
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) {
        if (r0 + r >= rows || at_s[r0 + r].pos < 0) continue;  // the same for the whole block
        const RowAt place = at_s[r0 + r];
        float x[4] = {x4[r].x, x4[r].y, x4[r].z, x4[r].w};
        if (turn) {
          // glc_rope's arithmetic: every product and sum rounded on its own
          const float a0 = __fsub_rn(__fmul_rn(x[0], co[r].x), __fmul_rn(x[1], si[r].x));
          const float b0 = __fadd_rn(__fmul_rn(x[0], si[r].x), __fmul_rn(x[1], co[r].x));
          const float a1 = __fsub_rn(__fmul_rn(x[2], co[r].y), __fmul_rn(x[3], si[r].y));
          const float b1 = __fadd_rn(__fmul_rn(x[2], si[r].y), __fmul_rn(x[3], co[r].y));
          x[0] = a0, x[1] = b0, x[2] = a1, x[3] = b1;
        }
        if (is_q)
          *reinterpret_cast<float4*>(q_out + (t0 + r0 + r) * q_out_ld + static_cast<size_t>(h) * c.head_dim + 4 * at) =
              make_float4(x[0], x[1], x[2], x[3]);
        if (__all_sync(~0u, is_q)) continue;
        // the element of largest magnitude among the 32, the first of equals, and
        // whether all are finite; no early exit, so every lane takes the shuffles
        float m = x[0];
        bool fine = fabsf(x[0]) <= FLT_MAX;
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          if (fabsf(x[i]) > fabsf(m)) m = x[i];
          fine = fine && fabsf(x[i]) <= FLT_MAX;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          const float pm = __shfl_xor_sync(~0u, m, o);
          if (fabsf(pm) > fabsf(m) || (fabsf(pm) == fabsf(m) && (lane & o))) m = pm;
        }
        const unsigned all_fine = __ballot_sync(~0u, fine);
        if (!some || is_q || place.page < 0) continue;
        const bool nan = ((all_fine >> (lane & 24)) & 0xffu) != 0xffu;
        const __half d16 = nan ? __ushort_as_half(0x7e00)
                               : __float2half_rn(fminf(fmaxf(__fmul_rn(m, -0.125f), -65504.f), 65504.f));
        const float d = __half2float(d16);
        unsigned bits = 0x8888u;
        if (!nan && d != 0.f) {
          // the whole number nearest to the exact x / d: x (1 / d) is off by 2^-24 of
          // itself, so below 12 it rounds to the same one unless it is within 10^-6 of
          // a half (or d was held to the largest half)
          const float rd = __frcp_rn(d);
          constexpr float ROUND = 12582912.f;  // 1.5 2^23: the nearest whole number in the low bits of a sum
          float off = fabsf(m) <= 524032.f ? 0.f : 1.f;
          bits = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float sum = fmaf(x[i], rd, ROUND);
            off = fmaxf(off, fabsf(fmaf(x[i], rd, ROUND - sum)));
            const int n = static_cast<int>(__float_as_uint(sum)) - 0x4b400000 + 8;
            bits |= static_cast<unsigned>(n < 0 ? 0 : n > 15 ? 15 : n) << (4 * i);
          }
          if (off > 0.499998f) bits = nearest_codes(x, d, rd);
        }
        uint8_t* to = (is_k ? c.k : c.v) + (static_cast<size_t>(place.page) * c.kv_heads + h) * c.chunk;
        reinterpret_cast<uint16_t*>(to + static_cast<size_t>(place.slot) * half)[at] = static_cast<uint16_t>(bits);
        if ((lane & 7) == 0)
          reinterpret_cast<__half*>(to + c.scales_at)[place.slot * (c.head_dim / KV_GROUP) + (at >> 3)] = d16;
      }
    }
  }
  look_at_all(c, s, lookers, err);
}

// A thread reads 4 codes (2 bytes) and their scale and writes 4 floats; rows as above.
__global__ void __launch_bounds__(256, 8)
    kv_read_kernel(KvPools c, KvSeqs s, float* __restrict__ k, size_t k_ld, float* __restrict__ v, size_t v_ld,
                   int step, int lookers, int* __restrict__ err) {
  GLC_PDL_ENTRY();
  __shared__ RowAt at_s[ROWS];
  const int quads = c.head_dim >> 2;
  int u = blockIdx.x * blockDim.x + threadIdx.x;
  const int one = c.kv_heads * quads;
  // with one of k and v missing, the units are the other's alone
  const bool some = u < one * ((k ? 1 : 0) + (v ? 1 : 0));
  const bool is_k = k && u < one;
  if (k && !is_k) u -= one;
  const int h = u / quads, at = u - h * quads;
  const uint8_t* from = (is_k ? c.k : c.v) + static_cast<size_t>(h) * c.chunk;
  const size_t page_bytes = c.chunk * c.kv_heads;
  float* to = (is_k ? k : v) + static_cast<size_t>(h) * c.head_dim + 4 * at;
  const size_t ld = is_k ? k_ld : v_ld;
  const int end = min(s.rows, (static_cast<int>(blockIdx.y) + 1) * step);
  for (int t0 = blockIdx.y * step; t0 < end; t0 += ROWS) {
    const int rows = min(ROWS, end - t0);
    __syncthreads();
    if (threadIdx.x < rows) at_s[threadIdx.x] = row_at(c, s, t0 + threadIdx.x, INT_MAX, err);
    __syncthreads();
    if (!some) continue;
    for (int r0 = 0; r0 < rows; r0 += AHEAD) {
      uint32_t w[AHEAD];
      __half d[AHEAD];
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) {
        w[r] = 0;
        d[r] = __ushort_as_half(0);
        if (r0 + r < rows && at_s[r0 + r].page >= 0) {
          const uint8_t* p = from + static_cast<size_t>(at_s[r0 + r].page) * page_bytes;
          const int slot = at_s[r0 + r].slot;
          w[r] = reinterpret_cast<const uint16_t*>(p + static_cast<size_t>(slot) * (c.head_dim >> 1))[at];
          d[r] = reinterpret_cast<const __half*>(p + c.scales_at)[slot * (c.head_dim / KV_GROUP) + (at >> 3)];
        }
      }
#pragma unroll
      for (int r = 0; r < AHEAD; ++r) {
        if (r0 + r >= rows || at_s[r0 + r].page < 0) continue;
        const float f = __half2float(d[r]);
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(f, static_cast<float>(static_cast<int>((w[r] >> (4 * i)) & 15u) - 8));
        *reinterpret_cast<float4*>(to + (t0 + r0 + r) * ld) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
  }
  look_at_all(c, s, lookers, err);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Blocks of 256 units by runs of rows: of one row while there are few, of up to
// `most` where the device is full anyway, since a run looks its rows up once.  Runs
// of 8 and 16: 28.2 and 33.0 us at 4 x 1024 tokens of 32/4 heads of 64, 160.6 and
// 156.4 us at 13916 of 32/8 heads of 128, both with their read-back.
struct RowGrid {
  dim3 grid;
  int step;
  int lookers;  // rows of blocks that look at the sequences
};
RowGrid row_grid(const Context* ctx, int units, int rows, int seqs, int most) {
  const int bx = (units + 255) / 256;
  const long long blocks = static_cast<long long>(bx) * rows, full = 8LL * ctx->num_sms;
  int step = 1;
  while (step < most && blocks > full * step) step *= 2;
  while ((rows + step - 1) / step > 65535) step *= 2;
  const int by = (rows + step - 1) / step, look = (seqs + 256 * bx - 1) / (256 * bx);
  return {dim3(bx, by), step, look < by ? look : by};
}

int cache_check(const char* what, const glc_kv_cache* c, std::string* msg) {
  auto no = [&](const char* why) {
    *msg = std::string(what) + ": " + why;
    return GLC_ERR_INVALID;
  };
  if (!c) return no("no cache given");
  if (c->num_pages <= 0 || c->num_kv_heads <= 0) return no("num_pages and num_kv_heads must be positive");
  if (c->page_size <= 0 || c->page_size % 16 || c->page_size > 65536)
    return no("page_size must be a multiple of 16, at most 65536");
  if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128) {
    *msg = std::string(what) + ": head_dim must be 32, 64, 96 or 128";
    return GLC_ERR_UNSUPPORTED;
  }
  // sizes and offsets are counted in 64 bits
  if (static_cast<double>(c->num_pages) * c->num_kv_heads * static_cast<double>(kv_pools(*c).chunk) > 4e18)
    return no("num_pages, num_kv_heads and page_size are too large together");
  return GLC_OK;
}

}  // namespace

int kv_check(Context* ctx, const char* what, const glc_kv_cache* cache, const glc_kv_batch* batch) {
  std::string msg;
  const int rc = cache_check(what, cache, &msg);
  if (rc) return ctx->fail(rc, msg);
  auto no = [&](const char* why) { return ctx->fail(GLC_ERR_INVALID, std::string(what) + ": " + why); };
  if (!cache->k || !cache->v || !aligned16(cache->k) || !aligned16(cache->v))
    return no("the cache's pools must be 16-byte aligned device memory");
  if (!batch) return no("no batch given");
  if (batch->num_seqs < 0 || batch->num_rows < 0 || batch->max_pages <= 0) return no("bad batch sizes");
  if (batch->num_seqs > 0 && (!batch->page_table || !batch->lens)) return no("page_table and lens must be given");
  if ((reinterpret_cast<uintptr_t>(batch->page_table) | reinterpret_cast<uintptr_t>(batch->lens) |
       reinterpret_cast<uintptr_t>(batch->starts)) & 3)
    return no("page_table, lens and starts must be 4-byte aligned");
  if (!batch->starts && batch->num_rows < batch->num_seqs)
    return no("without starts, num_rows must be at least num_seqs");
  if (static_cast<long long>(batch->max_pages) * cache->page_size > 0x40000000)
    return no("max_pages * page_size must be at most 2^30");
  return GLC_OK;
}

}  // namespace glc

using glc::Context;

extern "C" {

int glc_kv_cache_bytes(const glc_kv_cache* cache, size_t* bytes) {
  std::string msg;
  if (!bytes) return GLC_ERR_INVALID;
  const int rc = glc::cache_check("kv_cache_bytes", cache, &msg);
  if (rc) {
    glc::host_error() = msg;
    return rc;
  }
  *bytes = static_cast<size_t>(cache->num_pages) * cache->num_kv_heads * glc::kv_pools(*cache).chunk;
  return GLC_OK;
}

int glc_kv_append(glc_ctx* ctx, const glc_kv_cache* cache, const glc_kv_batch* batch, const float* q, int q_ld,
                  float* q_out, int q_out_ld, int num_heads, const float* k, int k_ld, const float* v, int v_ld,
                  const float* cos_t, const float* sin_t, int table_rows) {
  if (!ctx) return GLC_ERR_INVALID;
  Context* c = reinterpret_cast<Context*>(ctx);
  int rc = glc::kv_check(c, "kv_append", cache, batch);
  if (rc) return rc;
  auto no = [&](const char* why) { return c->fail(GLC_ERR_INVALID, std::string("kv_append: ") + why); };
  const long long kv_width = static_cast<long long>(cache->num_kv_heads) * cache->head_dim;
  const long long q_width = q ? static_cast<long long>(num_heads) * cache->head_dim : 0;
  if ((q == nullptr) != (q_out == nullptr)) return no("q and q_out must both be given, or neither");
  if (q && q == q_out && q_ld != q_out_ld) return no("q_out may be q where their strides are equal");
  if (q && num_heads <= 0) return no("num_heads must be positive");
  if ((cos_t == nullptr) != (sin_t == nullptr)) return no("cos_t and sin_t must both be given, or neither");
  if (cos_t && table_rows <= 0) return no("table_rows must be positive");
  if (!k || !v) return no("k and v must be given");
  if ((q && (q_ld < q_width || q_out_ld < q_width || ((q_ld | q_out_ld) & 3))) || k_ld < kv_width ||
      v_ld < kv_width || ((k_ld | v_ld) & 3))
    return no("row strides must be multiples of 4 and at least the row's width");
  if (!glc::aligned16(q) || !glc::aligned16(q_out) || !glc::aligned16(k) || !glc::aligned16(v) ||
      !glc::aligned16(cos_t) || !glc::aligned16(sin_t))
    return no("pointers must be 16-byte aligned");
  if (q_width + 2 * kv_width > (1 << 26)) return no("the rows are too wide");
  if (batch->num_rows == 0 || batch->num_seqs == 0) return GLC_OK;
  glc::DeviceScope on(c);
  const int heads = q ? num_heads : 0;
  const int units = (heads + 2 * cache->num_kv_heads) * (cache->head_dim / 4);
  const double moved = static_cast<double>(batch->num_rows) *
                       (8.0 * q_width + (8.0 + 9.0 / 8.0) * kv_width);
  glc::ProfScope prof(c, glc::PROF_OTHER, moved, c->stream);
  const glc::RowGrid g = glc::row_grid(c, units, batch->num_rows, batch->num_seqs, glc::MOST);
  glc::launch_pdl(c, glc::kv_append_kernel, g.grid, 256, 0, c->stream,
                  glc::kv_pools(*cache), glc::kv_seqs(*batch), q, static_cast<size_t>(q_ld), q_out,
                  static_cast<size_t>(q_out_ld), heads, k, static_cast<size_t>(k_ld), v, static_cast<size_t>(v_ld),
                  cos_t, sin_t, table_rows, g.step, g.lookers, c->d_err);
  GLC_LAUNCH_CHECK(c, "kv_append");
  return GLC_OK;
}

int glc_kv_read(glc_ctx* ctx, const glc_kv_cache* cache, const glc_kv_batch* batch, float* k, int k_ld, float* v,
                int v_ld) {
  if (!ctx) return GLC_ERR_INVALID;
  Context* c = reinterpret_cast<Context*>(ctx);
  int rc = glc::kv_check(c, "kv_read", cache, batch);
  if (rc) return rc;
  auto no = [&](const char* why) { return c->fail(GLC_ERR_INVALID, std::string("kv_read: ") + why); };
  const long long width = static_cast<long long>(cache->num_kv_heads) * cache->head_dim;
  if (!k && !v) return no("k or v must be given");
  if ((k && (k_ld < width || (k_ld & 3))) || (v && (v_ld < width || (v_ld & 3))))
    return no("row strides must be multiples of 4 and at least the row's width");
  if (!glc::aligned16(k) || !glc::aligned16(v)) return no("pointers must be 16-byte aligned");
  if (width > (1 << 26)) return no("the rows are too wide");
  if (batch->num_rows == 0 || batch->num_seqs == 0) return GLC_OK;
  glc::DeviceScope on(c);
  const int sides = (k ? 1 : 0) + (v ? 1 : 0);
  const int units = sides * cache->num_kv_heads * (cache->head_dim / 4);
  glc::ProfScope prof(c, glc::PROF_OTHER, static_cast<double>(batch->num_rows) * sides * width * (4.0 + 9.0 / 16.0),
                      c->stream);
  const glc::RowGrid g = glc::row_grid(c, units, batch->num_rows, batch->num_seqs, glc::MOST);
  glc::launch_pdl(c, glc::kv_read_kernel, g.grid, 256, 0, c->stream,
                  glc::kv_pools(*cache), glc::kv_seqs(*batch), k, static_cast<size_t>(k_ld), v,
                  static_cast<size_t>(v_ld), g.step, g.lookers, c->d_err);
  GLC_LAUNCH_CHECK(c, "kv_read");
  return GLC_OK;
}

}  // extern "C"
