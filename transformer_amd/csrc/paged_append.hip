// Appending to a paged latent cache with the rotation on the way, and reading rows back out of pages (gfx950).
//
// Both move each value once, 16 bytes a thread and access.  Measured (kernel trace; a copy in HBM reaches 4.7 TB/s): 8 prompts' chunks of up
// to 2048 tokens, 8450 in all, into 4-bit pages 16.6 us (63 MB, 3.8 TB/s; VALU busy 84 % of the time, most of it the quotients); 32000
// rows of 1280 values out of 16-bit pages, 20300 of them tokens, 20.5 (134 MB; 28 where all of it comes from and goes to HBM: a copy's
// rate).  Few rows are bound by the launch and by start, page and store one after the other: one token 2.2, 64 tokens 3.1.  In 4 bits the
// runs' exchanges and quotients stand in between: one token 3.0, 64 tokens 4.0 with 14 keys and 5.9 with one (why more is not known).
#include "paged.h"
#include "rope_append.h"

namespace mla {

struct PagedAppendParams {
  PagedParams c;
  const bf16 *qk, *c_new, *cos, *sin;
  bf16* q_out;
  const int32_t *starts, *counts;
  Divisor by_heads, by_T, by_row;
  uint32_t T, H, heads, DL, vectors, chunks;  // heads: H + Hr; vectors, chunks: threads of each part
  int limit;                                  // positions
  mla_strides qk_s;
  int64_t c_sb, c_st;
};

// A thread's position, -1 where its token is skipped.
__device__ __forceinline__ int append_position(const PagedAppendParams& a, uint32_t b, uint32_t t) {
  const int count = a.counts ? a.counts[b] : (int)a.T;
  const int64_t p = (int64_t)a.starts[b] + t;
  return (int)t < count && p >= 0 && p < a.limit ? (int)p : -1;
}

// y1 = x1 c - x2 s, y2 = x1 s + x2 c, each rounded to bf16 once, and to 4 bits from that, so that both caches hold what the rotation gave.
//
// Blocks [0, ceil(vectors / 256)): 4 threads a head vector, each 8 + 8 of its values (x[i] with x[i + 32]).  The others: a thread
// for 8 values of a latent row, so 8 neighbouring threads hold a run and its largest magnitude takes three exchanges.  One launch for
// both: a token's latency is the launch.
template <bool FOUR>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams a) {
  const uint32_t rope_blocks = (a.vectors + 255) / 256;
  float v[16];
  uint32_t b, col;
  int p;
  const bool rope = blockIdx.x < rope_blocks;
  const int part = threadIdx.x & (rope ? 3 : 7);
  if (rope) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.vectors) return;
    const uint32_t bt = a.by_heads.of(i >> 2), j = (i >> 2) - bt * a.heads;
    b = a.by_T.of(bt);
    const uint32_t t = bt - b * a.T;
    p = append_position(a, b, t);
    bf16* q = a.q_out + ((int64_t)bt * a.H + j) * 64 + 8 * part;
    if (p < 0) {
      if (j < a.H) {
        stg16(q, u32x4{0u, 0u, 0u, 0u});
        stg16(q + 32, u32x4{0u, 0u, 0u, 0u});
      }
      return;
    }
    const bf16* x = a.qk + b * a.qk_s.b + t * a.qk_s.t + j * a.qk_s.h + 8 * part;
    bf16x8 x1 = as_bf16x8(ldg16(x)), x2 = as_bf16x8(ldg16(x + 32));
    rope_rotate8(x1, x2, ldg16(a.cos + (int64_t)p * 32 + 8 * part), ldg16(a.sin + (int64_t)p * 32 + 8 * part));
    if (j < a.H) {
      stg16(q, as_u32x4(x1));
      stg16(q + 32, as_u32x4(x2));
      return;
    }
    col = a.DL + 64 * (j - a.H);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = (float)x1[e];
      v[8 + e] = (float)x2[e];
    }
  } else {
    const uint32_t i = (blockIdx.x - rope_blocks) * 256 + threadIdx.x;
    if (i >= a.chunks) return;
    const uint32_t bt = a.by_row.of(i);
    b = a.by_T.of(bt);
    col = (i - bt * (a.DL >> 3)) * 8;
    p = append_position(a, b, bt - b * a.T);
    if (p < 0) return;
    RopeIO<bf16>::load8(a.c_new + b * a.c_sb + (bt - b * a.T) * a.c_st + col, v);
  }
  const int page = a.c.by_size.of(p), slot = p - page * a.c.size, id = page_of(a.c, b, page);
  if (id < 0) return;  // (the threads of a run leave together)
  unsigned char* row = a.c.pages + id * a.c.page_stride + (int64_t)slot * a.c.row_bytes;
  if (!FOUR) {
    bf16* out = reinterpret_cast<bf16*>(row) + col + (rope ? 8 * part : 0);
    RopeIO<bf16>::store8(out, v);
    if (rope) RopeIO<bf16>::store8(out + 32, v + 8);
    return;
  }
  // (whole blocks rotate or copy: the second half of v is the rotating ones')
  auto largest = [](float a, float b) { return b > a || b != b ? b : a; };  // a NaN stays
  float amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = largest(amax, fabsf(v[e]));
  if (rope) {
#pragma unroll
    for (int e = 8; e < 16; ++e) amax = largest(amax, fabsf(v[e]));
  } else {
    amax = largest(amax, wave_shfl_xor(amax, 4));
  }
  amax = largest(amax, wave_shfl_xor(amax, 2));
  amax = largest(amax, wave_shfl_xor(amax, 1));
  const bf16 sc = run_scale(amax);
  const float scale = (float)sc;
  uint32_t w = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= code4(v[e], scale) << (4 * e);
  *reinterpret_cast<uint32_t*>(row + col / 2 + (rope ? 4 * part : 0)) = w;
  if (rope) {
    w = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= code4(v[8 + e], scale) << (4 * e);
    *reinterpret_cast<uint32_t*>(row + col / 2 + 16 + 4 * part) = w;
  }
  if (part == 0) a.c.scales[id * a.c.scale_stride + (int)(col >> 6) * a.c.size + slot] = sc;
}

struct PagedReadParams {
  PagedParams c;
  bf16 *latent, *k_rope;
  const int32_t *starts, *counts;
  Divisor by_row, by_T;
  uint32_t T, DL, Hr, chunks;
};

// A thread for 8 values of a row.
template <bool FOUR>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedReadParams a) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.chunks) return;
  const uint32_t bt = a.by_row.of(i), b = a.by_T.of(bt), t = bt - b * a.T, col = (i - bt * (a.c.groups * 8)) * 8;
  const int count = a.counts ? a.counts[b] : (int)a.T;
  const int64_t p = (int64_t)(a.starts ? a.starts[b] : 0) + t;
  u32x4 out = u32x4{0u, 0u, 0u, 0u};
  const int page = p >= 0 && p < (1ll << 31) ? (int)a.c.by_size.of((uint32_t)p) : -1;
  const int id = (int)t < count ? page_of(a.c, b, page) : -1;
  if (id >= 0) {
    const int slot = (int)p - page * a.c.size;
    const unsigned char* row = a.c.pages + id * a.c.page_stride + (int64_t)slot * a.c.row_bytes;
    if (!FOUR) {
      out = ldg16(row + 2 * col);
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(row + col / 2);
      const float s = (float)a.c.scales[id * a.c.scale_stride + (int)(col >> 6) * a.c.size + slot];
      for (int e = 0; e < 4; ++e)
        out[e] = pack_bf16x2((float)((int)((w >> (8 * e)) & 15) - 8) * s, (float)((int)((w >> (8 * e + 4)) & 15) - 8) * s);
    }
  }
  bf16* to = col < a.DL ? a.latent + (int64_t)bt * a.DL + col : a.k_rope + ((int64_t)(b * a.Hr + ((col - a.DL) >> 6)) * a.T + t) * 64 + (col & 63);
  stg16(to, out);
}

}  // namespace mla

using namespace mla;

extern "C" int mla_paged_append(const mla_paged_append_args* a, void* stream) {
  const char* op = "mla_paged_append";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_CHECK(a->B >= 0 && a->T >= 0 && a->H >= 0 && a->H <= 1024 && a->table_rows >= 0 && a->B < (1 << 24) && a->T < (1 << 24),
            MLA_ERR_INVALID_ARG, "%s: a size is out of range", op);
  PagedAppendParams p;
  MLA_TRY(paged_setup(a->cache, op, a->B, p.c));
  if (a->B == 0 || a->T == 0) return MLA_OK;
  const void* ptrs[] = {a->qk, a->c_new, a->cos, a->sin, a->q_out};
  for (const void* q : ptrs)
    MLA_CHECK((q || (q == a->q_out && a->H == 0)) && ((uintptr_t)q & 15) == 0, MLA_ERR_INVALID_ARG,
              "%s: a pointer is null or not 16-byte aligned", op);
  MLA_CHECK(a->starts && ((uintptr_t)a->starts & 3) == 0 && ((uintptr_t)a->counts & 3) == 0, MLA_ERR_INVALID_ARG,
            "%s: starts is null, or starts or counts is not 4-byte aligned", op);
  const int64_t st[] = {a->qk_stride.b, a->qk_stride.t, a->qk_stride.h, a->c_new_sb, a->c_new_st};
  for (int64_t s : st) MLA_CHECK(s >= 0 && (s & 7) == 0, MLA_ERR_INVALID_ARG, "%s: strides must be non-negative multiples of 8", op);
  p.qk = (const bf16*)a->qk;
  p.c_new = (const bf16*)a->c_new;
  p.cos = (const bf16*)a->cos;
  p.sin = (const bf16*)a->sin;
  p.q_out = (bf16*)a->q_out;
  p.starts = a->starts;
  p.counts = a->counts;
  const int64_t heads = a->H + a->cache.n_k_rope_heads, vectors = a->B * a->T * heads * 4, chunks = a->B * a->T * (a->cache.d_latent / 8);
  MLA_CHECK(vectors < (1ll << 31) - 256 && chunks < (1ll << 31) - 256, MLA_ERR_INVALID_ARG, "%s: too many rows", op);
  p.T = (uint32_t)a->T;
  p.H = (uint32_t)a->H;
  p.heads = (uint32_t)heads;
  p.DL = (uint32_t)a->cache.d_latent;
  p.vectors = (uint32_t)vectors;
  p.chunks = (uint32_t)chunks;
  p.by_heads = Divisor(p.heads);
  p.by_T = Divisor(p.T);
  p.by_row = Divisor(p.DL / 8);
  p.limit = (int)std::min(std::min(a->table_rows, a->cache.table_pages * a->cache.page_size), (int64_t)0x7fffffff);
  p.qk_s = a->qk_stride;
  p.c_sb = a->c_new_sb;
  p.c_st = a->c_new_st;
  const int64_t blocks = (vectors + 255) / 256 + (chunks + 255) / 256;
  if (p.c.scales)
    paged_append_kernel<true><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(p);
  else
    paged_append_kernel<false><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(p);
  return launch_status(op);
}

extern "C" int mla_paged_read(const mla_paged_read_args* a, void* stream) {
  const char* op = "mla_paged_read";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_CHECK(a->B >= 0 && a->T >= 0 && a->B < (1 << 24) && a->T < (1 << 24), MLA_ERR_INVALID_ARG, "%s: a size is out of range", op);
  PagedReadParams p;
  MLA_TRY(paged_setup(a->cache, op, a->B, p.c));
  if (a->B == 0 || a->T == 0) return MLA_OK;
  MLA_CHECK(a->latent && a->k_rope && ((uintptr_t)a->latent & 15) == 0 && ((uintptr_t)a->k_rope & 15) == 0, MLA_ERR_INVALID_ARG,
            "%s: latent or k_rope is null or not 16-byte aligned", op);
  MLA_CHECK(((uintptr_t)a->starts & 3) == 0 && ((uintptr_t)a->counts & 3) == 0, MLA_ERR_INVALID_ARG,
            "%s: starts or counts is not 4-byte aligned", op);
  p.latent = (bf16*)a->latent;
  p.k_rope = (bf16*)a->k_rope;
  p.starts = a->starts;
  p.counts = a->counts;
  const int64_t chunks = a->B * a->T * p.c.groups * 8, blocks = (chunks + 255) / 256;
  MLA_CHECK(chunks < (1ll << 31) - 256, MLA_ERR_INVALID_ARG, "%s: too many rows", op);
  p.T = (uint32_t)a->T;
  p.DL = (uint32_t)a->cache.d_latent;
  p.Hr = (uint32_t)a->cache.n_k_rope_heads;
  p.chunks = (uint32_t)chunks;
  p.by_row = Divisor((uint32_t)p.c.groups * 8);
  p.by_T = Divisor(p.T);
  if (p.c.scales)
    paged_read_kernel<true><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(p);
  else
    paged_read_kernel<false><<<dim3((unsigned)blocks), 256, 0, (hipStream_t)stream>>>(p);
  return launch_status(op);
}
