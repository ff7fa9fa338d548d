// The paged latent cache (mla_paged_cache): where a token's row lies, its 4-bit form, and the checks of the entry points.
#pragma once
#include "mla_common.h"

namespace mla {

// Division of n < 2^31 by a number that is known at the launch: mul = ceil(2^(31 + l) / d) with 2^(l - 1) < d <= 2^l, so that n mul / 2^(31 + l)
// is off by less than 1 / d.  (A 64-bit division is over a hundred instructions, more than all else that a thread of the appending and
// reading kernels does.)
struct Divisor {
  uint32_t mul, d;
  int shift;
  Divisor() = default;
  explicit Divisor(uint32_t by) : d(by) {
    int l = 0;
    while ((1u << l) < by) ++l;
    mul = (uint32_t)((((uint64_t)1 << (31 + l)) + by - 1) / by);
    shift = l - 1;
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1 ? n : __umulhi(n, mul) >> shift; }
};

struct PagedParams {
  unsigned char* pages;
  bf16* scales;  // null: 16 bits
  const int32_t* table;
  int64_t page_stride, scale_stride, table_stride;
  Divisor by_size;
  int n_pages, size, table_pages, row_bytes, groups;  // row_bytes: of a row of a page; groups: runs of 64 values of a row
};

// The page of position p of sequence b, or -1: p >= 0 within the table, the entry one of the cache's pages.
__device__ __forceinline__ int page_of(const PagedParams& c, int64_t b, int64_t page) {
  if (page < 0 || page >= c.table_pages) return -1;
  const int id = c.table[b * c.table_stride + page];
  return id >= 0 && id < c.n_pages ? id : -1;
}

// A run's scale from its largest magnitude, and a value's code: exactly as stated, in correctly rounded fp32 (bf16 operands: no
// quotient rounds to a half that was none).  A NaN or infinity makes the scale one, which then makes every value of the run NaN.
__device__ __forceinline__ bf16 run_scale(float amax) { return (bf16)(amax / 7.0f); }
__device__ __forceinline__ uint32_t code4(float x, float scale) {
  const float c = rintf(x / scale);
  return scale > 0.f && c == c ? (uint32_t)(8 + (int)fminf(fmaxf(c, -7.f), 7.f)) : 8u;
}

inline int paged_setup(const mla_paged_cache& c, const char* op, int64_t B, PagedParams& p) {
  MLA_CHECK(c.d_latent == 64 || c.d_latent == 128 || c.d_latent == 256 || c.d_latent == 384 || c.d_latent == 512,
            MLA_ERR_UNSUPPORTED, "%s: d_latent %lld not built", op, (long long)c.d_latent);
  MLA_CHECK(c.n_k_rope_heads >= 1 && c.n_k_rope_heads <= 1024, MLA_ERR_INVALID_ARG, "%s: n_k_rope_heads %lld is not in 1 .. 1024", op,
            (long long)c.n_k_rope_heads);
  MLA_CHECK(c.page_size >= 16 && c.page_size <= 4096 && c.page_size % 16 == 0, MLA_ERR_INVALID_ARG,
            "%s: page_size %lld is not a multiple of 16 up to 4096", op, (long long)c.page_size);
  MLA_CHECK(c.n_pages >= 0 && c.n_pages < (1ll << 31) && c.table_pages >= 0 && c.table_pages < (1ll << 31) / c.page_size,
            MLA_ERR_INVALID_ARG, "%s: n_pages %lld or table_pages %lld is out of range", op, (long long)c.n_pages,
            (long long)c.table_pages);
  const int64_t W = c.d_latent + 64 * c.n_k_rope_heads, row = c.scales ? W / 2 : 2 * W;
  MLA_CHECK(c.pages || c.n_pages == 0, MLA_ERR_INVALID_ARG, "%s: pages is null", op);
  MLA_CHECK(c.block_table || B == 0 || c.table_pages == 0, MLA_ERR_INVALID_ARG, "%s: block_table is null", op);
  MLA_CHECK(((uintptr_t)c.block_table & 3) == 0, MLA_ERR_INVALID_ARG, "%s: block_table must be 4-byte aligned", op);
  MLA_CHECK(((uintptr_t)c.pages & 15) == 0 && ((uintptr_t)c.scales & 15) == 0, MLA_ERR_INVALID_ARG,
            "%s: pages and scales must be 16-byte aligned", op);
  MLA_CHECK(c.n_pages <= 1 || (c.page_stride >= c.page_size * row && c.page_stride % 16 == 0), MLA_ERR_INVALID_ARG,
            "%s: page_stride %lld must be a multiple of 16 that covers a page (%lld)", op, (long long)c.page_stride,
            (long long)(c.page_size * row));
  MLA_CHECK(!c.scales || c.n_pages <= 1 || (c.scale_stride >= c.page_size * (W / 64) && c.scale_stride % 8 == 0), MLA_ERR_INVALID_ARG,
            "%s: scale_stride %lld must be a multiple of 8 that covers a page's scales (%lld)", op, (long long)c.scale_stride,
            (long long)(c.page_size * (W / 64)));
  MLA_CHECK(B <= 1 || c.table_stride >= 0, MLA_ERR_INVALID_ARG, "%s: table_stride is negative", op);
  p.pages = (unsigned char*)c.pages;
  p.scales = (bf16*)c.scales;
  p.table = c.block_table;
  p.page_stride = c.page_stride;
  p.scale_stride = c.scale_stride;
  p.table_stride = c.table_stride;
  p.n_pages = (int)c.n_pages;
  p.size = (int)c.page_size;
  p.by_size = Divisor((uint32_t)c.page_size);
  p.table_pages = (int)c.table_pages;
  p.row_bytes = (int)row;
  p.groups = (int)(W / 64);
  return MLA_OK;
}

}  // namespace mla
