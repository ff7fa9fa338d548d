// Host-side checks and launch shapes of the linear layers' entry points.
#pragma once

#include "gemm_core.h"

namespace mla {

constexpr int64_t kLinearMaxM = 1 << 30, kLinearMaxN = 1 << 20, kLinearMaxStride = 1 << 22;

// Sizes of a product: rows of 16-byte chunks, 32-bit indexes of rows and tiles.  K = 0 (an empty sum) is refused.
inline int check_linear_sizes(const char* op, int64_t M, int64_t N, int64_t K) {
  MLA_CHECK(M >= 0 && N >= 0 && K >= 0 && M < kLinearMaxM && N < kLinearMaxN && K < kLinearMaxN, MLA_ERR_INVALID_ARG,
            "%s: size out of range", op);
  MLA_CHECK(N % 8 == 0 && K % 8 == 0 && N > 0 && K > 0, MLA_ERR_UNSUPPORTED,
            "%s: N = %lld and K = %lld must be positive multiples of 8", op, (long long)N, (long long)K);
  // tiles of 64 columns at least
  MLA_CHECK((M / 128 + 1) * (N / 64 + 1) < (1ll << 30) && (M / 128 + 1) * (K / 64 + 1) < (1ll << 30), MLA_ERR_INVALID_ARG,
            "%s: too many tiles", op);
  return MLA_OK;
}

// bf16 rows of `width` columns: a tile's 256 rows are addressed with 32-bit offsets from its first
inline int check_rows(const char* op, const char* name, const void* ptr, int64_t width, int64_t stride) {
  MLA_CHECK(ptr, MLA_ERR_INVALID_ARG, "%s: %s is null", op, name);
  MLA_CHECK(((uintptr_t)ptr & 15) == 0, MLA_ERR_INVALID_ARG, "%s: %s must be 16-byte aligned", op, name);
  MLA_CHECK(stride >= width && stride % 8 == 0, MLA_ERR_INVALID_ARG,
            "%s: %s's row stride %lld must cover a row and be a multiple of 8", op, name, (long long)stride);
  MLA_CHECK(stride < kLinearMaxStride, MLA_ERR_UNSUPPORTED, "%s: %s's row stride %lld is too large", op, name,
            (long long)stride);
  return MLA_OK;
}

// a weight read along its rows' direction is addressed as a whole with 32-bit byte offsets
inline int check_weight_reach(const char* op, const char* name, int64_t rows, int64_t stride) {
  MLA_CHECK((rows + 64) * stride * 2 < (1ll << 31), MLA_ERR_UNSUPPORTED, "%s: %s of 2 GiB or more", op, name);
  return MLA_OK;
}

// The plan's tiles and pieces; `cols` tile columns of an output column (2 for a pair of weights).  Without a workspace that
// is large enough a plan that cuts tiles is refused.
inline int gemm_apply(const char* op, GemmArgs& g, const GemmPlan& pl, void* workspace, size_t bytes, int cols = 1) {
  const GemmTile t = kGemmTiles[pl.tile];
  g.n_mt = (int)((g.M + t.m - 1) / t.m);
  g.n_nt = (int)(((int64_t)g.N * cols + t.n - 1) / t.n);
  g.gm = 8;
  const int tiles = g.n_mt * g.n_nt, slots = (int)t.slots;
  g.S = pl.S;
  g.per = pl.per;
  g.full = pl.S > 1 ? tiles / slots * slots : tiles;
  g.part = (float*)workspace;
  MLA_CHECK(pl.part_bytes == 0 || (workspace && bytes >= (size_t)pl.part_bytes && ((uintptr_t)workspace & 255) == 0),
            MLA_ERR_WORKSPACE, "%s: workspace of %lld bytes (256-byte aligned) needed, %zu given", op, (long long)pl.part_bytes,
            bytes);
  return MLA_OK;
}

// one workgroup per CU, or two that share one
template <class C>
inline unsigned gemm_grid(const GemmArgs& g) {
  const int64_t tiles = (int64_t)g.n_mt * g.n_nt, items = g.full + (tiles - g.full) * g.S;
  const int64_t most = C::LDS > 80 * 1024 ? 256 : 512;
  return (unsigned)(items < most ? items : most);
}
template <class C>
inline unsigned gemm_finish_grid(const GemmArgs& g) {
  return (unsigned)((g.n_mt * g.n_nt - g.full) * C::XJ);
}

}  // namespace mla
