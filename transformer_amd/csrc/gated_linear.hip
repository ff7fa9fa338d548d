// The first half of a gated feed-forward block (gfx950): h = bf16(act(x Wg^T) o (x Wu^T)), both products of a tile in one
// pass over x, and its gradient through the second product: dh = dy Wd stays in the accumulators, where the saved g and u turn
// it into dg and du.  The products are gemm_core.h's tiles.
//
// One kernel for both products reads x once and leaves h alone: apart, g and u would be written and read again (12288 x 4608:
// 453 MB of traffic more).  12288 rows, 1792 -> 2 x 4608, us: 331 without and 378 with the kept g and u (340 MB; 1070 TFLOP/s),
// backward 279 (730 TFLOP/s beside 340 MB of kept values read and 226 MB stored).
//
// Rounded to bf16 once each: h, dg and du, because the next products' matrix instructions take bf16 operands (fp32 ones would
// run at a sixteenth of the rate and move twice the bytes).  Relative rms of y against 64 bits 0.0018 to 0.0019 (a lone rounding of
// y 0.0017), of the gradients 0.0023 to 0.0024 (0.0017).
#include "gemm_epilogue.h"
#include "linear_checks.h"
#include "rows_core.h"

namespace mla {

struct GatedParams {
  GemmArgs g;
  bf16* out;             // h [M][N], or dgu [M][2 N]
  unsigned char* saved;  // g and u: blocks of 32 x 32, g's then u's of each
  int64_t os;
};

__device__ __forceinline__ unsigned char* gated_saved_at(const GatedParams& p, int m, int n) {
  return p.saved + ((int64_t)(m >> 5) * ((p.g.N + 31) >> 5) + (n >> 5)) * (2 * kSavedBlock);
}

// A tile covers TW / 2 columns of both weights, a wave's first blocks the gate's and the others the same columns of the up
// projection, so that a lane holds g and u of one output in the same registers of two blocks.  The epilogue of the blocks
// [j0, j1) of each wave: all of them at once, or (ALL false) one.
template <class C, int ACT, bool ALL>
__device__ __forceinline__ void gated_epilogue(const GatedParams& p, GemmAcc<C>& acc, int m0, int n0, unsigned char* s0,
                                               unsigned char* s1, int j0, int j1) {
  const WavePos<C> at;
  const StagedRows<C, C::TN> st{s0, s1};
  constexpr int HB = C::NB / 2;
  const int mv = min(C::TM, p.g.M - m0), nv = min(C::TN, p.g.N - n0);
#pragma unroll
  for (int j = 0; j < C::XJ; ++j) {
    if (j < j0 || j >= j1) continue;
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const f32x16 &g = acc.a[i][j], &u = acc.a[HB + i][j];
      const int mb = 32 * (C::XJ * at.wm + j), nb = 32 * (at.wn * HB + i);
      if (p.saved && mb < mv && nb < nv) {
        unsigned char* to = gated_saved_at(p, m0 + mb, n0 + nb);
        saved_store(to, at.lane, g);
        saved_store(to + kSavedBlock, at.lane, u);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = act_value<ACT>(g[4 * q + e]) * u[4 * q + e];
        sts8(st.at((ALL ? mb : 32 * at.wm) + at.l32, nb / 8 + q) + 8 * at.hk,
             u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
      }
    }
  }
  __syncthreads();
  store_rows<C>(st, at.tid, ALL ? C::TM : 32 * C::WM, p.out + (int64_t)m0 * p.os + n0, p.os, mv, nv,
                [&](int r) { return ALL ? r : pass_row<C>(r, j0); });
  __syncthreads();
}

template <class C, int ACT>
__global__ __launch_bounds__(C::THREADS, 2) void gated_linear_kernel(GatedParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
  gemm_tiles<C>(p.g, lds, [&](GemmAcc<C>& acc, int m0, int n0, unsigned char* s0, unsigned char* s1, int j0, int j1) {
    gated_epilogue<C, ACT, true>(p, acc, m0, n0, s0, s1, j0, j1);
  });
}

template <class C, int ACT>
__global__ __launch_bounds__(C::THREADS, 1) void gated_linear_finish_kernel(GatedParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[C::XSLOT + C::WSLOT];
  gemm_finish<C>(p.g, lds, [&](GemmAcc<C>& acc, int m0, int n0, unsigned char* s0, unsigned char* s1, int j0, int j1) {
    gated_epilogue<C, ACT, false>(p, acc, m0, n0, s0, s1, j0, j1);
  });
}

// Small tiles at any size: the saved values' loads and the two outputs' stores of one workgroup run under the products of the
// CU's other one (12288 x 4608 over 1792 270-280 us, 331 to 452 with tiles of 256 x 256, 277 with 256 x 128, which lose 12 to
// 35 % at 300 to 3000 rows; the product with a plain store takes 235).
template <class C, int ACT>
__global__ __launch_bounds__(C::THREADS, 2) void gated_linear_bwd_kernel(GatedParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
  gemm_tiles<C>(p.g, lds, [&](GemmAcc<C>& acc, int m0, int n0, unsigned char* s0, unsigned char* s1, int, int) {
    const WavePos<C> at;
    const StagedRows<C, C::TW> st{s0, s1};
    const int mv = min(C::TM, p.g.M - m0), nv = min(C::TW, p.g.N - n0);
    const int sr = 32 * at.wm + at.l32;
    bf16* out = p.out + (int64_t)m0 * p.os + n0;
    // g and u of a pass's blocks, read together and, for the second pass, under the first one's stores (a block without
    // outputs to store reads another one's)
    SavedRegs g[C::NB], u[C::NB];
    auto fetch = [&](int j) {
#pragma unroll
      for (int i = 0; i < C::NB; ++i) {
        const int mb = 32 * (C::XJ * at.wm + j), nb = 32 * (at.wn * C::NB + i);
        const unsigned char* from = gated_saved_at(p, m0 + (mb < mv ? mb : 0), n0 + (nb < nv ? nb : 0));
        g[i] = saved_load(from, at.lane);
        u[i] = saved_load(from + kSavedBlock, at.lane);
      }
    };
    fetch(0);
#pragma unroll
    for (int j = 0; j < C::XJ; ++j) {
#pragma unroll
      for (int i = 0; i < C::NB; ++i) {
        f32x16& dh = acc.a[i][j];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float dg[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float value, slope;
            act_both<ACT>(saved_value(g[i], 4 * q + e), value, slope);
            dg[e] = dh[4 * q + e] * saved_value(u[i], 4 * q + e) * slope;
            dh[4 * q + e] *= value;  // du
          }
          sts8(st.at(sr, 4 * (at.wn * C::NB + i) + q) + 8 * at.hk,
               u32x2{pack_bf16x2(dg[0], dg[1]), pack_bf16x2(dg[2], dg[3])});
        }
      }
      if (j + 1 < C::XJ) fetch(j + 1);
      __syncthreads();
      store_rows<C>(st, at.tid, 32 * C::WM, out, p.os, mv, nv, [&](int r) { return pass_row<C>(r, j); });
      __syncthreads();
#pragma unroll
      for (int i = 0; i < C::NB; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& du = acc.a[i][j];
          sts8(st.at(sr, 4 * (at.wn * C::NB + i) + q) + 8 * at.hk,
               u32x2{pack_bf16x2(du[4 * q], du[4 * q + 1]), pack_bf16x2(du[4 * q + 2], du[4 * q + 3])});
        }
      __syncthreads();
      store_rows<C>(st, at.tid, 32 * C::WM, out + p.g.N, p.os, mv, nv, [&](int r) { return pass_row<C>(r, j); });
      __syncthreads();
    }
  });
}

template <int MB, int CG, int ACT>
__global__ __launch_bounds__(64 * kRcWaves) void gated_linear_rows_kernel(GatedParams p, RowsArgs r) {
  typedef RowsProduct<MB, CG, true> Product;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Product::LDS];
  Product t;
  t.run(r, lds);
  if (!t.mine) return;
  const f32x4 g = t.sum[0], u = t.sum[1];
  if (p.saved) {
    unsigned char* to = gated_saved_at(p, t.m, t.n);
    saved_store4(to, t.m, t.n, g);
    saved_store4(to + kSavedBlock, t.m, t.n, u);
  }
  f32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = act_value<ACT>(g[e]) * u[e];
  stg8(p.out + t.m * p.os + t.n, u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
}

template <int CG, int ACT>
static void gated_rows_launch(const GatedParams& p, hipStream_t s) {
  const RowsArgs r{p.g.x, p.g.w0, p.g.w1, p.g.xs, p.g.ws0, p.g.ws1, p.g.M, p.g.N, p.g.K};
  const dim3 grid((unsigned)((r.N + CG - 1) / CG)), wg(64 * kRcWaves);
  if (r.M <= 16) gated_linear_rows_kernel<1, CG, ACT><<<grid, wg, 0, s>>>(p, r);
  else if (r.M <= 32) gated_linear_rows_kernel<2, CG, ACT><<<grid, wg, 0, s>>>(p, r);
  else gated_linear_rows_kernel<4, CG, ACT><<<grid, wg, 0, s>>>(p, r);
}
template <int ACT>
static void gated_rows_go(const GatedParams& p, hipStream_t s) {
  if (rows_columns(p.g.N) == 16) gated_rows_launch<16, ACT>(p, s);
  else gated_rows_launch<32, ACT>(p, s);
}

template <class C, bool BWD, int ACT>
static void gated_go(const GatedParams& p, hipStream_t s) {
  if constexpr (BWD) {
    gated_linear_bwd_kernel<C, ACT><<<dim3(gemm_grid<C>(p.g)), dim3(C::THREADS), 0, s>>>(p);
  } else {
    gated_linear_kernel<C, ACT><<<dim3(gemm_grid<C>(p.g)), dim3(C::THREADS), 0, s>>>(p);
    if (p.g.S > 1) gated_linear_finish_kernel<C, ACT><<<dim3(gemm_finish_grid<C>(p.g)), dim3(C::THREADS), 0, s>>>(p);
  }
}

template <class C, bool BWD>
static void gated_launch(const GatedParams& p, int act, hipStream_t s) {
  if (act == MLA_ACT_RELU) gated_go<C, BWD, MLA_ACT_RELU>(p, s);
  else if (act == MLA_ACT_SILU) gated_go<C, BWD, MLA_ACT_SILU>(p, s);
  else gated_go<C, BWD, MLA_ACT_GELU_TANH>(p, s);
}

static int check_gate(const char* op, int act) {
  MLA_CHECK(act > MLA_ACT_NONE && act <= MLA_ACT_GELU_TANH, MLA_ERR_UNSUPPORTED, "%s: activation %d", op, act);
  return MLA_OK;
}

}  // namespace mla

using namespace mla;

extern "C" size_t mla_gated_linear_workspace_bytes(const mla_gated_linear_args* a) {
  // 0 for the sizes mla_gated_linear rejects
  if (!a || check_linear_sizes("mla_gated_linear", a->M, a->N, a->K) != MLA_OK || a->M <= kRcMaxRows) return 0;
  return (size_t)gemm_plan(a->M, 2 * a->N, a->K, 1).part_bytes;
}

extern "C" int mla_gated_linear(const mla_gated_linear_args* a, void* stream) {
  const char* op = "mla_gated_linear";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_TRY(check_linear_sizes(op, a->M, a->N, a->K));
  MLA_TRY(check_gate(op, a->activation));
  if (a->M == 0) return MLA_OK;
  MLA_TRY(check_rows(op, "x", a->x, a->K, a->x_stride));
  MLA_TRY(check_rows(op, "w_gate", a->w_gate, a->K, a->w_gate_stride));
  MLA_TRY(check_rows(op, "w_up", a->w_up, a->K, a->w_up_stride));
  MLA_TRY(check_rows(op, "h", a->h, a->N, a->h_stride));
  MLA_CHECK(((uintptr_t)a->saved & 15) == 0, MLA_ERR_INVALID_ARG, "%s: saved must be 16-byte aligned", op);
  GatedParams p{};
  p.g.x = (const bf16*)a->x, p.g.w0 = (const bf16*)a->w_gate, p.g.w1 = (const bf16*)a->w_up;
  p.g.xs = a->x_stride, p.g.ws0 = a->w_gate_stride, p.g.ws1 = a->w_up_stride;
  p.g.M = (int)a->M, p.g.N = (int)a->N, p.g.K = (int)a->K, p.g.parts = 1;
  p.out = (bf16*)a->h;
  p.saved = (unsigned char*)a->saved;
  p.os = a->h_stride;
  hipStream_t s = (hipStream_t)stream;
  if (a->M <= kRcMaxRows) {
    if (a->activation == MLA_ACT_RELU) gated_rows_go<MLA_ACT_RELU>(p, s);
    else if (a->activation == MLA_ACT_SILU) gated_rows_go<MLA_ACT_SILU>(p, s);
    else gated_rows_go<MLA_ACT_GELU_TANH>(p, s);
    return launch_status(op);
  }
  const GemmPlan pl = gemm_plan(a->M, 2 * a->N, a->K, 1);
  MLA_TRY(gemm_apply(op, p.g, pl, a->workspace, a->workspace_bytes, 2));
  if (pl.tile == kGemmLarge) gated_launch<GemmCfg<256, 256, 2, 4, false, true>, false>(p, a->activation, s);
  else if (pl.tile == kGemmHalf) gated_launch<GemmCfg<256, 128, 2, 4, false, true>, false>(p, a->activation, s);
  else gated_launch<GemmCfg<128, 128, 2, 2, false, true>, false>(p, a->activation, s);
  return launch_status(op);
}

extern "C" int mla_gated_linear_bwd(const mla_gated_linear_bwd_args* a, void* stream) {
  const char* op = "mla_gated_linear_bwd";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_TRY(check_linear_sizes(op, a->M, a->N, a->K));
  MLA_TRY(check_gate(op, a->activation));
  if (a->M == 0) return MLA_OK;
  MLA_TRY(check_rows(op, "dy", a->dy, a->K, a->dy_stride));
  MLA_TRY(check_rows(op, "w_down", a->w_down, a->N, a->w_stride));
  MLA_TRY(check_weight_reach(op, "w_down", a->K, a->w_stride));
  MLA_TRY(check_rows(op, "dgu", a->dgu, 2 * a->N, a->dgu_stride));
  MLA_CHECK(a->saved && ((uintptr_t)a->saved & 15) == 0, MLA_ERR_INVALID_ARG, "%s: saved must be given, 16-byte aligned", op);
  GatedParams p{};
  p.g.x = (const bf16*)a->dy, p.g.w0 = (const bf16*)a->w_down;
  p.g.xs = a->dy_stride, p.g.ws0 = a->w_stride;
  p.g.M = (int)a->M, p.g.N = (int)a->N, p.g.K = (int)a->K, p.g.parts = 1;
  p.out = (bf16*)a->dgu;
  p.saved = (unsigned char*)const_cast<void*>(a->saved);
  p.os = a->dgu_stride;
  hipStream_t s = (hipStream_t)stream;
  MLA_TRY(gemm_apply(op, p.g, GemmPlan{kGemmSmall, 1, 0, 0}, nullptr, 0));
  gated_launch<GemmCfg<128, 128, 2, 2, true, false>, true>(p, a->activation, s);
  return launch_status(op);
}
