// Linear layers with their epilogue (gfx950): y = bf16(act(x W^T + bias) + residual), and the input gradient dx = dy W of one
// layer or of two over the same input (one fp32 sum).  The products are gemm_core.h's tiles; the epilogue works on the fp32
// accumulators, so bias, activation and residual cost no pass over y and no rounding of their own.
//
// Bound by the products (gemm_core.h), up to 64 rows by reading the weight (rows_core.h).  12288 rows, us: 1792 -> 4608 with bias,
// gelu and the kept pre-activations (302 MB out) 224 + 20 for the tiles cut along k (830 TFLOP/s; the epilogue's arithmetic and
// stores run with the matrix units idle), 4608 -> 1792 178 + 16, dx of the former 187 + 14, of two layers 1792 -> 4608 together
// 346 + 15 (1120 TFLOP/s).

#include "gemm_epilogue.h"
#include "linear_checks.h"
#include "rows_core.h"

namespace mla {

struct LinearParams {
  GemmArgs g;
  const void* bias;
  const bf16* residual;
  bf16* y;
  unsigned char* saved;
  int64_t rs, ys;
  bool bias_f32;
};

// b[q] = bias[n .. n + 3] for n = at(q), a multiple of 4
template <int Q, class At>
__device__ __forceinline__ void linear_bias(const LinearParams& p, f32x4 (&b)[Q], At&& at) {
  if (p.bias_f32) {
#pragma unroll
    for (int q = 0; q < Q; ++q) b[q] = __builtin_bit_cast(f32x4, ldg16((const float*)p.bias + at(q)));
  } else {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const u32x2 v = ldg8((const bf16*)p.bias + at(q));
      b[q] = f32x4{lo_bf16(v[0]), hi_bf16(v[0]), lo_bf16(v[1]), hi_bf16(v[1])};
    }
  }
}

// The epilogue of the blocks [j0, j1) of each wave
template <class C, int ACT>
__device__ __forceinline__ void linear_epilogue(const LinearParams& p, GemmAcc<C>& acc, int m0, int n0,
                                                unsigned char* s0, unsigned char* s1, int j0, int j1) {
  const WavePos<C> at;
  const StagedRows<C, C::TW> st{s0, s1};
  constexpr int R = 32 * C::WM, CH = C::TW / 8;
  const int mv = min(C::TM, p.g.M - m0), nv = min(C::TW, p.g.N - n0);
  const int sr = 32 * at.wm + at.l32;
#pragma unroll
  for (int j = 0; j < C::XJ; ++j) {
    if (j < j0 || j >= j1) continue;
    if (p.residual) {
      const bf16* res = p.residual + (int64_t)m0 * p.rs + n0;
#pragma unroll 4
      for (int c = at.tid; c < R * CH; c += C::THREADS) {
        const int r = c / CH, ch = c % CH, m = pass_row<C>(r, j);
        if (m < mv && 8 * ch < nv) sts16(st.at(r, ch), ldg16(res + m * p.rs + 8 * ch));
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < C::NB; ++i) {
      f32x16 a = acc.a[i][j];
      const int nb = (at.wn * C::NB + i) * 32;  // the block's first column within the tile
      if (p.bias) {  // (columns past the last are not stored; one branch on the type a block, whose loads go out together)
        f32x4 b[4];
        linear_bias(p, b, [&](int q) { return n0 + min(nb + 8 * q + 4 * at.hk, nv - 4); });
#pragma unroll
        for (int e = 0; e < 16; ++e) a[e] += b[e >> 2][e & 3];
      }
      const int mb = 32 * (C::XJ * at.wm + j);
      if (p.saved && mb < mv && nb < nv)
        saved_store(p.saved + ((int64_t)((m0 + mb) >> 5) * ((p.g.N + 31) >> 5) + ((n0 + nb) >> 5)) * kSavedBlock, at.lane, a);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        unsigned char* to = st.at(sr, nb / 8 + q) + 8 * at.hk;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = act_value<ACT>(a[4 * q + e]);
        if (p.residual) {
          const u32x2 b = lds8(to);
          v[0] += lo_bf16(b[0]);
          v[1] += hi_bf16(b[0]);
          v[2] += lo_bf16(b[1]);
          v[3] += hi_bf16(b[1]);
        }
        sts8(to, u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
      }
    }
    __syncthreads();
    store_rows<C>(st, at.tid, R, p.y + (int64_t)m0 * p.ys + n0, p.ys, mv, nv, [&](int r) { return pass_row<C>(r, j); });
    __syncthreads();
  }
}

template <class C, int ACT>
__global__ __launch_bounds__(C::THREADS, 2) void linear_act_kernel(LinearParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[C::LDS];
  gemm_tiles<C>(p.g, lds, [&](GemmAcc<C>& acc, int m0, int n0, unsigned char* s0, unsigned char* s1, int j0, int j1) {
    linear_epilogue<C, ACT>(p, acc, m0, n0, s0, s1, j0, j1);
  });
}

template <class C, int ACT>
__global__ __launch_bounds__(C::THREADS, 1) void linear_act_finish_kernel(LinearParams p) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[C::XSLOT + C::WSLOT];
  gemm_finish<C>(p.g, lds, [&](GemmAcc<C>& acc, int m0, int n0, unsigned char* s0, unsigned char* s1, int j0, int j1) {
    linear_epilogue<C, ACT>(p, acc, m0, n0, s0, s1, j0, j1);
  });
}

template <int MB, int CG, int ACT>
__global__ __launch_bounds__(64 * kRcWaves) void linear_act_rows_kernel(LinearParams p, RowsArgs r) {
  typedef RowsProduct<MB, CG, false> Product;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Product::LDS];
  Product t;
  t.run(r, lds);
  if (!t.mine) return;
  f32x4 v = t.sum[0];
  if (p.bias) {
    f32x4 b[1];
    linear_bias(p, b, [&](int) { return t.n; });
    v += b[0];
  }
  if (p.saved) saved_store4(p.saved + ((int64_t)(t.m >> 5) * ((r.N + 31) >> 5) + (t.n >> 5)) * kSavedBlock, t.m, t.n, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = act_value<ACT>(v[e]);
  if (p.residual) {
    const u32x2 b = ldg8(p.residual + t.m * p.rs + t.n);
    v += f32x4{lo_bf16(b[0]), hi_bf16(b[0]), lo_bf16(b[1]), hi_bf16(b[1])};
  }
  stg8(p.y + t.m * p.ys + t.n, u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
}

template <int CG, int ACT>
static void linear_act_rows_launch(const LinearParams& p, hipStream_t s) {
  const RowsArgs r{p.g.x, p.g.w0, nullptr, p.g.xs, p.g.ws0, 0, p.g.M, p.g.N, p.g.K};
  const dim3 grid((unsigned)((r.N + CG - 1) / CG)), wg(64 * kRcWaves);
  if (r.M <= 16) linear_act_rows_kernel<1, CG, ACT><<<grid, wg, 0, s>>>(p, r);
  else if (r.M <= 32) linear_act_rows_kernel<2, CG, ACT><<<grid, wg, 0, s>>>(p, r);
  else linear_act_rows_kernel<4, CG, ACT><<<grid, wg, 0, s>>>(p, r);
}
template <int ACT>
static void linear_act_rows_go(const LinearParams& p, hipStream_t s) {
  if (rows_columns(p.g.N) == 16) linear_act_rows_launch<16, ACT>(p, s);
  else linear_act_rows_launch<32, ACT>(p, s);
}

template <class C, int ACT>
static void linear_act_go(const LinearParams& p, hipStream_t s) {
  linear_act_kernel<C, ACT><<<dim3(gemm_grid<C>(p.g)), dim3(C::THREADS), 0, s>>>(p);
  if (p.g.S > 1) linear_act_finish_kernel<C, ACT><<<dim3(gemm_finish_grid<C>(p.g)), dim3(C::THREADS), 0, s>>>(p);
}

// dx is a product without an epilogue of its own
template <class C>
static void linear_act_launch(const LinearParams& p, int act, hipStream_t s) {
  if constexpr (!C::KMAJOR) {
    if (act == MLA_ACT_RELU) return linear_act_go<C, MLA_ACT_RELU>(p, s);
    if (act == MLA_ACT_SILU) return linear_act_go<C, MLA_ACT_SILU>(p, s);
    if (act == MLA_ACT_GELU_TANH) return linear_act_go<C, MLA_ACT_GELU_TANH>(p, s);
  }
  linear_act_go<C, MLA_ACT_NONE>(p, s);
}

template <bool KMAJOR>
static int linear_tiles(const char* op, LinearParams& p, int act, void* workspace, size_t bytes, hipStream_t s) {
  const GemmPlan pl = gemm_plan(p.g.M, p.g.N, p.g.K, p.g.parts);
  MLA_TRY(gemm_apply(op, p.g, pl, workspace, bytes));
  if (pl.tile == kGemmLarge) linear_act_launch<GemmCfg<256, 256, 2, 4, KMAJOR, false>>(p, act, s);
  else if (pl.tile == kGemmHalf) linear_act_launch<GemmCfg<256, 128, 2, 4, KMAJOR, false>>(p, act, s);
  else linear_act_launch<GemmCfg<128, 128, 2, 2, KMAJOR, false>>(p, act, s);
  return launch_status(op);
}

static int linear_act_check(const mla_linear_act_args* a) {
  const char* op = "mla_linear_act";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_TRY(check_linear_sizes(op, a->M, a->N, a->K));
  MLA_CHECK(a->activation >= MLA_ACT_NONE && a->activation <= MLA_ACT_GELU_TANH, MLA_ERR_UNSUPPORTED,
            "%s: activation %d", op, a->activation);
  if (a->M == 0 || a->N == 0) return MLA_OK;
  MLA_TRY(check_rows(op, "x", a->x, a->K, a->x_stride));
  MLA_TRY(check_rows(op, "w", a->w, a->K, a->w_stride));
  MLA_TRY(check_rows(op, "y", a->y, a->N, a->y_stride));
  if (a->bias) {
    MLA_CHECK(a->bias_dtype == MLA_DTYPE_BF16 || a->bias_dtype == MLA_DTYPE_F32, MLA_ERR_UNSUPPORTED, "%s: bias dtype", op);
    const uintptr_t at = a->bias_dtype == MLA_DTYPE_F32 ? 16 : 8;
    MLA_CHECK((uintptr_t)a->bias % at == 0, MLA_ERR_INVALID_ARG, "%s: bias must be %d-byte aligned", op, (int)at);
  }
  if (a->residual) MLA_TRY(check_rows(op, "residual", a->residual, a->residual_stride ? a->N : 0, a->residual_stride));
  MLA_CHECK(((uintptr_t)a->saved & 15) == 0, MLA_ERR_INVALID_ARG, "%s: saved must be 16-byte aligned", op);
  return MLA_OK;
}

static int linear_dx_check(const mla_linear_dx_args* a) {
  const char* op = "mla_linear_dx";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_TRY(check_linear_sizes(op, a->M, a->N, a->K));
  if (a->M == 0 || a->K == 0) return MLA_OK;
  const int64_t parts = a->w1 ? 2 : 1;
  MLA_TRY(check_rows(op, "dy", a->dy, parts * a->N, a->dy_stride));
  MLA_TRY(check_rows(op, "w0", a->w0, a->K, a->w0_stride));
  MLA_TRY(check_rows(op, "dx", a->dx, a->K, a->dx_stride));
  MLA_TRY(check_weight_reach(op, "w0", a->N, a->w0_stride));
  if (a->w1) {
    MLA_TRY(check_rows(op, "w1", a->w1, a->K, a->w1_stride));
    MLA_CHECK(a->w1_stride == a->w0_stride, MLA_ERR_UNSUPPORTED, "%s: the weights' row strides must be the same", op);
  }
  return MLA_OK;
}

}  // namespace mla

using namespace mla;

extern "C" size_t mla_linear_saved_size(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || M >= kLinearMaxM || N >= kLinearMaxN) return 0;
  return (size_t)((M + 31) / 32) * (size_t)((N + 31) / 32) * kSavedBlock;
}

extern "C" size_t mla_linear_act_workspace_bytes(const mla_linear_act_args* a) {
  // 0 for the sizes mla_linear_act rejects
  if (!a || check_linear_sizes("mla_linear_act", a->M, a->N, a->K) != MLA_OK || a->M <= kRcMaxRows) return 0;
  return (size_t)gemm_plan(a->M, a->N, a->K, 1).part_bytes;
}

extern "C" int mla_linear_act(const mla_linear_act_args* a, void* stream) {
  const char* op = "mla_linear_act";
  MLA_TRY(linear_act_check(a));
  if (a->M == 0 || a->N == 0) return MLA_OK;
  LinearParams p{};
  p.g.x = (const bf16*)a->x, p.g.w0 = (const bf16*)a->w;
  p.g.xs = a->x_stride, p.g.ws0 = a->w_stride;
  p.g.M = (int)a->M, p.g.N = (int)a->N, p.g.K = (int)a->K, p.g.parts = 1;
  p.bias = a->bias;
  p.bias_f32 = a->bias_dtype == MLA_DTYPE_F32;
  p.residual = (const bf16*)a->residual;
  p.y = (bf16*)a->y;
  p.saved = (unsigned char*)a->saved;
  p.rs = a->residual_stride;
  p.ys = a->y_stride;
  hipStream_t s = (hipStream_t)stream;
  if (a->M > kRcMaxRows) return linear_tiles<false>(op, p, a->activation, a->workspace, a->workspace_bytes, s);
  if (a->activation == MLA_ACT_RELU) linear_act_rows_go<MLA_ACT_RELU>(p, s);
  else if (a->activation == MLA_ACT_SILU) linear_act_rows_go<MLA_ACT_SILU>(p, s);
  else if (a->activation == MLA_ACT_GELU_TANH) linear_act_rows_go<MLA_ACT_GELU_TANH>(p, s);
  else linear_act_rows_go<MLA_ACT_NONE>(p, s);
  return launch_status(op);
}

extern "C" size_t mla_linear_dx_workspace_bytes(const mla_linear_dx_args* a) {
  // 0 for the sizes mla_linear_dx rejects
  if (!a || check_linear_sizes("mla_linear_dx", a->M, a->N, a->K) != MLA_OK) return 0;
  return (size_t)gemm_plan(a->M, a->K, a->N, a->w1 ? 2 : 1).part_bytes;
}

extern "C" int mla_linear_dx(const mla_linear_dx_args* a, void* stream) {
  MLA_TRY(linear_dx_check(a));
  if (a->M == 0) return MLA_OK;
  LinearParams p{};
  p.g.x = (const bf16*)a->dy, p.g.w0 = (const bf16*)a->w0, p.g.w1 = (const bf16*)a->w1;
  p.g.xs = a->dy_stride, p.g.ws0 = a->w0_stride, p.g.ws1 = a->w1_stride;
  p.g.M = (int)a->M, p.g.N = (int)a->K, p.g.K = (int)a->N, p.g.parts = a->w1 ? 2 : 1;
  p.y = (bf16*)a->dx;
  p.ys = a->dx_stride;
  return linear_tiles<true>("mla_linear_dx", p, MLA_ACT_NONE, a->workspace, a->workspace_bytes, (hipStream_t)stream);
}
