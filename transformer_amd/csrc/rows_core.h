// A few rows of x against a weight (a token of each sequence of a batch): bound by reading the weight once.
//
// A workgroup of eight waves takes CG (16 or 8) columns, or CG of each of two weights, over all of k: wave w the steps of 64 k
// w, w + 8, ..., so that the eight read 1 KiB of every weight row at a time.  Fragments go from memory straight into registers
// (v_mfma_f32_16x16x32_bf16: lane l takes row l % 16 and chunk l / 16 of 8 k; the two halves of a step make whole 128-byte
// lines), several steps ahead of their products: 64 to 128 KiB of a CU's reads are in flight.  The waves' sums are added
// through LDS in wave order.
#pragma once

#include "act.h"

namespace mla {

constexpr int kRcWaves = 8, kRcMaxRows = 64;

struct RowsArgs {
  const bf16 *x, *w0, *w1;
  int64_t xs, ws0, ws1;
  int M, N, K;
  int cg;  // columns of a workgroup
};

// MB blocks of 16 rows (M <= 16 MB).  On return wave i < MB holds rows 16 i + l % 16 of both products, columns
// n0 + 4 (l / 16) + [0, 4), and `mine` says whether the lane's are to be stored; the other waves hold nothing.
template <int MB, bool PAIR>
struct RowsProduct {
  static constexpr int NW = PAIR ? 2 : 1;
  static constexpr int BATCH = MB <= 2 ? 4 : 2;  // steps whose fragments are loaded together
  f32x4 sum[NW];
  int m, n;
  bool mine;

  __device__ __forceinline__ void run(const RowsArgs& p, f32x4 (*red)[MB * NW][64]) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * p.cg, nv = min(p.cg, p.N - n0);
    // rows past the last valid one read it again; k past the end reads past the descriptor, which gives zeros
    const buf_rsrc rx = make_rsrc(p.x, rows_bytes(p.M, p.xs, p.K * 2));
    const buf_rsrc r0 = make_rsrc(p.w0 + (int64_t)n0 * p.ws0, rows_bytes(nv, p.ws0, p.K * 2));
    const buf_rsrc r1 = PAIR ? make_rsrc(p.w1 + (int64_t)n0 * p.ws1, rows_bytes(nv, p.ws1, p.K * 2)) : r0;
    const int wr = min(l16 & (p.cg - 1), nv - 1);
    const uint32_t wo0 = (uint32_t)(wr * p.ws0 * 2), wo1 = PAIR ? (uint32_t)(wr * p.ws1 * 2) : 0u;
    uint32_t xo[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) xo[i] = (uint32_t)(min(16 * i + l16, p.M - 1) * p.xs * 2);
    struct Step {
      u32x4 w[NW][2], x[MB][2];
    };
    auto load = [&](int t, Step& s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = 8 * t + 4 * h + q;
        const bool in = 8 * c < p.K;
        const uint32_t at = 16u * (uint32_t)c, out = 0x80000000u;
        s.w[0][h] = bld16(r0, in ? wo0 + at : out);
        if (PAIR) s.w[NW - 1][h] = bld16(r1, in ? wo1 + at : out);
#pragma unroll
        for (int i = 0; i < MB; ++i) s.x[i][h] = bld16(rx, in ? xo[i] + at : out);
      }
    };
    f32x4 acc[NW][MB];
#pragma unroll
    for (int a = 0; a < NW; ++a)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[a][i] = f32x4{};
    const int steps = (p.K + 63) / 64;
    Step s[2][BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) load(w + kRcWaves * b, s[0][b]);  // (steps past the last load nothing and add zeros)
    auto batch = [&](int t, Step (&now)[BATCH], Step (&next)[BATCH]) {
      if (t + kRcWaves * BATCH < steps) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) load(t + kRcWaves * (BATCH + b), next[b]);
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int a = 0; a < NW; ++a)
#pragma unroll
            for (int i = 0; i < MB; ++i) acc[a][i] = mfma16(as_bf16x8(now[b].w[a][h]), as_bf16x8(now[b].x[i][h]), acc[a][i]);
    };
    for (int t = w; t < steps; t += 2 * kRcWaves * BATCH) {
      batch(t, s[0], s[1]);
      if (t + kRcWaves * BATCH < steps) batch(t + kRcWaves * BATCH, s[1], s[0]);
    }
#pragma unroll
    for (int a = 0; a < NW; ++a)
#pragma unroll
      for (int i = 0; i < MB; ++i) red[w][a * MB + i][lane] = acc[a][i];
    __syncthreads();
    mine = false;
    if (w >= MB) return;
#pragma unroll
    for (int a = 0; a < NW; ++a) {
      sum[a] = red[0][a * MB + w][lane];
#pragma unroll
      for (int v = 1; v < kRcWaves; ++v) sum[a] += red[v][a * MB + w][lane];
    }
    m = 16 * w + l16;
    n = n0 + 4 * q;
    mine = m < p.M && 4 * q < nv;
  }
};

// columns of a workgroup: 16, or 8 (half of the products go unused) where 16 would leave CUs without one
inline int rows_columns(int64_t N) { return N / 16 < 200 ? 8 : 16; }

// the 4 consecutive n that a lane holds, in the layout of act.h's blocks
__device__ __forceinline__ void saved_store4(unsigned char* block, int m, int n, const f32x4& v) {
  const int lane = 32 * ((n >> 2) & 1) + (m & 31), e = 4 * ((n & 31) >> 3);
  uint32_t b[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(v[k]);
  stg8(block + (e >> 3) * 1024 + lane * 16 + (e & 7) * 2,
       u32x2{(b[0] >> 16) | (b[1] & 0xffff0000u), (b[2] >> 16) | (b[3] & 0xffff0000u)});
  *(uint32_t*)(block + 2048 + lane * 16 + e) =
      ((b[0] >> 8) & 255u) | (b[1] & 0xff00u) | ((b[2] << 8) & 0xff0000u) | ((b[3] << 16) & 0xff000000u);
}

}  // namespace mla
