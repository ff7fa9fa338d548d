// The gradient of a linear layer's epilogue (gfx950): dz = bf16(dy act'(z)) from the z that the forward kept (rounded because the
// products that follow take bf16 operands), and the bias gradient db = sum over rows of dy act'(z), of the fp32 values, in one
// pass over dy.  HBM bound: 2 + 3 bytes read and 2 written per element.
//
// A wave owns 32 columns and walks 32-row blocks, a lane one row's four quads of a block, as z was kept (act.h).  A lane
// adds its rows' gradients in fp32; at the end the 32 lanes of a column are added and the segment's sum stored.  A second
// kernel adds the segments in order: no atomics, results repeat bit for bit.  Up to 128 rows are one segment, whose sums are db
// (four blocks in a row take less than a second launch).  12288 x 4608 with db: 79 us, 5.0 TB/s, and 5 us for the segments.
#include <algorithm>

#include "act.h"
#include "linear_checks.h"

namespace mla {

struct ActGradParams {
  const bf16* dy;
  const unsigned char* saved;
  bf16* dz;
  float* part;  // [segments][N]; null for one segment
  void* db;
  int M, N, seg;  // 32-row blocks of a segment
  int n_seg, db_f32;
  int64_t dys, dzs;
};

__device__ __forceinline__ void act_grad_store(const ActGradParams& p, int n, float v) {
  if (p.db_f32) ((float*)p.db)[n] = v;
  else ((bf16*)p.db)[n] = (bf16)v;
}

constexpr int kAgCols = 128;  // columns of a workgroup, 32 a wave

// dy arrives and dz leaves in rows of 256 bytes through an LDS tile of 32 rows (a lane's quads straight from memory would be
// 16 bytes of each of 32 rows an instruction: 2.5 TB/s); chunk c of 16 bytes of row r lies at c ^ (r mod 16), which spreads a
// quad's 32 rows over the banks.  The next tile's loads are in flight under this one's arithmetic.
template <int ACT>
__global__ __launch_bounds__(256) void act_grad_kernel(ActGradParams p) {
  __shared__ __attribute__((aligned(16))) unsigned char tile[32 * 256];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hk = lane >> 5, w = tid >> 6;
  const int n0 = blockIdx.x * kAgCols, wn = n0 + 32 * w;
  const int64_t hb = (p.N + 31) >> 5;
  const int b0 = blockIdx.y * p.seg, b1 = min(b0 + p.seg, (p.M + 31) >> 5);
  // this thread's two chunks of a tile: rows tid / 16 and 16 more, chunk tid % 16 (N is whole chunks)
  const int cr = tid >> 4, cc = tid & 15;
  const bool col = n0 + 8 * cc < p.N;
  unsigned char* const mine[2] = {tile + cr * 256 + ((cc ^ cr) * 16), tile + (cr + 16) * 256 + ((cc ^ cr) * 16)};
  const bool live = wn < p.N;  // (wave-uniform) the wave's columns exist
  u32x4 d[2];
  SavedRegs z{};
  auto load = [&](int b) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = 32 * b + cr + 16 * e;
      d[e] = col && m < p.M ? ldg16(p.dy + (int64_t)m * p.dys + n0 + 8 * cc) : u32x4{0u, 0u, 0u, 0u};
    }
    if (ACT != MLA_ACT_NONE && live) z = saved_load(p.saved + (b * hb + (wn >> 5)) * kSavedBlock, lane);
  };
  float sum[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum[e] = 0.f;
  load(b0);
  for (int b = b0; b < b1; ++b) {
    sts16(mine[0], d[0]);
    sts16(mine[1], d[1]);
    const SavedRegs zb = z;
    __syncthreads();
    if (b + 1 < b1) load(b + 1);
    const bool row = 32 * b + l32 < p.M;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      unsigned char* at = tile + l32 * 256 + (((4 * w + q) ^ (l32 & 15)) * 16) + 8 * hk;
      const u32x2 x = lds8(at);
      float v[4] = {lo_bf16(x[0]), hi_bf16(x[0]), lo_bf16(x[1]), hi_bf16(x[1])};
      if (ACT != MLA_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float value, slope;
          act_both<ACT>(saved_value(zb, 4 * q + e), value, slope);
          v[e] *= slope;
        }
        sts8(at, u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])});
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[4 * q + e] += row ? v[e] : 0.f;  // (what z holds past the last row may be NaN)
    }
    __syncthreads();
    if (ACT != MLA_ACT_NONE) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int m = 32 * b + cr + 16 * e;
        if (col && m < p.M) stg16(p.dz + (int64_t)m * p.dzs + n0 + 8 * cc, lds16(mine[e]));
      }
    }
  }
  if (!p.db || !live) return;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) sum[e] += wave_shfl_xor(sum[e], s);
  }
  if (l32 == 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = wn + 8 * q + 4 * hk;
      if (n >= p.N) continue;
      const f32x4 v{sum[4 * q], sum[4 * q + 1], sum[4 * q + 2], sum[4 * q + 3]};
      if (p.part) {
        stg16(p.part + (int64_t)blockIdx.y * p.N + n, __builtin_bit_cast(u32x4, v));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) act_grad_store(p, n + e, v[e]);
      }
    }
  }
}

__global__ __launch_bounds__(64) void act_grad_sum_kernel(ActGradParams p) {
  const int n = blockIdx.x * 64 + threadIdx.x;
  if (n >= p.N) return;
  float sum = 0.f;
  for (int s0 = 0; s0 < p.n_seg; s0 += 16) {
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = p.part[(int64_t)min(s0 + e, p.n_seg - 1) * p.N + n];
#pragma unroll
    for (int e = 0; e < 16; ++e) sum += s0 + e < p.n_seg ? v[e] : 0.f;
  }
  act_grad_store(p, n, sum);
}

// segments of rows so that some 2048 workgroups of four waves share the pass; up to four blocks are one
static void act_grad_segments(int64_t M, int64_t N, int& seg, int& n_seg) {
  const int64_t blocks = (M + 31) / 32, strips = (N + kAgCols - 1) / kAgCols;
  const int64_t want = blocks <= 4 ? 1 : std::min(blocks, std::max<int64_t>(1, 2048 / strips));
  seg = (int)((blocks + want - 1) / want);
  n_seg = (int)((blocks + seg - 1) / seg);
}

}  // namespace mla

using namespace mla;

extern "C" size_t mla_act_grad_workspace_bytes(const mla_act_grad_args* a) {
  if (!a || a->M <= 0 || a->N <= 0 || a->M >= kLinearMaxM || a->N >= kLinearMaxN || !a->db) return 0;
  int seg, n_seg;
  act_grad_segments(a->M, a->N, seg, n_seg);
  return n_seg == 1 ? 0 : (size_t)n_seg * (size_t)a->N * 4;
}

extern "C" int mla_act_grad(const mla_act_grad_args* a, void* stream) {
  const char* op = "mla_act_grad";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_TRY(check_linear_sizes(op, a->M, a->N, 8));
  MLA_CHECK(a->activation >= MLA_ACT_NONE && a->activation <= MLA_ACT_GELU_TANH, MLA_ERR_UNSUPPORTED, "%s: activation %d", op,
            a->activation);
  const bool act = a->activation != MLA_ACT_NONE;
  MLA_CHECK(a->M > 0, MLA_ERR_INVALID_ARG, "%s: M = 0", op);
  MLA_TRY(check_rows(op, "dy", a->dy, a->N, a->dy_stride));
  if (act) {
    MLA_TRY(check_rows(op, "dz", a->dz, a->N, a->dz_stride));
    MLA_CHECK(a->saved && ((uintptr_t)a->saved & 15) == 0, MLA_ERR_INVALID_ARG, "%s: saved must be given, 16-byte aligned", op);
  }
  if (a->db) {
    MLA_CHECK(a->db_dtype == MLA_DTYPE_F32 || a->db_dtype == MLA_DTYPE_BF16, MLA_ERR_UNSUPPORTED, "%s: db dtype", op);
    MLA_CHECK(((uintptr_t)a->db & 3) == 0, MLA_ERR_INVALID_ARG, "%s: db must be 4-byte aligned", op);
    const size_t need = mla_act_grad_workspace_bytes(a);
    MLA_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace & 15) == 0), MLA_ERR_WORKSPACE,
              "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", op, need, a->workspace_bytes);
  }
  if (!act && !a->db) return MLA_OK;
  ActGradParams p{(const bf16*)a->dy, (const unsigned char*)a->saved, (bf16*)a->dz, nullptr, a->db,
                  (int)a->M, (int)a->N, 0, 0, a->db_dtype == MLA_DTYPE_F32, a->dy_stride, a->dz_stride};
  act_grad_segments(a->M, a->N, p.seg, p.n_seg);
  if (a->db && p.n_seg > 1) p.part = (float*)a->workspace;
  const dim3 grid((unsigned)((a->N + kAgCols - 1) / kAgCols), (unsigned)p.n_seg);
  hipStream_t s = (hipStream_t)stream;
  if (a->activation == MLA_ACT_RELU) act_grad_kernel<MLA_ACT_RELU><<<grid, 256, 0, s>>>(p);
  else if (a->activation == MLA_ACT_SILU) act_grad_kernel<MLA_ACT_SILU><<<grid, 256, 0, s>>>(p);
  else if (a->activation == MLA_ACT_GELU_TANH) act_grad_kernel<MLA_ACT_GELU_TANH><<<grid, 256, 0, s>>>(p);
  else act_grad_kernel<MLA_ACT_NONE><<<grid, 256, 0, s>>>(p);
  MLA_TRY(launch_status(op));
  if (p.part) {
    act_grad_sum_kernel<<<dim3((unsigned)((a->N + 63) / 64)), 64, 0, s>>>(p);
    MLA_TRY(launch_status(op));
  }
  return MLA_OK;
}
