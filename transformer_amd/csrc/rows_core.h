// A few rows of x against a weight (a token of each sequence of a batch): bound by reading the weight once.
//
// A workgroup of eight waves takes CG columns of the weight, or of each of two weights, over all of k, in chunks of 256.  A chunk
// of the CG weight rows and of all x rows (512 contiguous bytes of each) comes by direct-to-LDS loads into a ring that keeps up to
// 144 KiB of a CU's reads in flight; wave w multiplies k 32 w .. 32 w + 31 of it (v_mfma_f32_16x16x32_bf16), and the waves' sums
// are added through LDS in wave order.  Calls in a row, us (fragments straight from memory, 16 rows x 64 bytes an
// instruction, in brackets): one row against 2 x 4608 x 1792 7.6 (10.3), 4.4 TB/s; 32 against 2 x 4608 x 2048 9.4 (18.0), 4.0
// TB/s; 64 against 2 x 4608 x 1792 10.7 (22); one against 1792 x 4608 7.0 (7.3), 32 against 2048 x 4608 9.2 (14.3): 112 and 128
// workgroups, whose chunks follow each other at the latency of the ring.
// mla_linear_rows is the framework's other product of few rows: over groups, K a multiple of 128 up to 4096, no epilogue.  Against
// it (replayed graphs, us, linear_rows in brackets) 1 row of 4608 x 1792 6.3 (6.1), 16 rows 6.4 (8.3), 64 rows 8.3 (22); 1 row of 9216
// x 2048 14.2 (11.1), 32 rows 16.2 (20.6); 2048 x 2048 5.3 (4.7), 5.5 (6.1), 7.5 (8.8).  The decode step keeps linear_rows (one of
// its launches holds the RoPE append too); what has an epilogue or another K runs here.
//
// A staged row's chunk c of 16 bytes lies at c ^ (row mod 16): the 16 rows of a fragment fall on different banks.
#pragma once

#include "act.h"
#include "gemm_core.h"

namespace mla {

constexpr int kRcWaves = 8, kRcMaxRows = 64, kRcK = 256;

struct RowsArgs {
  const bf16 *x, *w0, *w1;
  int64_t xs, ws0, ws1;
  int M, N, K;
};

// MB blocks of 16 rows (M <= 16 MB); CG columns: 16 or 32
template <int MB, int CG, bool PAIR>
struct RowsProduct {
  static constexpr int NW = PAIR ? 2 : 1, CB = CG / 16;           // weights; blocks of 16 of their columns
  static constexpr int WROWS = NW * CG, ROWS = WROWS + 16 * MB;   // staged rows
  static constexpr int SLOT = ROWS * 2 * kRcK;
  static constexpr int FIT = 144 * 1024 / SLOT, RING = FIT < 8 ? FIT : 8;
  static constexpr int LOADS = ROWS / 2 / kRcWaves;               // of a wave per chunk, two rows each: CB per weight, MB of x
  static constexpr int BLOCKS = NW * CB * MB;                         // 16 x 16 products of a wave
  static constexpr int RED = kRcWaves * BLOCKS * 1024;
  static constexpr int LDS = RING * SLOT > RED ? RING * SLOT : RED;
  static_assert(RING >= 2 && LDS <= 160 * 1024 && (RING - 1) * LOADS <= 63 && CB * MB <= kRcWaves, "a workgroup's shape");
  f32x4 sum[NW];  // of rows m, columns n .. n + 3, where `mine`
  int m, n;
  bool mine;

  __device__ __forceinline__ void run(const RowsArgs& p, unsigned char* lds) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, q = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * CG, nv = min(CG, p.N - n0);
    // rows past the last valid one and k past the end are not loaded (the descriptors are made in scalar registers: see GemmSpan)
    const buf_rsrc rx = gemm_span(p.x, rows_bytes(p.M, p.xs, p.K * 2)).rsrc();
    const buf_rsrc r0 = gemm_span(p.w0 + (int64_t)n0 * p.ws0, rows_bytes(nv, p.ws0, p.K * 2)).rsrc();
    const buf_rsrc r1 = PAIR ? gemm_span(p.w1 + (int64_t)n0 * p.ws1, rows_bytes(nv, p.ws1, p.K * 2)).rsrc() : r0;
    const uint32_t lds0 = lds_addr(lds);
    const int chunks = (p.K + kRcK - 1) / kRcK;
    uint32_t off[LOADS];  // this lane's bytes in each of the wave's loads, at k = 0
    int at[LOADS];        // its chunk of 16 bytes within a row's 512
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {  // load j of every wave has the same source: CB of w0, CB of w1, MB of x
      const int row = 2 * (w + kRcWaves * j) + (lane >> 5), base = j < CB ? 0 : j < NW * CB ? CG : WROWS;
      at[j] = (lane & 31) ^ (row & 15);
      off[j] = (uint32_t)((row - base) * (j < CB ? p.ws0 : j < NW * CB ? p.ws1 : p.xs) * 2) + 16u * (uint32_t)at[j];
    }
    auto issue = [&](int c, int slot) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        dma16(j < CB ? r0 : j < NW * CB ? r1 : rx, kRcK * c + 8 * at[j] < p.K ? off[j] + (uint32_t)(c * 2 * kRcK) : 0x80000000u,
              (uint32_t)__builtin_amdgcn_readfirstlane((int)lds0 + slot * SLOT + (w + kRcWaves * j) * 1024));
    };
    f32x4 acc[NW][CB][MB];
#pragma unroll
    for (int a = 0; a < NW; ++a)
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[a][b][i] = f32x4{};
#pragma unroll
    for (int c = 0; c + 1 < RING; ++c) issue(c, c);
    const int ch = 4 * w + q;  // this lane's chunk of a staged row
    for (int c = 0, slot = 0; c < chunks; ++c) {
      // chunk c has landed when only the RING - 2 behind it are in flight; past the barrier every wave has read chunk c - 1
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * LOADS) : "memory");
      __syncthreads();
      issue(c + RING - 1, slot == 0 ? RING - 1 : slot - 1);
      const int k0 = kRcK * c + 32 * w;
      if (k0 < p.K) {  // (wave-uniform)
        const unsigned char* st = lds + slot * SLOT;
        const bool in = k0 + 8 * q < p.K;  // k is whole chunks: the lane's 8 are in or out together
        const u32x4 z{0u, 0u, 0u, 0u};
        bf16x8 fw[NW][CB], fx[MB];
#pragma unroll
        for (int a = 0; a < NW; ++a)
#pragma unroll
          for (int b = 0; b < CB; ++b) {
            const int row = a * CG + 16 * b + l16;
            const u32x4 v = lds16(st + row * 512 + ((ch ^ (row & 15)) * 16));
            fw[a][b] = as_bf16x8(in ? v : z);
          }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const int row = WROWS + 16 * i + l16;
          const u32x4 v = lds16(st + row * 512 + ((ch ^ (row & 15)) * 16));
          fx[i] = as_bf16x8(in ? v : z);
        }
#pragma unroll
        for (int a = 0; a < NW; ++a)
#pragma unroll
          for (int b = 0; b < CB; ++b)
#pragma unroll
            for (int i = 0; i < MB; ++i) acc[a][b][i] = mfma16(fw[a][b], fx[i], acc[a][b][i]);
      }
      slot = slot + 1 == RING ? 0 : slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (no load lands in what follows)
    __syncthreads();
    f32x4* const red = reinterpret_cast<f32x4*>(lds) + lane;
#pragma unroll
    for (int a = 0; a < NW; ++a)
#pragma unroll
      for (int b = 0; b < CB; ++b)
#pragma unroll
        for (int i = 0; i < MB; ++i) red[(w * BLOCKS + (a * CB + b) * MB + i) * 64] = acc[a][b][i];
    __syncthreads();
    mine = false;
    if (w >= CB * MB) return;
    const int b = w / MB, i = w % MB;
#pragma unroll
    for (int a = 0; a < NW; ++a) {
      sum[a] = red[((a * CB + b) * MB + i) * 64];
#pragma unroll
      for (int v = 1; v < kRcWaves; ++v) sum[a] += red[(v * BLOCKS + (a * CB + b) * MB + i) * 64];
    }
    m = 16 * i + l16;
    n = n0 + 16 * b + 4 * q;
    mine = m < p.M && 16 * b + 4 * q < nv;
  }
};

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
