// What the epilogues of gemm_core.h's tiles share: outputs leave through LDS, so that memory sees whole row segments.
//
// An accumulator quad is 4 consecutive n of one row m (8 bytes in bf16); stored straight, an instruction would touch 32 rows
// with 16 bytes each.  A pass writes quads to rows of COLS columns in the two slots that the tile read last and stores 16
// bytes a lane from there.  Chunk c of 16 bytes of row r lies at c ^ (r mod chunks): the 32 rows of a wave's quads then fall
// on different banks.
#pragma once

#include "act.h"
#include "gemm_core.h"

namespace mla {

// A thread's place in the workgroup, made anew for each epilogue: what derives from it would otherwise be formed before the
// loop over tiles and kept in registers that the products need.
template <class C>
struct WavePos {
  int tid, lane, wn, wm, l32, hk;
  __device__ __forceinline__ WavePos() {
    tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    wn = w % C::WN;
    wm = w / C::WN;
    l32 = lane & 31;
    hk = lane >> 5;
  }
};

template <class C, int COLS>
struct StagedRows {
  static constexpr int RB = COLS * 2, CH = COLS / 8, PER = C::XSLOT / RB;  // bytes and chunks of a row, rows of the first slot
  unsigned char *s0, *s1;
  __device__ __forceinline__ unsigned char* at(int r, int chunk) const {
    unsigned char* row = r < PER ? s0 + r * RB : s1 + (r - PER) * RB;
    return row + ((chunk ^ (r & (CH - 1))) * 16);
  }
};

// Rows of pass j: staged row r holds row m0 + 32 (XJ (r / 32) + j) + r % 32 of the output (one 32-row block of every wave row)
template <class C>
__device__ __forceinline__ int pass_row(int r, int j) {
  return 32 * (C::XJ * (r >> 5) + j) + (r & 31);
}

// The staged rows [0, R) to out (at the tile's first row and column): rows below mv, columns below nv (a multiple of 8)
template <class C, int COLS, class RowOf>
__device__ __forceinline__ void store_rows(const StagedRows<C, COLS>& st, int tid, int R, bf16* out, int64_t stride, int mv, int nv,
                                           RowOf&& row_of) {
  constexpr int CH = COLS / 8;
#pragma unroll 4
  for (int c = tid; c < R * CH; c += C::THREADS) {
    const int r = c / CH, ch = c % CH, m = row_of(r);
    if (m < mv && 8 * ch < nv) stg16(out + m * stride + 8 * ch, lds16(st.at(r, ch)));
  }
}

}  // namespace mla
