// The tile product that the linear layers' kernels share (linear_act.hip, gated_linear.hip): C^T [n][m] = W . x^T over k, bf16
// operands, fp32 sums, on v_mfma_f32_32x32x16_bf16.  x [M][K] has k contiguous; W either has too (rows of a layer's weight:
// y = x W^T) or has n contiguous (the same weight read from its other side: dx = dy W), in which case its fragments come by
// transpose reads.
//
// A workgroup of WN x WM waves computes tiles of TM x TW outputs, one after the other, k in stages of 64.  A stage is a slot of
// x's TM rows x 64 k and one of W's TW, filled by direct-to-LDS loads.  Square tiles use one ring of five slots (three stages of
// 256 x 256 do not fit the LDS): when the first step of a stage has read the rest of its x, that slot takes W of the stage after
// next, and W's, read at the end, x of the one behind it.  Tiles of 256 x 128 use a ring of three for each, filled two stages
// ahead with one barrier a stage.  The loads run on across the end of a tile, so that the next tile's first stage lands under
// this tile's last products and its epilogue, which has the two slots last read for its own use.  Loads past the last tile have
// empty descriptors.
//
// A staged row of 64 k (128 bytes: pieces of 64 bytes reach half the rate, 60 against 95-130 bytes/ns per CU measured) holds
// its chunk c of 16 bytes at c ^ ((row / 2) mod 8), so that 16 rows x one chunk are free of bank conflicts; a staged k row of TW
// n holds chunk c at c ^ 4 (row mod 4), so that the four rows of a half-wave's transpose read fall on four different 64-byte bank
// groups.  A step's products run under the reads of the next one, the last step's under the next stage's first.
//
// What bounds it: a stage of 256 x 256 takes 0.86 us of matrix instructions, 0.96 with its LDS reads, and with random operands on
// all 256 CUs 1.31 us (1640 TFLOP/s: the clock that power allows), 1.4 to 1.6 us as loads come from beyond the L2.  Smaller
// tiles read more LDS and load more for their products: 1.05 us a stage for two workgroups of 128 x 128 on a CU, 1.04 for one of
// 256 x 128 (half the outputs of 1.57); they win where the large ones leave CUs idle (gemm_plan in plans.h).  Operands that lie
// in HBM and not in the last-level cache add 10 to 40 us where a product has one round of tiles (3001 x 2048 over 5464: 88 and
// 129 us).  Whole products, 12288 rows, in a training pass: 4608 -> 1792 194 us (1050 TFLOP/s), 2 x 4608 <- 1792 361 us (1120);
// 8192 cubed 840 us (1310; the library 775).
// Measured and not kept, for a tile of 128 x 128 alone on its CU (50 us at 1999 x 2048 over 4608; its LDS traffic, 64 KiB read and
// 32 written a stage, is 0.42 us of the 0.55 a stage takes): nine slots and eight waves (the same there, slower at larger sizes),
// whole stages read ahead into a second set of registers over rings of five (53), two groups of waves that share its k (51; 5 us
// less with the operands in HBM, 1 to 2 more at short k).  For 256 x 128, four waves of 128 x 64 (3 to 10 % slower).  For 256 x
// 256, four waves of 128 x 128 (they spill; 907 against 840 at 8192 cubed).  Waves of their own for loads and for stores (2 %),
// stores past the caches for y (1 %).
#pragma once

#include <type_traits>

#include "mla_common.h"

namespace mla {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

// TM x TW outputs of WN x WM waves; KMAJOR: W is [k][n]; PAIR: a tile's W rows come from two weights of N columns each, TW / 2
// of each, a wave's first NB / 2 blocks from w0, the rest from w1 at the same columns
template <int TM_, int TW_, int WN_, int WM_, bool KMAJOR_, bool PAIR_>
struct GemmCfg {
  static constexpr int TM = TM_, TW = TW_, WN = WN_, WM = WM_, BK = 64, HS = BK / 16;
  static constexpr bool KMAJOR = KMAJOR_, PAIR = PAIR_;
  static constexpr int WAVES = WN * WM, THREADS = 64 * WAVES;
  static constexpr int NB = TW / WN / 32, XJ = TM / WM / 32;  // 32 x 32 blocks per wave
  static constexpr int TN = PAIR ? TW / 2 : TW;               // columns of the weights that a tile covers
  static constexpr int XSLOT = TM * BK * 2, WSLOT = TW * BK * 2;  // TM, TW rows of 64 k, or 64 k rows of TW
  static constexpr bool FIVE = TM == TW;                      // one ring of five slots, or rings of three for x and for W
  static constexpr int RING = FIVE ? 5 : 3;
  static constexpr int LX = XSLOT / 1024 / WAVES, LW = WSLOT / 1024 / WAVES;  // loads of a wave per slot
  static constexpr int LDS = FIVE ? RING * XSLOT : RING * (XSLOT + WSLOT);
  static __device__ __forceinline__ int x_at(int slot) { return slot * XSLOT; }
  static __device__ __forceinline__ int w_at(int slot) { return FIVE ? slot * XSLOT : RING * XSLOT + slot * WSLOT; }
  static_assert(XSLOT % (1024 * WAVES) == 0 && WSLOT % (1024 * WAVES) == 0 && LDS <= 160 * 1024, "the ring fits the LDS");
};

// y (a tile's outputs, as an epilogue defines them) over rows m of x, columns n of W; k runs over `parts` segments of K each:
// x's columns p K .. (p + 1) K with w0, then w1
struct GemmArgs {
  const bf16* x;   // [M][parts K], row stride xs
  const bf16* w0;  // [N][K] row stride ws0, or KMAJOR [K][N]
  const bf16* w1;  // PAIR: the second weight; parts == 2: that of the second part
  int64_t xs, ws0, ws1;
  int M, N, K, parts;
  int n_mt, n_nt;  // tiles
  int gm;          // m tiles of a block of tiles (see gemm_tile_at)
  // The first `full` tiles are whole; each of the others is cut along k into S pieces of `per` stages, whose fp32 sums go to
  // `part` ([piece][tile][wave][block][quad][lane]) for gemm_finish.
  int full, S, per;
  float* part;
};

template <int N>
__device__ __forceinline__ void gemm_wait_vmem() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ int gemm_swz(int row) { return (row >> 1) & 7; }

// What a descriptor is made of, the same in every lane; made where it is used, from scalar registers (the compiler does not see
// that of values which a loop carries past a branch).
struct GemmSpan {
  uint64_t base;
  uint32_t bytes;
  __device__ __forceinline__ buf_rsrc rsrc() const {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(base >> 32));
    return make_rsrc((const void*)(((uint64_t)hi << 32) | lo), (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes));
  }
};
__device__ __forceinline__ GemmSpan gemm_span(const void* p, uint32_t bytes) { return GemmSpan{(uint64_t)(uintptr_t)p, bytes}; }

template <class C>
struct GemmAcc {
  f32x16 a[C::NB][C::XJ];
};

// Tile `id` of n_mt x n_nt: consecutive logical ids run on one XCD (the hardware places workgroup id on XCD id % 8) and walk
// blocks of gm m tiles x all n tiles, m fastest, so that the tiles an XCD runs at once share their rows in its L2.
__device__ __forceinline__ void gemm_tile_at(const GemmArgs& a, int id, int& mt, int& nt) {
  const int n_wg = a.n_mt * a.n_nt;
  const int q = n_wg >> 3, r = n_wg & 7, xcd = id & 7;
  id = xcd * q + min(xcd, r) + (id >> 3);
  const int per = a.gm * a.n_nt, grp = id / per, in = id - grp * per;
  const int rows = min(a.gm, a.n_mt - grp * a.gm);
  mt = grp * a.gm + in % rows;
  nt = in / rows;
}

// An item of work: a tile, or a piece of one, as stages [beg, end) of all its parts' stages.
struct GemmItem {
  int tile, beg, end;
};
__device__ __forceinline__ GemmItem gemm_item(const GemmArgs& a, int id, int n_all) {
  if (id < a.full) return GemmItem{id, 0, n_all};
  const int rest = a.n_mt * a.n_nt - a.full, e = id - a.full, piece = e / rest;
  return GemmItem{a.full + e - piece * rest, piece * a.per, min(n_all, (piece + 1) * a.per)};
}

// Runs the items blockIdx.x, blockIdx.x + gridDim.x, ...: for each whole tile epi(acc, m0, n0, stage0, stage1, 0, XJ), where
// the two stages are SLOT bytes each that the epilogue may use until its last barrier (every wave must have passed it before
// it returns), and the last two arguments the range of 32-row blocks j of each wave to be stored.
template <class C, class Epi>
__device__ __forceinline__ void gemm_tiles(const GemmArgs& p, unsigned char* lds, Epi&& epi) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = w % C::WN, wm = w / C::WN;
  const int l32 = lane & 31, hk = lane >> 5;
  const int n_tiles = p.n_mt * p.n_nt;
  const int n_st = (p.K + C::BK - 1) / C::BK, n_all = n_st * p.parts;
  const int n_items = p.full + (n_tiles - p.full) * p.S;
  const int last_k = p.K - (n_st - 1) * C::BK;  // k of a part's last stage, a multiple of 8

  // ---- loads: a cursor for x and one for W, each (tile, part, stage) with the descriptors of its tile and part, which end at
  // the last valid row; lanes past them load nothing, and the outputs that such rows reach are not stored
  const uint32_t lds0 = lds_addr(lds);
  uint32_t xoff[C::LX], woff[C::LW];  // this lane's bytes in each of the wave's loads, at k = 0
  bool second[C::LW];                    // PAIR (wave-uniform): the load is of w1's rows
#pragma unroll
  for (int j = 0; j < C::LX; ++j) {
    const int row = 8 * (w + C::WAVES * j) + (lane >> 3);
    xoff[j] = (uint32_t)(row * p.xs * 2) + (uint32_t)(((lane & 7) ^ gemm_swz(row)) * 16);
  }
#pragma unroll
  for (int j = 0; j < C::LW; ++j) {
    const int i = w + C::WAVES * j, row = 8 * i + (lane >> 3);
    second[j] = false;
    if (C::KMAJOR) {
      const int at = i * 1024 + lane * 16, kr = at / (C::TW * 2), pos = (at % (C::TW * 2)) >> 4;
      woff[j] = (uint32_t)(kr * p.ws0 * 2) + (uint32_t)((pos ^ (4 * (kr & 3))) * 16);
    } else {
      int src = row;
      if (C::PAIR) {
        const int b = (8 * i) / 32, per = C::NB / 2;  // block b of the tile, b % NB of its wave
        second[j] = b % C::NB >= per;
        src = (b / C::NB * per + b % per) * 32 + (row & 31);
      }
      woff[j] = (uint32_t)(src * (C::PAIR && second[j] ? p.ws1 : p.ws0) * 2) + (uint32_t)(((lane & 7) ^ gemm_swz(row)) * 16);
    }
  }
  struct Cursor {
    int item, part, st, left;  // left: stages of the item from this one on
  };
  auto enter = [&](Cursor& c) {
    const GemmItem t = gemm_item(p, min(c.item, n_items - 1), n_all);
    c.part = t.beg >= n_st;  // (at most two parts)
    c.st = t.beg - c.part * n_st;
    c.left = t.end - t.beg;
  };
  auto advance = [&](Cursor& c) -> bool {  // whether the descriptors change
    if (--c.left == 0) {
      c.item = c.item < n_items ? c.item + (int)gridDim.x : c.item;
      enter(c);
      return true;
    }
    if (++c.st < n_st) return false;
    c.st = 0;
    ++c.part;
    return true;
  };
  GemmSpan rx, rw0, rw1;
  auto point_x = [&](const Cursor& c) {
    int mt, nt;
    gemm_tile_at(p, gemm_item(p, min(c.item, n_items - 1), n_all).tile, mt, nt);
    const int m0 = mt * C::TM;
    rx = gemm_span(p.x + (int64_t)m0 * p.xs + (int64_t)c.part * p.K,
                   c.item < n_items ? rows_bytes(min(C::TM, p.M - m0), p.xs, p.K * 2) : 0u);
  };
  auto point_w = [&](const Cursor& c) {
    int mt, nt;
    gemm_tile_at(p, gemm_item(p, min(c.item, n_items - 1), n_all).tile, mt, nt);
    const int n0 = nt * C::TN, nv = min(C::TN, p.N - n0);
    const bool live = c.item < n_items;
    const bf16* wp = !C::PAIR && c.part ? p.w1 : p.w0;
    const int64_t ws = !C::PAIR && c.part ? p.ws1 : p.ws0;
    if (C::KMAJOR) {
      rw0 = gemm_span(wp + n0, live ? rows_bytes(p.K, ws, nv * 2) : 0u);
    } else {
      rw0 = gemm_span(wp + (int64_t)n0 * ws, live ? rows_bytes(nv, ws, p.K * 2) : 0u);
      if (C::PAIR) rw1 = gemm_span(p.w1 + (int64_t)n0 * p.ws1, live ? rows_bytes(nv, p.ws1, p.K * 2) : 0u);
    }
  };
  Cursor cx{(int)blockIdx.x, 0, 0, 0}, cw;
  auto done_x = [&]() {
    if (advance(cx)) point_x(cx);
  };
  auto load_x = [&](const buf_rsrc& r, int slot, int j) {
    dma16(r, xoff[j] + (uint32_t)(cx.st * C::BK * 2), lds0 + (uint32_t)(C::x_at(slot) + (w + C::WAVES * j) * 1024));
  };
  auto issue_x = [&](int slot) {
    const buf_rsrc r = rx.rsrc();
#pragma unroll
    for (int j = 0; j < C::LX; ++j) load_x(r, slot, j);
    done_x();
  };
  const uint32_t wstep = C::KMAJOR ? (uint32_t)(C::BK * p.ws0 * 2) : (uint32_t)(C::BK * 2);
  auto done_w = [&]() {
    if (advance(cw)) point_w(cw);
  };
  auto load_w = [&](const buf_rsrc& r0, const buf_rsrc& r1, int slot, int j) {
    dma16(C::PAIR && second[j] ? r1 : r0, woff[j] + (uint32_t)cw.st * wstep,
          lds0 + (uint32_t)(C::w_at(slot) + (w + C::WAVES * j) * 1024));
  };
  auto issue_w = [&](int slot) {
    const buf_rsrc r0 = rw0.rsrc(), r1 = C::PAIR ? rw1.rsrc() : r0;
#pragma unroll
    for (int j = 0; j < C::LW; ++j) load_w(r0, r1, slot, j);
    done_w();
  };

  // ---- fragment reads: lane (l32, hk) takes row l32 of a block and k = 16 h + 8 hk + [0, 8).  Transpose reads: lane
  // (hk, l16) addresses 4 columns of row 8 hk + l16 / 4 (+ 4, + 16 h); 32-column block b of a row sits at 64 (b ^ (row mod 4))
  // within its 256 bytes.
  int offw[C::KMAJOR ? C::NB : C::HS], offx[C::HS];
  if (C::KMAJOR) {
    const int l16 = lane & 15, r2 = l16 >> 2;
#pragma unroll
    for (int i = 0; i < C::NB; ++i) {
      const int b = wn * C::NB + i;
      offw[i] = (8 * hk + r2) * (C::TW * 2) + 256 * (b >> 2) + 64 * ((b & 3) ^ r2) + 32 * ((lane >> 4) & 1) + 8 * (l16 & 3);
    }
  }
#pragma unroll
  for (int h = 0; h < C::HS; ++h) {
    const int rw_ = 32 * C::NB * wn + l32;  // the block's row within the tile is + 32 i (the swizzle unchanged)
    if (!C::KMAJOR) offw[h] = rw_ * 128 + (((2 * h + hk) ^ gemm_swz(rw_)) * 16);
    const int rx_ = 32 * C::XJ * wm + l32;
    offx[h] = rx_ * 128 + (((2 * h + hk) ^ gemm_swz(rx_)) * 16);
  }
  bf16x8 fx[C::HS][C::XJ], fw[2][C::NB];  // x of a stage's four steps, W of this step and the next
  auto read_x = [&](int slot, int h) {
    const unsigned char* xt = lds + C::x_at(slot);
#pragma unroll
    for (int j = 0; j < C::XJ; ++j) fx[h][j] = as_bf16x8(lds16(xt + offx[h] + j * 32 * 128));
  };
  auto read_w = [&](int slot, int h) {
    const unsigned char* wt = lds + C::w_at(slot);
#pragma unroll
    for (int i = 0; i < C::NB; ++i) {
      if (C::KMAJOR) {
        const unsigned char* a = wt + offw[i] + 16 * h * (C::TW * 2);
        const s16x4_t lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)a);
        const s16x4_t hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(a + 4 * (C::TW * 2)));
        const u32x2 l = __builtin_bit_cast(u32x2, lo4), hh = __builtin_bit_cast(u32x2, hi4);
        fw[h & 1][i] = as_bf16x8(u32x4{l[0], l[1], hh[0], hh[1]});
      } else {
        fw[h & 1][i] = as_bf16x8(lds16(wt + offw[h] + i * 32 * 128));
      }
    }
  };
  GemmAcc<C> acc;
  auto multiply = [&](int h) {
#pragma unroll
    for (int i = 0; i < C::NB; ++i)
#pragma unroll
      for (int j = 0; j < C::XJ; ++j) acc.a[i][j] = mfma32(fw[h & 1][i], fx[h][j], acc.a[i][j]);
  };
  // A step's products with the wave's loads of one slot between them: one behind the other, the loads would wait for each other
  // in the memory pipe, and the wave's next products for them.
  auto multiply_loading = [&](int h, auto loads, auto&& load) {
#pragma unroll
    for (int i = 0; i < C::NB; ++i)
#pragma unroll
      for (int j = 0; j < C::XJ; ++j) {
        constexpr int products = C::NB * C::XJ, L = decltype(loads)::value;
        acc.a[i][j] = mfma32(fw[h & 1][i], fx[h][j], acc.a[i][j]);
        const int n = i * C::XJ + j;
#pragma unroll
        for (int l = n * L / products; l < (n + 1) * L / products; ++l) load(l);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  // the reads go out between the step's first products (left alone, the compiler moves them to their use)
  auto interleave = [&]() {
    constexpr int reads = C::XJ + (C::KMAJOR ? 2 : 1) * C::NB, products = C::NB * C::XJ;
    constexpr int each = (reads + products - 1) / products;
#pragma unroll
    for (int n = 0; n < products; ++n) {
      __builtin_amdgcn_sched_group_barrier(0x100, each, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // step h of a part's last stage: k past its end (whole chunks: the lane's 8 k are in or out together) becomes zero in both
  auto cut = [&](int h, int tail) {
    const bool in = 16 * h + 8 * hk < tail;
    const u32x4 z{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < C::XJ; ++j) fx[h][j] = as_bf16x8(in ? as_u32x4(fx[h][j]) : z);
#pragma unroll
    for (int i = 0; i < C::NB; ++i) fw[h & 1][i] = as_bf16x8(in ? as_u32x4(fw[h & 1][i]) : z);
  };

  if ((int)blockIdx.x >= n_items) return;
  enter(cx);
  cw = cx;
  point_x(cx);
  point_w(cw);
  if (C::FIVE) {
    issue_x(0);
    issue_w(1);
    issue_x(2);
    issue_w(3);
    issue_x(4);
    gemm_wait_vmem<2 * C::LX + C::LW>();
  } else {
    issue_x(0);
    issue_w(0);
    issue_x(1);
    issue_w(1);
    gemm_wait_vmem<C::LX + C::LW>();
  }
  __syncthreads();
  int sx = 0, sw = C::FIVE ? 1 : 0;  // the slots of the stage being multiplied
  auto next_slots = [&]() {
    if (C::FIVE) {
      sx = sx >= C::RING - 2 ? sx - (C::RING - 2) : sx + 2;
      sw = sw >= C::RING - 2 ? sw - (C::RING - 2) : sw + 2;
    } else {
      sx = sw = sx == C::RING - 1 ? 0 : sx + 1;
    }
  };
  auto read_first = [&]() {  // what a stage's slots give before its first step's products
    read_w(sw, 0);
#pragma unroll
    for (int h = 0; h + 1 < C::HS; ++h) read_x(sx, h);
  };
  auto behind = [&](int s) { return s == 0 ? C::RING - 1 : s - 1; };  // rings of three: the slot of the stage after next
  read_first();
  for (int id = blockIdx.x; id < n_items; id += gridDim.x) {
    const GemmItem item = gemm_item(p, id, n_all);
#pragma unroll
    for (int i = 0; i < C::NB; ++i)
#pragma unroll
      for (int j = 0; j < C::XJ; ++j) acc.a[i][j] = f32x16{};
    for (int g = item.beg; g < item.end;) {
      const int part_end = g < n_st ? n_st : n_all, stop = min(item.end, part_end);
      const int tail = stop == part_end ? last_k : C::BK;
      for (; g + 1 < stop; ++g) {
        read_x(sx, C::HS - 1);
        read_w(sw, 1);
        multiply(0);
        interleave();
        if (C::FIVE) __syncthreads();  // every wave holds the stage's x in registers
        read_w(sw, 2);
        __builtin_amdgcn_sched_barrier(0);
        const buf_rsrc r0 = rw0.rsrc(), r1 = C::PAIR ? rw1.rsrc() : r0;
        const int s2 = behind(sx);
        multiply_loading(1, std::integral_constant<int, C::LW>{}, [&](int j) { load_w(r0, r1, C::FIVE ? sx : s2, j); });
        done_w();
        read_w(sw, 3);
        if (C::FIVE) {
          multiply(2);
          interleave();
          // every wave holds the stage in registers and the next one has landed: all but the one behind it
          gemm_wait_vmem<C::LX + C::LW>();
          __syncthreads();
          const int s1 = sw;
          next_slots();
          read_first();
          __builtin_amdgcn_sched_barrier(0);
          const buf_rsrc r = rx.rsrc();
          multiply_loading(3, std::integral_constant<int, C::LX>{}, [&](int j) { load_x(r, s1, j); });
          done_x();
        } else {
          __builtin_amdgcn_sched_barrier(0);
          const buf_rsrc r = rx.rsrc();
          multiply_loading(2, std::integral_constant<int, C::LX>{}, [&](int j) { load_x(r, s2, j); });
          done_x();
          gemm_wait_vmem<C::LX + C::LW>();
          __syncthreads();
          next_slots();
          read_first();
          multiply(3);
        }
      }
      if (!C::FIVE) {
        issue_w(behind(sx));
        issue_x(behind(sx));
      }
      read_x(sx, C::HS - 1);
#pragma unroll
      for (int h = 0; h + 1 < C::HS; ++h) {
        read_w(sw, h + 1);
        cut(h, tail);
        multiply(h);
      }
      cut(C::HS - 1, tail);
      gemm_wait_vmem<C::FIVE ? C::LX : C::LX + C::LW>();
      __syncthreads();
      const int s0 = sx, s1 = sw;
      next_slots();
      __builtin_amdgcn_sched_barrier(0);
      multiply(C::HS - 1);
      ++g;
      if (g == item.end) {
        if (id >= p.full && p.S > 1) {
          int ln = lane;
          asm volatile("" : "+v"(ln));  // (addresses formed here, not kept through the products)
          f32x4* const dst = reinterpret_cast<f32x4*>(p.part) + (int64_t)(id - p.full) * (C::TM * C::TW / 4) +
                             w * (C::NB * C::XJ * 256) + ln;
#pragma unroll
          for (int i = 0; i < C::NB; ++i)
#pragma unroll
            for (int j = 0; j < C::XJ; ++j)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const f32x16& a = acc.a[i][j];
                dst[((i * C::XJ + j) * 4 + q) * 64] = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
              }
        } else {
          int mt, nt;
          gemm_tile_at(p, item.tile, mt, nt);
          epi(acc, mt * C::TM, nt * C::TN, lds + C::x_at(s0), lds + C::w_at(s1), 0, C::XJ);
        }
        gemm_wait_vmem<0>();  // (its stores share the counter that the stages' waits count down)
      }
      if (C::FIVE) {
        issue_w(s0);
        issue_x(s1);
      }
      read_first();
    }
  }
  gemm_wait_vmem<0>();  // no load is in flight into LDS when the workgroup ends
}

// The tiles that were cut: workgroup (tile, j) adds the pieces' sums of block row j in order and runs the epilogue on it.
// Bound by reading the pieces, once.  lds: XSLOT + WSLOT bytes.
template <class C, class Epi>
__device__ __forceinline__ void gemm_finish(const GemmArgs& p, unsigned char* lds, Epi&& epi) {
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rest = p.n_mt * p.n_nt - p.full, t = blockIdx.x / C::XJ, jj = blockIdx.x % C::XJ;
  const f32x4* src = reinterpret_cast<const f32x4*>(p.part) + (int64_t)t * (C::TM * C::TW / 4) + w * (C::NB * C::XJ * 256) + lane;
  const int64_t step = (int64_t)rest * (C::TM * C::TW / 4);
  GemmAcc<C> acc;
#pragma unroll
  for (int i = 0; i < C::NB; ++i)
#pragma unroll
    for (int j = 0; j < C::XJ; ++j) {
      acc.a[i][j] = f32x16{};
      if (j != jj) continue;
      for (int s0 = 0; s0 < p.S; s0 += 4) {  // four pieces' reads in flight
        f32x4 v[4][4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int q = 0; q < 4; ++q) v[s][q] = src[min(s0 + s, p.S - 1) * step + ((i * C::XJ + j) * 4 + q) * 64];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc.a[i][j][4 * q + e] += s0 + s < p.S ? v[s][q][e] : 0.f;
      }
    }
  int mt, nt;
  gemm_tile_at(p, p.full + t, mt, nt);
  epi(acc, mt * C::TM, nt * C::TN, lds, lds + C::XSLOT, jj, jj + 1);
}

}  // namespace mla
