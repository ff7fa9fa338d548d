// The host's choices of grid, tile and split that depend on nothing but sizes: plain C++, so that the tests can ask them.
#pragma once

#include <stdint.h>

namespace mla {

// ---- the attention kernels' grids (prefill_fwd.hip, prefill_bwd.hip)
// Whether a causal attention kernel's grid runs one tile of 128 rows per workgroup, longest first, instead of mirrored
// pairs (tiles r and n - 1 - r of one (b, h), always the same work together).  Pairs start a new round of workgroups for
// any remainder; single tiles fill the chip to the end but start twice as often, without the next tile's prefetch, and
// share less of a (b, h) in L2.  Results are the same bit for bit.  Times in units of a pair's, n_bh (b, h) of n tiles:
//   single tiles: the work over the workgroups that run at once, plus what the starts cost, at least the longest tile;
//   pairs: whole rounds; where two workgroups share a CU, a last round of one per CU takes a fraction of that.
// The constants are fitted, not derived; what they stand for is beside them.  Checked over 150 random sizes of both head
// layouts (14 heads of 64 + 64, 16 of 128 + 64 with shared k_rope; B to 24, T 150 to 8000, B T to 24000), each kernel timed
// in both grids: against pairs everywhere the forward takes 5.0 % less on average (at most 28 % less, 2.5 % more), the
// backward 4.7 % less through dK/dV (21 % less, 0.5 % more) and 1.2 % less through dQ (13 % less, 2.3 % more); against the
// faster grid of each size the rule leaves 1.3 %, 0.1 % and 1.6 %, the most (16 % of a forward, 13 % of a backward) where
// fewer than 256 pairs run one to a CU.  Examples, pairs -> single (us, B x T), forward / whole backward:
//   3 x 3000 180 -> 144 / 530 -> 468;  2 x 2600 76 -> 63 / 263 -> 191;  4 x 2900 148 -> 130 / 450 -> 418;  3 x 1900 60 ->
//   52 / 206 -> 169;  but whole rounds: 12 x 2048 265 -> 279 / 911 -> 990;  4 x 4096 319 -> 320 / 1060 -> 1076.
struct TileGrid {
  int64_t n_bh, n;
  bool square;  // causal from the first key: tile sizes 1 .. n, else alike
  double longest() const { return square ? (double)n / (double)(n + 1) : 0.5; }
  double work() const { return (double)n_bh * (double)n / 2; }
  int64_t pairs() const { return n_bh * ((n + 1) / 2); }
};
inline bool single_tiles_one_per_cu(const TileGrid& g) {  // 256 workgroups at once
  if (g.n < 2) return false;
  const double pair = (double)((g.pairs() + 255) / 256);
  // a start (nothing prefetched) costs a pair's tiles 1 / n of their time; never less than the longest tile
  const double most = g.work() / 256 * (1.0 + 1.0 / (double)g.n), single = most > g.longest() ? most : g.longest();
  return single < 0.97 * pair;  // (what is this close stays in pairs)
}
inline bool single_tiles_two_per_cu(const TileGrid& g) {  // 512, two on a CU
  if (g.n < 2) return false;
  const int64_t rest = g.pairs() % 512;
  // a last round of at most 160 pairs, alone on their CUs: 0.42 of a round of two a CU; to 256, where the dispatcher puts
  // some on one CU, up to 0.67; beyond, a whole round
  const double last = rest == 0 ? 0.0 : rest > 256 ? 1.0 : 0.42 + (rest > 160 ? 0.25 * (double)(rest - 160) / 96 : 0.0);
  const double pair = (double)(g.pairs() / 512) + last;
  // a start costs 0.6 / n (the other workgroup of the CU runs on); the longest tile, alone on its CU at the end, 0.8
  const double most = g.work() / 512 * (1.0 + 0.6 / (double)g.n), low = 0.8 * g.longest();
  return (most > low ? most : low) < 0.95 * pair;
}

// ---- norm_linear.hip's output tiles
constexpr int kNlBK = 32;  // k per stage

struct NlPlan {
  int kind;  // 0 NlWide (+ NlRest), 1 NlHalf, 2 NlSmall
  int64_t n_nt, n_wide, n_rest;
};

// The least of: rounds of 256 workgroups (one per CU) x (the tile's time per stage x stages + what a workgroup takes
// beside them), both fitted to the measured calls (us at M x N x K, wide / half / small tiles): 12288 x 2560 x 1792 129.0 /
// 146.0 / 168.8 (two full rounds of wide tiles), 8192 x 2624 x 2048 132.8 / 127.7 / 140.7, 2735 x 2000 x 1632 57.1 / 36.6 /
// 40.2, 1000 x 2624 x 2048 61.7 / 42.6 / 39.3 (wide tiles leave most of the chip idle).  Small tiles share a CU.
inline NlPlan nl_plan(int64_t M, int64_t N, int64_t K) {
  NlPlan best{};
  double best_t = 1e300;
  const double stages = (double)(K / kNlBK);
  static const int bn[3] = {256, 256, 128}, bm[3] = {256, 128, 128};
  static const double ts[3] = {1.0, 0.6, 0.39}, fixed[3] = {6.0, 4.0, 1.5};
  for (int kind = 0; kind < 3; ++kind) {
    const int64_t mt = (M + bm[kind] - 1) / bm[kind];
    int64_t nt = (N + bn[kind] - 1) / bn[kind], rest = 0;
    if (kind == 0 && nt > 1 && N % 256 != 0 && N % 256 <= 128) {
      --nt;
      rest = mt;
    }
    const int64_t wide = mt * nt;
    // the remainder's tiles fill the last round's free CUs first
    double rounds = (double)((wide + 255) / 256);
    const int64_t over = rest - (int64_t)(rounds * 256 - wide);
    if (over > 0) rounds += 0.6 * (double)((over + 255) / 256);
    const double t = rounds * (stages * ts[kind] + fixed[kind]);
    if (t < best_t) {
      best_t = t;
      best = NlPlan{kind, nt, wide, rest};
    }
  }
  return best;
}

// ---- wgrad.hip's output tiles and token segments
constexpr int kWgSt = 32;  // tokens per stage

struct WgPlan {
  int narrow, S, seg, nt, kt;
  int64_t part_bytes;
};

// The plan of least estimated time: rounds of 256 workgroups (one per CU), each its stages at the measured 1.05 us (wide
// tile: 128 stages of 4096 x 2048 took 124-134 us) or 0.62 us (narrow) plus 4 us of start and stores, and where the
// tokens are cut the second kernel with its partials at 4 TB/s.  Wide tiles stage fewer bytes per product, so they win
// where the weight has enough of them; narrow ones (and more segments) where it has few: 896 x 384 makes 12.
inline WgPlan wg_plan(int64_t M, int64_t N, int64_t K) {
  WgPlan best{};
  double best_t = 1e300;
  const int64_t st = (M + kWgSt - 1) / kWgSt;
  for (int narrow = 0; narrow < 2; ++narrow) {
    const int64_t TN = 256, TK = narrow ? 128 : 256;
    const int64_t nt = (N + TN - 1) / TN, kt = (K + TK - 1) / TK, tiles = nt * kt;
    const double ts = narrow ? 0.62 : 1.05;  // us per stage of a workgroup
    for (int64_t S = 1; S <= 32 && S <= st; ++S) {
      const int64_t per = (st + S - 1) / S;
      if ((st + per - 1) / per != S) continue;  // fewer segments hold the same stages
      const double rounds = (double)((tiles * S + 255) / 256);
      double t = rounds * ((double)per * ts + 4.0);
      const int64_t pb = S > 1 ? tiles * S * TN * TK * 4 : 0;
      if (S > 1) t += 4.0 + (double)pb / 4.0e6;
      if (pb > (256ll << 20)) continue;
      if (t < best_t) {
        best_t = t;
        best = WgPlan{narrow, (int)S, (int)(per * kWgSt), (int)nt, (int)kt, pb};
      }
    }
  }
  return best;
}

// ---- linear_act.hip's and gated_linear.hip's tiles (gemm_core.h)
enum { kGemmSmall = 0, kGemmHalf = 1, kGemmLarge = 2 };
struct GemmTile {
  int64_t m, n, slots;  // outputs, and how many run at once: one workgroup a CU, or two
  // us of a stage of 64 k with every slot taken, and of a tile's start and stores; of a stage of a round of r <= 256 workgroups,
  // one a CU: alone + share r / 256
  double stage, fixed, alone, share;
};
constexpr GemmTile kGemmTiles[3] = {
    {128, 128, 512, 1.05, 0.0, 0.40, 0.16}, {256, 128, 256, 1.04, 1.2, 0.63, 0.28}, {256, 256, 256, 1.57, 7.0, 0.99, 0.41}};

struct GemmPlan {
  int tile;    // of kGemmTiles
  int S, per;  // the tiles of an unfilled last round are cut along k into S pieces of `per` stages (1: not cut)
  int64_t part_bytes;
};

// The plan of least estimated time (us) for y [M, N] over parts x K: full rounds, the last one, and for pieces their fp32 sums
// (written and read at 6 TB/s together) and the kernel that adds them.  The constants are fitted to 1000 timings of 100 products
// (M 65 to 16000; N and K 256 to 5600; every tile, S to 8; inputs of three calls in turn), which they meet within 9 % (rms).  Over
// the products the rule's choice takes 0.5 % more than the fastest one on average and 12 % at most; without pieces it would take
// 17 % more, without the tiles of 256 x 128 2 %, without those of 128 x 128 9 %.  Examples (us; 128 x 128, 256 x 128, 256 x 256):
// 1999 x 2048 over 4608 50, 61, 97; 3001 x 2048 over 5464 101, 85, 114 (95 in two pieces); 12288 x 9216 over 1792 430, 426, 365;
// 12288 x 1792 over 2 x 4608 430, 403, 413 (348 in three pieces); 159 x 6080 over 5176 47, 62, 98 (31 in four pieces of 128 x 128).
// The timings are of products with a plain store, K a multiple of 64, operands near the caches.  Elsewhere calls take longer than
// estimated (estimate, call): 2500 x 1000 over 1800 with bias and silu 15, 25 (over 1792 14, 21: rows that no 128 bytes divide);
// 1999 x 2048 over 4608 40, 48; 12288 x 4608 over 1792 with kept values 191, 225; 12288 x 1792 over 2 x 4608 321, 359.  The choice
// holds there too: in twelve such calls, kept values, activations and both directions among them, it was within 2 % of the fastest
// tile (12288 x 4608 over 1792, gelu, kept: 240, 238, 224; profiles/linear_sizes.txt).
inline GemmPlan gemm_plan(int64_t M, int64_t N, int64_t K, int64_t parts) {
  GemmPlan best{};
  double best_t = 1e300;
  const int64_t n = (K + 63) / 64 * parts;
  for (int tile = kGemmLarge; tile >= kGemmSmall; --tile) {
    const GemmTile& T = kGemmTiles[tile];
    const int64_t tiles = ((M + T.m - 1) / T.m) * ((N + T.n - 1) / T.n), rest = tiles % T.slots;
    for (int64_t S = 1; S <= 8; ++S) {
      if (S > 1 && (S * 2 > n || rest == 0 || rest * S > T.slots)) break;
      const int64_t per = (n + S - 1) / S, items = rest * S;
      if ((n + per - 1) / per != S) continue;  // fewer pieces hold the same stages
      double t = (double)(tiles / T.slots) * ((double)n * T.stage + T.fixed);
      if (items > 256) t += (double)per * T.stage + T.fixed;
      else if (items > 0) t += (double)per * (T.alone + T.share * (double)items / 256) + T.fixed;
      const int64_t pb = S > 1 ? items * T.m * T.n * 4 : 0;
      if (S > 1) t += 3.0 + 0.6 * (double)S + (double)pb / 6e6;
      if (t < best_t) {
        best_t = t;
        best = GemmPlan{tile, (int)S, (int)per, pb};
      }
    }
  }
  return best;
}

// ---- rows_core.h's columns of a workgroup: 16, or 32 where 16 would make a second round (a CU alone moves several times its
// share of the memory's rate, and the wider workgroup reads x half as often).
inline int rows_columns(int64_t N) { return N <= 16 * 256 ? 16 : 32; }

}  // namespace mla
