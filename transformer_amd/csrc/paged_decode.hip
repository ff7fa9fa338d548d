// Absorbed latent decode over a paged cache in 16 or 4 bits (gfx950): one query token a sequence.
//
//   s_j = (q_lat . c_j + q_rope . k_j) scale,   ctx = softmax(s) c,   lse = logsumexp(s)
//
// over the rows [c | k] of a sequence's pages, each read once for the 16 heads of a head group: 1152 bytes a token in 16 bits
// (d_latent 512, one rotated key), 306 in 4, for 35 KFLOP.  16 bits are bound by memory and by what a workgroup takes to begin and end,
// 4 bits by the instructions that unpack.
//
// Measured (kernel trace; a stream that only reads reaches 6.0 TB/s), this kernel and the merge of the parts:
//   16 bits, 32 sequences up to 4096, 85 MB        22.4 + 4.3 us  (3.8 TB/s, 3.2 with the merge)
//   16 bits, one of 701 tokens, 14 keys            7.4 + 3.9
//   4 bits, 64 up to 16384, 179 MB                 58.6 + 6.3  (3.1 TB/s; VALU busy 65 % of the time)
//   4 bits, 64 up to 4000 with 14 keys, 87 MB      27.0 + 5.7  (3.2 TB/s)
//   4 bits, one of 3001                            9.9 + 3.9
// About 5 us of each are the launch, the lengths, the page look-ups and the first tile's way from memory.
//
// Work.  A unit is a sequence and head group, a tile 16 tokens of it (16 bits) or 64 (4 bits).  The tiles of all units in a row are
// cut into equal runs, one a workgroup, whatever the sequences' lengths: every workgroup adds the lengths up and finds its place
// itself, so nothing is planned on the host and a recorded call follows the lengths.  A unit that lies in one run is finished there;
// one that spans several leaves (m, l, O) of each in fp32, which the merge kernel adds in the runs' order (no atomics: results
// repeat bit for bit).
//
// A workgroup's tiles come through a ring of LDS slots by direct-to-LDS loads, which run on across its units.  16 tokens never
// straddle a page, so a buffer descriptor of the tokens that exist (none, where the entry is no page) bounds each load of rows: those
// behind a sequence's end read as zero.  The scales of 4 bits are read for all 16 tokens, whatever stands behind the end: the sums of O
// take zeros for those (the fp32 copies, or the scales in LDS, are cleared), and the scores, whose first product takes them as they are,
// are masked by the number of tokens.  Waves share the scores through LDS and each then owns some of the latent's columns, so no wave's
// O has to be merged with another's.  One barrier a tile.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace mla {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2 lds_i32x2;

struct PagedDecodeParams {
  PagedParams c;
  const bf16 *q_lat, *q_rope;
  const int32_t* seq_lens;
  bf16* ctx;
  float* lse;
  float* part_o;   // [2 runs][16][DL]: slot 2 run for a unit that begins before the run, 2 run + 1 for one that ends after it
  float* part_ml;  // [2 runs][16][2]: m (log2) and l
  int32_t* units;  // [B][n_hg]: the run that a unit with tiles begins in, and in how many runs it lies << 16
  int B, H, n_hg, runs;  // (runs * the places of one stays below 2^31)
  int pieces;          // 16-token pieces of a page
  uint32_t piece_magic;  // ceil(2^32 / pieces): the page of piece s < 2^24 is the high half of s times this (pieces > 1)
  int64_t q_lat_sb, q_lat_sh, q_rope_sb, q_rope_sh;
  float scale_log2;
};

constexpr uint32_t kPdNothing = 0x40000000u;  // an offset past every descriptor: reads as zero
constexpr float kPdRescale = 8.0f;  // growth of a head's running max (log2) that makes O be scaled again

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}
// a barrier that leaves the loads in flight alone
__device__ __forceinline__ void pd_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ int pd_len(const PagedDecodeParams& p, int b) {
  return min(max(p.seq_lens[b], 0), p.c.table_pages * p.c.size);
}
// the same for a b that is the same in all lanes, by a scalar load: a vector one would be waited for with all loads into the ring
__device__ __forceinline__ int pd_len1(const PagedDecodeParams& p, int b) {
  const auto* lens = (const __attribute__((address_space(4))) int32_t*)p.seq_lens;
  return min(max(lens[b], 0), p.c.table_pages * p.c.size);
}
__device__ __forceinline__ int pd_page(const PagedDecodeParams& p, int piece) {
  return p.pieces == 1 ? piece : (int)__umulhi((uint32_t)piece, p.piece_magic);
}

// A place in the units' tiles: tile `tile` of the `n` of (b, hg), the workgroup's tiles going to `end` in the line of all.
//
// On that line a unit takes COST places before its tiles: what its beginning and end cost in tiles (queries, stores), so that a
// workgroup whose run holds the ends of several gets fewer tiles.  A run has LEAST places at least: one sequence is not cut so finely
// that the parts take longer than the tiles (one of 701 tokens in 16 bits: 7.4 + 3.8 us with 3, 9.1 + 3.9 with 5; one of 3001 in 4 bits:
// 10.0 + 4.0 with 2, 9.1 + 4.9 with 1).  All numbers stay below 2^31.
template <class C>
struct PdCursor {
  int b, hg, tile, n, len, left;  // left: of the run's line, from this tile on
  int each;                       // places a run

  __device__ __forceinline__ bool more() const { return left > 0; }
  // the next tile of the run, or left <= 0
  __device__ __forceinline__ void next(const PagedDecodeParams& p) {
    --left;
    if (++tile < n) return;
    tile = 0;
    left -= C::COST;
    if (left <= 0 || ++hg < p.n_hg) return;
    hg = 0;
    do {
      len = pd_len1(p, ++b);
      n = (len + C::TT - 1) / C::TT;
    } while (n == 0 && b + 1 < p.B);
  }
};

__device__ __forceinline__ int wave_scan(int v) {  // the lanes up to and with this one
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // lane 15 of rows 0 and 2 into the next ones
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // lane 31 into rows 2 and 3
}
// The places on the line of one unit of each of the sequences up to and with lane's (b0 + lane); n: its tiles.
template <class C>
__device__ __forceinline__ int pd_scan(const PagedDecodeParams& p, int b0, int lane, int& n, int& len) {
  const int b = b0 + lane;
  len = b < p.B ? pd_len(p, b) : 0;
  n = (len + C::TT - 1) / C::TT;
  return wave_scan(n ? n + C::COST : 0);
}
// The cursor of a run; left <= 0 where it has no tile.
template <class C>
__device__ __forceinline__ PdCursor<C> pd_begin(const PagedDecodeParams& p, int run, int lane) {
  PdCursor<C> c = {0, 0, 0, 0, 0, 0, 0};
  int n, len, upto = pd_scan<C>(p, 0, lane, n, len), before = 0, total = __builtin_amdgcn_readlane(upto, 63);
  for (int b0 = 64; b0 < p.B; b0 += 64) {
    int nb, lb;
    total += __builtin_amdgcn_readlane(pd_scan<C>(p, b0, lane, nb, lb), 63);
  }
  total *= p.n_hg;
  const int each = max((int)((uint32_t)(total + p.runs - 1) / (uint32_t)p.runs), C::LEAST), from = run * each;
  if (from >= total) return c;
  for (int b0 = 0;;) {
    const uint64_t past = __ballot((before + upto) * p.n_hg > from);
    if (past) {
      const int at = __builtin_ctzll(past);
      c.b = b0 + at;
      c.n = __builtin_amdgcn_readlane(n, at);
      c.len = __builtin_amdgcn_readlane(len, at);
      const int unit = c.n + C::COST, in = from - (before + __builtin_amdgcn_readlane(upto, at) - unit) * p.n_hg;
      c.hg = p.n_hg == 1 ? 0 : in / unit;
      c.tile = in - c.hg * unit - C::COST;
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    b0 += 64;
    upto = pd_scan<C>(p, b0, lane, n, len);
  }
  c.each = each;
  c.left = min(each, total - from);
  if (c.tile < 0) {  // the run begins among the unit's first places
    c.left += c.tile;
    c.tile = 0;
  }
  return c;
}

// Where the 16-token piece `piece` of each of the next 64 tiles lies, a tile a lane, and how many of its tokens there are (none without
// a page).  Looked up together: in scalar operations each tile's address was most of a loading wave's time.
template <class C>
struct PdPieces {
  int first, b;
  uint32_t rows_lo, rows_hi, scales_lo, scales_hi;
  int tokens;

  // the lane of tile c.tile
  __device__ __forceinline__ int lane_of(const PagedDecodeParams& p, const PdCursor<C>& c, int piece, int lane) {
    if (c.b != b || c.tile - first >= 64 || c.tile < first) {
      b = c.b;
      first = c.tile;
      const int sub = (first + lane) * (C::TT / 16) + piece, page = pd_page(p, sub), in = sub - page * p.pieces;
      const int id = sub * 16 < c.len ? page_of(p.c, b, page) : -1;
      tokens = id < 0 ? 0 : min(16, c.len - sub * 16);
      const uint64_t rows = (uint64_t)p.c.pages + max(id, 0) * p.c.page_stride + (int64_t)in * 16 * p.c.row_bytes;
      const uint64_t scales = (uint64_t)p.c.scales + 2 * (max(id, 0) * p.c.scale_stride + in * 16);
      rows_lo = (uint32_t)rows;
      rows_hi = (uint32_t)(rows >> 32);
      scales_lo = (uint32_t)scales;
      scales_hi = (uint32_t)(scales >> 32);
      asm volatile("" : "+v"(tokens));  // waited for here: at its use in each tile it would be with all loads into the ring
    }
    return c.tile - first;
  }
  __device__ __forceinline__ int tokens_of(int at) const { return __builtin_amdgcn_readlane(tokens, at); }
  __device__ __forceinline__ buf_rsrc rows_of(int at, uint32_t nbytes) const {
    const uint32_t lo = __builtin_amdgcn_readlane((int)rows_lo, at), hi = __builtin_amdgcn_readlane((int)rows_hi, at);
    return make_rsrc((const void*)((uint64_t)hi << 32 | lo), nbytes);
  }
  __device__ __forceinline__ buf_rsrc scales_of(int at, uint32_t nbytes) const {
    const uint32_t lo = __builtin_amdgcn_readlane((int)scales_lo, at), hi = __builtin_amdgcn_readlane((int)scales_hi, at);
    return make_rsrc((const void*)((uint64_t)hi << 32 | lo), nbytes);
  }
};

// Stores of a unit's 16 heads x 4 columns a lane: the result, or the run's part.
template <int DL>
struct PdOut {
  bool whole;
  int slot;
  int runs;  // that the unit lies in; 0 where it began before this one
  // a unit of n tiles whose tiles from .. tile are the run's
  template <class C>
  __device__ __forceinline__ PdOut(const PdCursor<C>& c, int from, int tile, int n)
      : whole(from == 0 && tile + 1 == n),
        slot(2 * (int)blockIdx.x + (from == 0 ? 1 : 0)),
        runs(from ? 0 : whole ? 1 : 1 + (int)((uint32_t)(n - tile - 2 + c.each) / (uint32_t)c.each)) {}
  __device__ __forceinline__ void columns(const PagedDecodeParams& p, int b, int h, int l16, int col, f32x4 o, float inv) const {
    if (!whole) {
      *reinterpret_cast<f32x4*>(p.part_o + ((int64_t)slot * 16 + l16) * DL + col) = o;
    } else if (h < p.H) {
      o *= inv;
      stg8(p.ctx + ((int64_t)b * p.H + h) * DL + col, u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])});
    }
  }
  __device__ __forceinline__ void sums(const PagedDecodeParams& p, int b, int hg, int h, int l16, float m, float l) const {
    if (l16 == 0 && runs) p.units[(int64_t)b * p.n_hg + hg] = (int)blockIdx.x | runs << 16;
    if (!whole) {
      p.part_ml[(slot * 16 + l16) * 2] = m;
      p.part_ml[(slot * 16 + l16) * 2 + 1] = l;
    } else if (h < p.H) {
      p.lse[(int64_t)b * p.H + h] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * kLn2;
    }
  }
};

// ------------------------------------------------------------------------------------------------ 16 bits

// Rows [latent | shared key] (or the latent alone) lie in a slot as 16-byte chunks, chunk c of token t at c ^ tok_swz(t), RS chunks a
// row (RS = 8 mod 16): the QK reads (16 tokens x one chunk) and the transpose reads (4 tokens x 2 chunks a 16 lanes) are free of bank
// conflicts.  Keys of their own lie head by head, 16 tokens x 8 chunks, chunk c at c ^ (t / 2): in a ring one slot shorter, since only
// the scores read them.
//
// Four waves compute and two load.  A load into LDS holds its wave up (about 90 cycles while all waves of the workgroup issue some),
// which the computing waves do not have between two barriers; and theirs are the only vector loads that the compiler does not see, so it
// may wait for the others (queries) as it likes.  (All four waves loading and computing: 32.4 us for the 85 MB, with these 23.6.)
// Keys of heads' own take 3 or 4 slots, whatever fits.
template <int DL, bool SHARED>
struct Pd16 {
  static constexpr int TT = 16, COST = 3, LEAST = 3;
  static constexpr int NCH = DL / 8 + (SHARED ? 8 : 0), RS = NCH % 16 == 8 ? NCH : NCH + 8;
  static constexpr int NKS = NCH / 4, NKW = (NKS + 3) / 4;  // k-steps of the scores; of a wave
  static constexpr int NB = DL / 64;                        // column blocks of 16 a wave
  static constexpr int SLOT = 16 * RS * 16, ROPE = SHARED ? 0 : 16 * 2048, SX = 2 * 4096;
  static constexpr int LIMIT = 160 * 1024;
  static constexpr int NS = SHARED ? std::min(8, (LIMIT - SX - 64) / SLOT) : 4 * SLOT + 3 * ROPE + SX <= LIMIT ? 4 : 3;
  static constexpr int LDS = NS * SLOT + (NS - 1) * ROPE + SX;
  static constexpr int NI = RS / 4 + (SHARED ? 0 : 32), ND = NI / 2;  // loads of 1 KiB a tile; of a loading wave
  static constexpr int THREADS = 384;
  static_assert(NI % 2 == 0 && (NS - 2) * ND <= 63, "vmcnt");
};

__device__ __forceinline__ int tok_swz16(int t) { return ((t >> 2) & 1) | (((t >> 3) & 1) << 1) | (((t >> 1) & 1) << 2); }

// The loading waves: tile k + NS - 1 goes into the slot of tile k - 1 once every wave is done with that (the barrier of tile k), and
// tile k + 1 has landed before that barrier.  The first tiles go out two at a time, so that the first is not waited for behind a whole
// ring.  Past the end nothing is loaded (descriptors of no bytes), so the counts stay the same.
template <int DL, bool SHARED>
__device__ __forceinline__ void paged_load16(const PagedDecodeParams& p, unsigned char* lds, PdCursor<Pd16<DL, SHARED>> load, int lw,
                                             int lane) {
  using C = Pd16<DL, SHARED>;
  constexpr int NR = C::RS / 4;  // row pieces; then 32 key pieces (head j / 2, tokens 8 (j % 2) ..)
  PdPieces<C> pieces = {0, -1, 0, 0, 0, 0, 0};
  PdCursor<C> use = load;
  uint32_t off[NR / 2], roff;
#pragma unroll
  for (int i = 0; i < NR / 2; ++i) {
    const int q = 64 * (lw + 2 * i) + lane, row = q / C::RS, c = (q - row * C::RS) ^ tok_swz16(row);
    off[i] = c < C::NCH ? (uint32_t)(row * p.c.row_bytes + 16 * c) : kPdNothing;
  }
  {
    const int t = 8 * lw + (lane >> 3);
    roff = (uint32_t)(t * p.c.row_bytes + 2 * DL + 16 * ((lane & 7) ^ (t >> 1)));
  }
  uint32_t to = lds_addr(lds) + lw * 1024;
  const uint32_t end = to + C::NS * C::SLOT;
  uint32_t rto = lds_addr(lds) + C::NS * C::SLOT + lw * 1024;
  const uint32_t rend = rto + (C::NS - 1) * C::ROPE;
  auto issue = [&]() {
    int at = 0, nv = 0;
    const int hg = load.hg;
    if (load.more()) {
      at = pieces.lane_of(p, load, 0, lane);
      nv = pieces.tokens_of(at);
      load.next(p);
    }
    const buf_rsrc r = pieces.rows_of(at, (uint32_t)(nv * p.c.row_bytes));
    dma16<VECTOR_DESC>(r, off[0], to);
#pragma unroll
    for (int i = 1; i < NR / 2; ++i) dma16(r, off[i], to + i * 2048);
    if constexpr (!SHARED) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int h = hg * 16 + i;
        dma16(r, h < p.H ? roff + (uint32_t)h * 128 : kPdNothing, rto + i * 2048);
      }
      rto = rto + C::ROPE == rend ? rend - (C::NS - 1) * C::ROPE : rto + C::ROPE;
    }
    to = to + C::SLOT == end ? end - C::NS * C::SLOT : to + C::SLOT;
  };
  issue();
  issue();
  wait_loads<C::ND>();
  pd_barrier();
  constexpr int more = std::min(2, C::NS - 3), ramp = std::max(0, C::NS - 5);
#pragma unroll
  for (int i = 0; i < more; ++i) issue();
  auto ramp_up = [&](auto k) {
    if (!use.more()) return;
    wait_loads<(k + 2) * C::ND>();
    pd_barrier();
    issue();
    issue();
    use.next(p);
  };
  if constexpr (ramp > 0) ramp_up(std::integral_constant<int, 0>{});
  if constexpr (ramp > 1) ramp_up(std::integral_constant<int, 1>{});
  if constexpr (ramp > 2) ramp_up(std::integral_constant<int, 2>{});
  static_assert(ramp <= 3, "");
#pragma unroll 1
  for (; use.more(); use.next(p)) {
    wait_loads<(C::NS - 3) * C::ND>();
    pd_barrier();
    issue();
  }
  wait_loads<0>();  // (loads of nothing into the ring)
}

template <int DL, bool SHARED>
__global__ __launch_bounds__(384, 1) void paged_decode16_kernel(PagedDecodeParams p) {
  using C = Pd16<DL, SHARED>;
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  unsigned char* ropes = lds + C::NS * C::SLOT;
  f32x4* sx = reinterpret_cast<f32x4*>(ropes + (C::NS - 1) * C::ROPE);  // [2][4 waves][64]
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, G = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  PdCursor<C> use = pd_begin<C>(p, blockIdx.x, lane);
  if (!use.more()) return;
  if (w >= 4) {
    paged_load16<DL, SHARED>(p, lds, use, w - 4, lane);
    return;
  }

  const int swA = tok_swz16(l16);
  const int offA = l16 * C::RS * 16 + ((4 * (w & 1) + G) ^ swA) * 16 + (w >> 1) * 128;  // k-step w; w + 4 i: + 256 i
  const int rowB = 4 * G + (l16 >> 2), swB = tok_swz16(rowB);
  const int offB = rowB * C::RS * 16 + (((2 * w) ^ (swB & 6)) + ((((l16 & 3) >> 1) ^ swB) & 1)) * 16 + (l16 & 1) * 8;  // block w + 4 i: + 128 i
  const int offR = l16 * 128 + ((G ^ (l16 >> 1)) * 16);  // k-step 1: chunk 4 further, ^ 64

  PdPieces<C> pieces = {0, -1, 0, 0, 0, 0, 0};
  u32x4 q[C::NKW], qr[SHARED ? 1 : 8];
  f32x4 o[C::NB];
  float m_run = 0.f, l_part = 0.f;
  int slot = 0, rope = 0, par = 0, from = 0;
  bool first = true, started = false;
  while (true) {
    if (first) {  // a unit begins
      const int h = use.hg * 16 + l16;
      const bf16* ql = p.q_lat + use.b * p.q_lat_sb + (int64_t)h * p.q_lat_sh;
      const bf16* qp = p.q_rope + use.b * p.q_rope_sb + (int64_t)h * p.q_rope_sh;
#pragma unroll
      for (int i = 0; i < C::NKW; ++i) {
        const int c = 4 * (w + 4 * i) + G;
        q[i] = u32x4{0u, 0u, 0u, 0u};
        if (w + 4 * i < C::NKS && h < p.H) q[i] = c < DL / 8 ? ldg16(ql + 8 * c) : ldg16(qp + 8 * (c - DL / 8));
      }
      if constexpr (!SHARED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // heads 4 w + j / 2, the same in every column
          const int hj = min(use.hg * 16 + 4 * w + (j >> 1), p.H - 1);
          qr[j] = ldg16(p.q_rope + use.b * p.q_rope_sb + (int64_t)hj * p.q_rope_sh + 32 * (j & 1) + 8 * G);
        }
      }
#pragma unroll
      for (int i = 0; i < C::NB; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run = -INFINITY;
      l_part = 0.f;
      from = use.tile;
      first = false;
      if (!started) pd_barrier();  // the first tile has landed
      started = true;
    }
    const int nv = pieces.tokens_of(pieces.lane_of(p, use, 0, lane));
    const unsigned char* buf = lds + slot * C::SLOT;
    // the wave's part of S^T: S[token 4 G + r][head l16]
    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
    u32x4 a[C::NKW];
#pragma unroll
    for (int i = 0; i < C::NKS / 4; ++i) a[i] = lds16(buf + offA + 256 * i);
    if (C::NKW > C::NKS / 4 && w < C::NKS % 4) {
      a[C::NKW - 1] = lds16(buf + offA + 256 * (C::NKW - 1));
      s = mfma16(as_bf16x8(a[C::NKW - 1]), as_bf16x8(q[C::NKW - 1]), s);
    }
#pragma unroll
    for (int i = 0; i < C::NKS / 4; ++i) s = mfma16(as_bf16x8(a[i]), as_bf16x8(q[i]), s);
    if constexpr (!SHARED) {
      const unsigned char* rb = ropes + rope * C::ROPE + 4 * w * 2048;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 d = mfma16(as_bf16x8(lds16(rb + j * 2048 + offR)), as_bf16x8(qr[2 * j]), f32x4{0.f, 0.f, 0.f, 0.f});
        d = mfma16(as_bf16x8(lds16(rb + j * 2048 + (offR ^ 64))), as_bf16x8(qr[2 * j + 1]), d);
        // (each head's own product: one chain over the heads would carry a head's infinities into the others)
        const bool mine = l16 == 4 * w + j;
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] += mine ? d[r] : 0.f;
      }
      rope = rope + 1 == C::NS - 1 ? 0 : rope + 1;
    }
    sx[(par * 4 + w) * 64 + lane] = s;
    pd_barrier();  // every part of S, the next tile, and every wave done with the last one's slot

    f32x4 x = sx[(par * 4) * 64 + lane];
    x += sx[(par * 4 + 1) * 64 + lane];
    x += sx[(par * 4 + 2) * 64 + lane];
    x += sx[(par * 4 + 3) * 64 + lane];
    par ^= 1;
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = 4 * G + r < nv ? x[r] * p.scale_log2 : -INFINITY;
      top = fmaxf(top, x[r]);
    }
    top = xor32_max(xor16_max(top));
    if (__any(top > m_run + kPdRescale)) {
      const float m_new = fmaxf(m_run, top), alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
      m_run = m_new;
      l_part *= alpha;
#pragma unroll
      for (int i = 0; i < C::NB; ++i) o[i] *= alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = fast_exp2(x[r] - m_use);
      l_part += x[r];
    }
    const s16x4 pa = __builtin_bit_cast(s16x4, u32x2{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])});
#pragma unroll
    for (int i = 0; i < C::NB; ++i) {
      const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(buf + offB + 128 * i));
      o[i] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, pa, o[i], 0, 0, 0);
    }
    slot = slot + 1 == C::NS ? 0 : slot + 1;

    const int b = use.b, hg = use.hg, n = use.n, tile = use.tile;
    use.next(p);
    if (tile + 1 == n || !use.more()) {
      const PdOut<DL> out(use, from, tile, n);
      const float l = xor32_sum(xor16_sum(l_part)), inv = l == 0.f ? 0.f : 1.f / l;
      const int h = hg * 16 + l16;
#pragma unroll
      for (int i = 0; i < C::NB; ++i) out.columns(p, b, h, l16, 16 * (w + 4 * i) + 4 * G, o[i], inv);
      if (w == 0 && G == 0) out.sums(p, b, hg, h, l16, m_run, l);
      first = true;
      if (!use.more()) break;
    }
  }
}

// ------------------------------------------------------------------------------------------------ 4 bits

// Codes are never turned into their values: (w >> s) & 0x00780078 | 0x41804180 makes two of a word's eight codes the bf16 numbers 16 +
// code, which the matrix instructions take as they are.  With u = 16 + code a run of 64 adds scale (sum u q - 24 sum q) to a score: the
// second sum is the accumulator's start, the scale a factor on the result, one a run and token.  For O the scale goes into p before p is
// rounded to bf16 (one rounding, as in 16 bits), and -24 sum p' is an accumulator of its own, added at the end; there the first two codes of
// eight are 128 + code, w & 0x000f000f | 0x43004300, without a shift.  (In the scores too that would put 1.6e-6 of a single token's lse out,
// 0.6e-6 with 16: these sums are in fp32, and the smaller what cancels the better.)  A code costs about a VALU operation each time,
// twice a token (scores, O); these and the scoring waves' way through a tile, not the memory, bound the kernel.
//
// So three kinds of waves work at once, a tile apart: four load tile i + NS - 2, four score tile i, NA add up tile i - 1.  A scoring wave
// takes 16 of the tile's tokens and leaves p relative to a running max of its own, with that max; an adding wave owns some of the
// latent's columns (a run of 64 where there are registers for a wave each), brings the four to a common max and adds.
// ds_read_b64_tr_b4 gives each lane one column's 16 tokens, those whose p the lane reads as the scores' accumulators left them: token
// 16 t + 4 G + r for t, r < 4.  Waves that did all three one after the other took 60.0 us for 87 MB where these took 33.8.  The scoring waves
// keep to one max (that of all four, a tile late), so that the adding ones seldom have anything to bring together.
//
// Not loading anything would save nothing of the 179 MB's time, not unpacking 11 %: what bounds a tile is a scoring wave's 3000 cycles for
// it, with two adding waves and a loading one on its SIMD.  Reading the next codes ahead took 2 % off, reading them all ahead put 5 % on.
//
// A slot holds rows of RS chunks of 16 bytes, RS odd, every second 16 rows 128 bytes further (2-way bank conflicts in the transpose
// reads, none in the scores' reads), then the runs' scales.  Keys of their own lie apart, [16 tokens' piece][head][token][32 bytes],
// in a ring one slot shorter: only the scores read them.  With a shared key there is room for the scales in fp32 as well, which the loading
// waves, who have time for it, write for all others; what lies behind the sequence's end gets 0, so that a p of 0 stays 0.
template <int DL, bool SHARED, int SLOTS>
struct Pd4 {
  static constexpr int TT = 64, COST = 2, LEAST = 2;
  static constexpr int NCH = DL / 32 + (SHARED ? 2 : 0), RS = NCH + 1;
  static constexpr int NL = DL / 64, NG = NL + (SHARED ? 1 : 16);  // runs of a row: the latent's; with the keys
  static constexpr int NA = SHARED ? NL : 4, NB = DL / 16 / NA;    // adding waves; column blocks of 16 of one
  static constexpr int SUB = 16 * RS * 16, ROWS = 4 * SUB + 256;
  static constexpr int SC = NG * 32;  // bytes of 16 tokens' scales
  static constexpr int SF = 4 * NG * 64;  // a tile's scales in fp32: [16 tokens' piece][run][token]; three tiles'
  static constexpr int SLOT = ROWS + 4 * SC, SX = 2 * 4096 + 2 * 256 + 2 * 256 + (SHARED ? 3 * SF : 1024), LIMIT = 160 * 1024;
  static constexpr int NS = SLOTS;
  // heads with keys of their own that SLOTS slots leave room for
  static constexpr int HEADS = SHARED ? 16 : std::min(16, (LIMIT - SX - NS * SLOT) / (NS - 1) / 2048 / 2 * 2);
  static constexpr int ROPE = SHARED ? 0 : HEADS * 2048;
  static constexpr int LDS = NS * SLOT + (NS - 1) * ROPE + SX;
  static constexpr int NR = (16 * RS + 63) / 64, ND = NR + 1 + (SHARED ? 0 : 8);  // loads of 16 rows; of a loading wave a tile
  static constexpr int THREADS = 64 * (8 + NA);
  static_assert(LDS <= LIMIT && (NS - 2) * ND <= 63 && 2 * NG <= 64 && NS >= 3, "");
};
// where 16-token piece t of a slot begins: pieces 1 and 2 lie 128 bytes off the others
template <int SUB>
__device__ __forceinline__ int piece_at(int t) { return t * SUB + (((t + 1) >> 1) << 7); }

// The masks and bases, as numbers that the compiler does not know: (w & mask) | base is then one instruction, of two literals it makes two.
// (Not the instruction itself in assembly: what it writes may be a matrix instruction's accumulator until just before, and the compiler
// waits for that only before instructions of its own.)
struct Pd4Codes {
  uint32_t mask0 = 0x000f000fu, mask1 = 0x00780078u, base0 = 0x43004300u, base1 = 0x41804180u;
  __device__ __forceinline__ Pd4Codes() {
    asm("" : "+s"(mask0), "+s"(mask1));
    asm("" : "+v"(base0), "+v"(base1));
  }
  __device__ __forceinline__ bf16x8 near(uint32_t w) const {  // 16 + code
    return as_bf16x8(u32x4{((w << 3) & mask1) | base1, ((w >> 1) & mask1) | base1, ((w >> 5) & mask1) | base1, ((w >> 9) & mask1) | base1});
  }
  __device__ __forceinline__ bf16x8 of(uint32_t w) const {  // the first two 128 + code: an operation fewer, sums of three times the size
    return as_bf16x8(u32x4{(w & mask0) | base0, ((w >> 1) & mask1) | base1, ((w >> 5) & mask1) | base1, ((w >> 9) & mask1) | base1});
  }
};
// 8 values in the order in which Pd4Codes leaves the codes: 0 4 1 5 2 6 3 7
__device__ __forceinline__ u32x4 order8(u32x4 v) {
  return u32x4{pack_lo16(v[0], v[2]), pack_hi16(v[0], v[2]), pack_lo16(v[1], v[3]), pack_hi16(v[1], v[3])};
}
__device__ __forceinline__ f32x4 floats4(u32x2 v) { return f32x4{lo_bf16(v[0]), hi_bf16(v[0]), lo_bf16(v[1]), hi_bf16(v[1])}; }
// what takes 16 + code, and 128 + code, back to code - 8
__device__ __forceinline__ bf16x8 minus24() { return as_bf16x8(u32x4{0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u}); }
__device__ __forceinline__ bf16x8 offsets8() { return as_bf16x8(u32x4{0xc308c308u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u}); }

// The loading waves, 16 tokens of a tile each: tile i + NS - 2 goes into the slot of tile i - 2 after the barrier before which tile i has
// landed and tile i - 2 was added up.  The first tiles go out two at a time; past the end nothing is loaded, so the counts stay the same.
template <class C, bool SHARED>
__device__ __forceinline__ void paged_load4(const PagedDecodeParams& p, unsigned char* lds, PdCursor<C> load, int lw, int lane) {
  PdPieces<C> pieces = {0, -1, 0, 0, 0, 0, 0};
  PdCursor<C> use = load;
  uint32_t off[C::NR];
#pragma unroll
  for (int i = 0; i < C::NR; ++i) {
    const int q = 64 * i + lane, row = q / C::RS, c = q - row * C::RS;
    off[i] = c < C::NCH ? (uint32_t)(row * p.c.row_bytes + 16 * c) : kPdNothing;
  }
  const uint32_t koff = (uint32_t)((lane & 31) / 2 * p.c.row_bytes + 32 * C::NL + 32 * (lane >> 5) + 16 * (lane & 1));
  const uint32_t base = lds_addr(lds), keys = base + C::NS * C::SLOT, dump = keys + (C::NS - 1) * C::ROPE + C::SX - 1024;
  const uint32_t scales_bytes = (uint32_t)((p.c.groups - 1) * p.c.size + 16) * 2;
  int slot = 0, kslot = 0;
  uint64_t slot_tokens = 0;  // 8 bits a slot
  auto issue = [&]() {
    const bool more = load.more();
    const int hg = load.hg;
    const uint32_t to = base + slot * C::SLOT;
    int g = lane >> 1;
    if (!SHARED && g >= C::NL) g += 16 * hg;
    const uint32_t sv = g < p.c.groups ? (uint32_t)(g * p.c.size * 2 + 16 * (lane & 1)) : kPdNothing;
    int at = 0, nv = 0;
    if (more) {
      at = pieces.lane_of(p, load, lw, lane);
      nv = pieces.tokens_of(at);
    }
    const buf_rsrc r = pieces.rows_of(at, (uint32_t)(nv * p.c.row_bytes));
    const uint32_t rows_to = to + piece_at<C::SUB>(lw);
    if (lane < 16 * C::RS) dma16<VECTOR_DESC>(r, off[0], rows_to);
#pragma unroll
    for (int i = 1; i < C::NR; ++i)
      if (64 * i + lane < 16 * C::RS) dma16(r, off[i], rows_to + i * 1024);
    const buf_rsrc rs = pieces.scales_of(at, nv ? scales_bytes : 0u);
    if (lane < 2 * C::NG) dma16<VECTOR_DESC>(rs, sv, to + C::ROWS + lw * C::SC);
    if constexpr (!SHARED) {
#pragma unroll
      for (int j = 0; j < 16; j += 2) {  // two heads; past the slot's heads nothing, into bytes that nobody reads
        const int h = hg * 16 + j;
        const uint32_t v = h + (lane >> 5) < p.H ? koff + (uint32_t)h * 32 : kPdNothing;
        dma16(r, j < C::HEADS ? v : kPdNothing, j < C::HEADS ? keys + kslot * C::ROPE + lw * C::HEADS * 512 + j * 512 : dump);
      }
    }
    if (more) load.next(p);
    if (SHARED) slot_tokens = (slot_tokens & ~(0xffull << (8 * slot))) | (uint64_t)nv << (8 * slot);
    slot = slot + 1 == C::NS ? 0 : slot + 1;
    kslot = kslot + 1 == C::NS - 1 ? 0 : kslot + 1;
  };
  // the scales of the next tile to be scored, which has landed, in fp32
  int sslot = 0, sbuf = 0;
  auto scales_out = [&]() {
    if constexpr (SHARED) {
      const int nv = (int)(slot_tokens >> (8 * sslot)) & 0xff, t = 4 * (lane & 3);
      if (lane < 4 * C::NG) {
        f32x4 v = floats4(lds8(lds + sslot * C::SLOT + C::ROWS + lw * C::SC + 8 * lane));
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = t + r < nv ? v[r] : 0.f;
        *reinterpret_cast<f32x4*>(lds + C::NS * C::SLOT + C::SX - 3 * C::SF + sbuf * C::SF + lw * C::NG * 64 + 16 * lane) = v;
      }
      sslot = sslot + 1 == C::NS ? 0 : sslot + 1;
      sbuf = sbuf == 2 ? 0 : sbuf + 1;
    }
  };
  issue();
  if constexpr (C::NS > 3) issue();
  constexpr int ramp = std::max(0, C::NS - 4);
  auto ramp_up = [&](auto k) {
    if (!use.more()) return;
    wait_loads<(k + 1) * C::ND>();
    scales_out();
    pd_barrier();
    issue();
    issue();
    use.next(p);
  };
  if constexpr (ramp > 0) ramp_up(std::integral_constant<int, 0>{});
  if constexpr (ramp > 1) ramp_up(std::integral_constant<int, 1>{});
  if constexpr (ramp > 2) ramp_up(std::integral_constant<int, 2>{});
  if constexpr (ramp > 3) ramp_up(std::integral_constant<int, 3>{});
  static_assert(ramp <= 4, "");
#pragma unroll 1
  for (; use.more(); use.next(p)) {
    wait_loads<(C::NS - 3) * C::ND>();
    scales_out();
    pd_barrier();
    issue();
  }
  pd_barrier();
  wait_loads<0>();  // (loads of nothing into the ring)
}

// p and the max and sum it is relative to, from the scoring waves to the adding ones; two tiles' worth
struct Pd4Shared {
  f32x4* p;  // [2][4 waves][64]
  float* m;  // [2][4][16]
  float* l;  // [2][4][16]: at a unit's end
  const unsigned char* scales;  // a shared key: [3] tiles' in fp32
};

// 4 tokens' scales of run g, in fp32 or bf16
template <bool FP32>
struct Pd4Scales {
  typename std::conditional<FP32, u32x4, u32x2>::type v;
  __device__ __forceinline__ void read(const unsigned char* at, int g) {
    if constexpr (FP32)
      v = lds16(at + 64 * g);
    else
      v = lds8(at + 32 * g);
  }
  __device__ __forceinline__ f32x4 floats() const {
    if constexpr (FP32)
      return __builtin_bit_cast(f32x4, v);
    else
      return floats4(v);
  }
};

template <class C, int DL, bool SHARED>
__device__ __forceinline__ void paged_score4(const PagedDecodeParams& p, unsigned char* lds, const Pd4Shared& x, PdCursor<C> use, int w,
                                             int lane) {
  const int l16 = lane & 15, G = lane >> 4;
  const int offA = piece_at<C::SUB>(w) + l16 * C::RS * 16 + 8 * G;
  PdPieces<C> pieces = {0, -1, 0, 0, 0, 0, 0};
  constexpr int NQ = C::NL + 1;  // the latent's runs, and the key: shared, or this lane's head's
  u32x4 q[2 * NQ];
  // The runs' -24 scale sum q come from one product: the tile's scales (rows: tokens) with -24 sum q in three bf16 pieces (24 bits) as
  // its columns: K slots 8 G .. of group G < 3 are piece G of the latent's runs, of group 3 the pieces of the shared key's.
  bf16x8 start;
  f32x4 key_start;  // keys of their own: of this lane's head's, the start of its sums
  float m_run = 0.f, l_part = 0.f;
  const int offS = ((l16 >> 2) & 3) * 32 + (l16 & 3) * 8;  // transpose read: row (run) i / 4, tokens 4 (i % 4) ..
  const Pd4Codes codes;
  int slot = 0, kslot = 0, par = 0, sbuf = 0;
  bool first = true;
#pragma unroll 1
  while (true) {
    if (first) {
      const int h = min(use.hg * 16 + l16, p.H - 1);  // (past the last head the last again: under a condition each load would be waited for)
      const bf16* ql = p.q_lat + use.b * p.q_lat_sb + (int64_t)h * p.q_lat_sh;
      const bf16* qp = p.q_rope + use.b * p.q_rope_sb + (int64_t)h * p.q_rope_sh;
#pragma unroll
      for (int i = 0; i < 2 * NQ; ++i) {
        const int c = 64 * (i >> 1) + 16 * G + 8 * (i & 1);
        q[i] = i < 2 * C::NL ? ldg16(ql + c) : ldg16(qp + c - DL);
      }
#pragma unroll
      for (int i = 0; i < 2 * NQ; ++i) q[i] = order8(q[i]);
      float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < NQ; ++g) {
        f32x4 d = mfma16(minus24(), as_bf16x8(q[2 * g]), f32x4{0.f, 0.f, 0.f, 0.f});
        d = mfma16(minus24(), as_bf16x8(q[2 * g + 1]), d);
        if (g < C::NL)
          z[g] = d[0];
        else
          key_start = d;
      }
      if (!SHARED && G == 3) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = 0.f;
      }
      if (SHARED && G == 3) {
        const bf16 hi = (bf16)key_start[0], mid = (bf16)(key_start[0] - (float)hi);
        z[0] = (float)hi;
        z[1] = (float)mid;
        z[2] = key_start[0] - (float)hi - (float)mid;
#pragma unroll
        for (int e = 3; e < 8; ++e) z[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float hi = (float)(bf16)z[e], mid = (float)(bf16)(z[e] - hi);
        start[e] = (bf16)(G == 0 || G == 3 ? z[e] : G == 1 ? z[e] - hi : z[e] - hi - mid);
      }
      m_run = -INFINITY;
      l_part = 0.f;
    }
    pd_barrier();  // the tile has landed, and the tile before the last is added up
    if (!first) {  // the largest of the four waves' maxima from now on, so that the adding waves find one for all (mostly it is)
      const float* m = x.m + (par ^ 1) * 64 + l16;
      const float top = fmaxf(fmaxf(m[0], m[16]), fmaxf(m[32], m[48]));
      if (__any(top > m_run)) {
        l_part *= top > m_run ? fast_exp2(m_run - top) : 1.f;
        m_run = fmaxf(m_run, top);
      }
    }
    const unsigned char* buf = lds + slot * C::SLOT;
    unsigned char* sc = lds + slot * C::SLOT + C::ROWS + w * C::SC;
    const int nv = pieces.tokens_of(pieces.lane_of(p, use, w, lane));
    if (!SHARED && nv < 16) {  // scales behind the sequence's end may be anything: 0, so that a p of 0 stays 0
      for (int i = lane; i < C::NG * 16; i += 64)
        if ((i & 15) >= nv) reinterpret_cast<unsigned short*>(sc)[i] = 0;
    }
    f32x4 s;
    {
      // rows 0 .. 3 and 4 .. 7 of the runs (past the latent's the first again: their pieces are 0); group 3: the key's, four times
      const int a0 = G == 3 && SHARED ? C::NL * 32 + (l16 & 3) * 8 : C::NL >= 4 ? offS : (l16 >> 2) < C::NL ? offS : (l16 & 3) * 8;
      const int a1 = C::NL >= 8 || (C::NL > 4 && 4 + (l16 >> 2) < C::NL) ? offS + 128 : (l16 & 3) * 8;
      const s16x4 r0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sc + a0));
      const s16x4 r1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sc + a1));
      const u32x2 w0 = __builtin_bit_cast(u32x2, r0), w1 = __builtin_bit_cast(u32x2, r1);
      s = mfma16(as_bf16x8(u32x4{w0[0], w0[1], w1[0], w1[1]}), start, f32x4{0.f, 0.f, 0.f, 0.f});
    }
    constexpr int RUNS = C::NL + (SHARED ? 1 : 0), AHEAD = SHARED ? 1 : 2;
    u32x2 codes_of[AHEAD + 1];
    Pd4Scales<SHARED> scales_of[AHEAD + 1];
    const unsigned char* scales = SHARED ? x.scales + sbuf * C::SF + w * C::NG * 64 + 16 * G : sc + 8 * G;
    auto read = [&](int g) {
      if (g >= RUNS) return;
      codes_of[g % (AHEAD + 1)] = lds8(buf + offA + 32 * g);
      scales_of[g % (AHEAD + 1)].read(scales, g);
    };
#pragma unroll
    for (int g = 0; g < AHEAD; ++g) read(g);
#pragma unroll
    for (int g = 0; g < RUNS; ++g) {
      read(g + AHEAD);
      asm volatile("" ::: "memory");  // (read here: left to itself the compiler reads and waits)
      const u32x2 c = codes_of[g % (AHEAD + 1)];
      const f32x4 k = scales_of[g % (AHEAD + 1)].floats();
      f32x4 d = mfma16(codes.near(c[0]), as_bf16x8(q[2 * g]), f32x4{0.f, 0.f, 0.f, 0.f});
      d = mfma16(codes.near(c[1]), as_bf16x8(q[2 * g + 1]), d);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(k[r], d[r], s[r]);
    }
    sbuf = sbuf == 2 ? 0 : sbuf + 1;
    if constexpr (!SHARED) {
      // head j's keys with every head's query: lane l16 keeps its own.  The scale of its key comes last.
      const unsigned char* kb = lds + C::NS * C::SLOT + kslot * C::ROPE + w * C::HEADS * 512 + l16 * 32 + 8 * G;
      f32x4 e = f32x4{0.f, 0.f, 0.f, 0.f};
      u32x2 ahead = lds8(kb);
      const u32x2 ks = lds8(sc + 32 * (C::NL + l16) + 8 * G);
#pragma unroll
      for (int j = 0; j < C::HEADS; ++j) {
        const u32x2 c = ahead;
        if (j + 1 < C::HEADS) ahead = lds8(kb + (j + 1) * 512);
        asm volatile("" ::: "memory");
        f32x4 d = mfma16(codes.near(c[0]), as_bf16x8(q[2 * C::NL]), key_start);
        d = mfma16(codes.near(c[1]), as_bf16x8(q[2 * C::NL + 1]), d);
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = l16 == j ? d[r] : e[r];
      }
      const f32x4 k = floats4(ks);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(k[r], e[r], s[r]);
      kslot = kslot + 1 == C::NS - 1 ? 0 : kslot + 1;
    }
    float top = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = 4 * G + r < nv ? s[r] * p.scale_log2 : -INFINITY;
      top = fmaxf(top, s[r]);
    }
    top = xor32_max(xor16_max(top));
    if (__any(top > m_run + kPdRescale)) {
      const float m_new = fmaxf(m_run, top);
      l_part *= m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
      m_run = m_new;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = fast_exp2(s[r] - m_use);
      l_part += s[r];
    }
    x.p[(par * 4 + w) * 64 + lane] = s;
    if (G == 0) x.m[(par * 4 + w) * 16 + l16] = m_run;
    const bool last = use.tile + 1 == use.n || use.left == 1;
    if (last) {
      const float l = xor32_sum(xor16_sum(l_part));
      if (G == 0) x.l[(par * 4 + w) * 16 + l16] = l;
    }
    par ^= 1;
    slot = slot + 1 == C::NS ? 0 : slot + 1;
    first = last;
    use.next(p);
    if (!use.more()) break;
  }
  pd_barrier();
}

template <class C, int DL, bool SHARED>
__device__ __forceinline__ void paged_add4(const PagedDecodeParams& p, const unsigned char* lds, const Pd4Shared& x, PdCursor<C> use, int w,
                                           int lane) {
  const int l16 = lane & 15, G = lane >> 4;
  // transpose reads: lane i of a group of 16 gives the row of token 16 (i / 4) + 4 G + i % 4
  const int offT = piece_at<C::SUB>(l16 >> 2) + (4 * G + (l16 & 3)) * C::RS * 16 + 8 * w * C::NB;
  const int g0 = w * C::NB / 4;  // the run of the wave's first column block
  f32x4 o[C::NB], os[2];
  const Pd4Codes codes;
  float M = 0.f;
  int slot = 0, par = 0, from = 0, sbuf = 0;
  bool first = true;
  pd_barrier();
#pragma unroll 1
  while (true) {
    if (first) {
#pragma unroll
      for (int i = 0; i < C::NB; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      os[0] = os[1] = f32x4{0.f, 0.f, 0.f, 0.f};
      M = -INFINITY;
      from = use.tile;
    }
    const unsigned char* buf = lds + slot * C::SLOT;
    const unsigned char* sc = buf + C::ROWS;
    i32x2 c[C::NB];  // (the tile landed a barrier ago)
#pragma unroll
    for (int i = 0; i < C::NB; ++i) c[i] = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2*)(buf + offT + 8 * i));
    pd_barrier();  // the tile is scored
    float m[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) m[t] = x.m[(par * 4 + t) * 16 + l16];
    f32x4 pv[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) pv[t] = x.p[(par * 4 + t) * 64 + lane];
    constexpr int NG = C::NB > 4 ? 2 : 1;  // runs that the wave's columns can touch
    Pd4Scales<SHARED> k[NG][4];
    const unsigned char* scales = SHARED ? x.scales + sbuf * C::SF + 16 * G : sc + 8 * G;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int t = 0; t < 4; ++t) k[g][t].read(scales + t * (SHARED ? C::NG * 64 : C::SC), min(g0 + g, C::NL - 1));
    sbuf = sbuf == 2 ? 0 : sbuf + 1;
    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    if (__any(top > M)) {
      const float m_new = fmaxf(M, top), alpha = m_new == -INFINITY ? 1.f : fast_exp2(M - m_new);
      M = m_new;
#pragma unroll
      for (int i = 0; i < C::NB; ++i) o[i] *= alpha;
      os[0] *= alpha;
      os[1] *= alpha;
    }
    if (__any(fminf(fminf(m[0], m[1]), fminf(m[2], m[3])) != M)) {  // what brings a wave's p (and l) to the common max
      const float M_use = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        m[t] = fast_exp2(m[t] - M_use);
        pv[t] *= m[t];
      }
    } else {
      m[0] = m[1] = m[2] = m[3] = 1.f;
    }
    bf16x8 pb[2];
#pragma unroll
    for (int i = 0; i < C::NB; ++i) {
      const int nb = w * C::NB + i, g = nb >> 2;
      if (i == 0 || (nb & 3) == 0) {  // the run's scales into p
        f32x4 e[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) e[t] = pv[t] * k[g == g0 ? 0 : 1][t].floats();
#pragma unroll
        for (int t = 0; t < 2; ++t)
          pb[t] = as_bf16x8(u32x4{pack_bf16x2(e[2 * t][0], e[2 * t + 1][0]), pack_bf16x2(e[2 * t][1], e[2 * t + 1][1]),
                                  pack_bf16x2(e[2 * t][2], e[2 * t + 1][2]), pack_bf16x2(e[2 * t][3], e[2 * t + 1][3])});
        if (g == g0) {
          os[0] = mfma16(offsets8(), pb[0], os[0]);
          os[0] = mfma16(offsets8(), pb[1], os[0]);
        } else {
          os[1] = mfma16(offsets8(), pb[0], os[1]);
          os[1] = mfma16(offsets8(), pb[1], os[1]);
        }
      }
      o[i] = mfma16(codes.of((uint32_t)c[i][0]), pb[0], o[i]);
      o[i] = mfma16(codes.of((uint32_t)c[i][1]), pb[1], o[i]);
    }
    slot = slot + 1 == C::NS ? 0 : slot + 1;
    const int b = use.b, hg = use.hg, n = use.n, tile = use.tile;
    use.next(p);
    first = tile + 1 == n || !use.more();
    if (first) {
      const PdOut<DL> out(use, from, tile, n);
      float l = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) l += x.l[(par * 4 + t) * 16 + l16] * m[t];
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int h = hg * 16 + l16;
#pragma unroll
      for (int i = 0; i < C::NB; ++i) {
        const int nb = w * C::NB + i;
        out.columns(p, b, h, l16, 16 * nb + 4 * G, o[i] + ((nb >> 2) == g0 ? os[0] : os[1]), inv);
      }
      if (w == 0 && G == 0) out.sums(p, b, hg, h, l16, M, l);
      if (!use.more()) break;
    }
    par ^= 1;
  }
}

template <int DL, bool SHARED, int SLOTS>
__global__ __launch_bounds__((Pd4<DL, SHARED, SLOTS>::THREADS), 1) void paged_decode4_kernel(PagedDecodeParams p) {
  using C = Pd4<DL, SHARED, SLOTS>;
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  unsigned char* at = lds + C::NS * C::SLOT + (C::NS - 1) * C::ROPE;
  const Pd4Shared x = {reinterpret_cast<f32x4*>(at), reinterpret_cast<float*>(at + 8192), reinterpret_cast<float*>(at + 8192 + 512), at + 8192 + 1024};
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const PdCursor<C> use = pd_begin<C>(p, blockIdx.x, lane);
  if (!use.more()) return;
  if (w < 4)
    paged_score4<C, DL, SHARED>(p, lds, x, use, w, lane);
  else if (w < 4 + C::NA)
    paged_add4<C, DL, SHARED>(p, lds, x, use, w - 4, lane);
  else {
    __builtin_amdgcn_s_setprio(3);  // (a load that goes out late delays all; 9.6 us for one sequence where it took 10.4)
    paged_load4<C, SHARED>(p, lds, use, w - 4 - C::NA, lane);
  }
}

// ------------------------------------------------------------------------------------------------ parts

// One workgroup a head of a sequence: nothing where one run finished it, zeros for a sequence without tokens, else the sum of the
// runs' parts, 2^(m - M) of each.  Which runs those are the first of them has left.  Latency: that, then m, l and 8 parts a thread at
// once (3.9 us for one sequence, 6 for 64 of 16 heads, of which a launch alone is 2).  The last run of a unit to end could add the parts instead.
template <int DL, class C>  // (C: the kernel whose parts they are, so that a trace tells)
__global__ __launch_bounds__(512) void paged_merge_kernel(PagedDecodeParams p) {
  constexpr int COLS = DL / 4, PARTS = 512 / COLS;  // threads of a part; parts at a time
  __shared__ f32x4 o_s[PARTS][COLS];
  const int b = blockIdx.x, h = blockIdx.y, hg = h >> 4, l16 = h & 15;
  const int tid = threadIdx.x, lane = tid & 63;
  const int len = pd_len(p, b), unit = p.units[(int64_t)b * p.n_hg + hg];
  const int64_t row = (int64_t)b * p.H + h;
  if (len == 0) {  // (no run has it)
    if (tid < COLS) stg8(p.ctx + row * DL + 4 * tid, u32x2{0u, 0u});
    if (tid == 0) p.lse[row] = -INFINITY;
    return;
  }
  const int run0 = unit & 0xffff, S = unit >> 16;
  if (S == 1) return;
  auto part_of = [&](int s) { return ((int64_t)2 * (run0 + s) + (s == 0 ? 1 : 0)) * 16 + l16; };
  const int part = tid / COLS, col = tid - part * COLS;
  const bool in = part < PARTS;  // (COLS need not divide the workgroup)
  float M = -INFINITY, L = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < S; s0 += 8 * PARTS) {
    f32x4 v[8];
    float m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[i] = -INFINITY;
      if (in && s0 + part + i * PARTS < S) {
        const int64_t at = part_of(s0 + part + i * PARTS);
        v[i] = *reinterpret_cast<const f32x4*>(p.part_o + at * DL + 4 * col);
        m[i] = p.part_ml[2 * at];
      }
    }
    static_assert(8 * PARTS <= 256, "");
    float ms = -INFINITY, ls = 0.f, mk[4], lk[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = s0 + lane + 64 * k;
      const bool is = lane + 64 * k < 8 * PARTS && s < S;
      const int64_t at = part_of(is ? s : 0);
      mk[k] = is ? p.part_ml[2 * at] : -INFINITY;
      lk[k] = is ? p.part_ml[2 * at + 1] : 0.f;
      ms = fmaxf(ms, mk[k]);
    }
    for (int x = 8; x; x >>= 1) ms = fmaxf(ms, wave_shfl_xor(ms, x));
    ms = fmaxf(M, xor32_max(xor16_max(ms)));
    const float mu = ms == -INFINITY ? 0.f : ms, a = fast_exp2(M - mu);  // (M = -inf: 0, and the sums are 0)
    M = ms;
#pragma unroll
    for (int k = 0; k < 4; ++k) ls += lk[k] * fast_exp2(mk[k] - mu);
    for (int x = 8; x; x >>= 1) ls += wave_shfl_xor(ls, x);
    L = L * a + xor32_sum(xor16_sum(ls));
    o *= a;
#pragma unroll
    for (int i = 0; i < 8; ++i) o += v[i] * fast_exp2(m[i] - mu);
  }
  if (in) o_s[part][col] = o;
  __syncthreads();
  if (part == 0) {
#pragma unroll
    for (int i = 1; i < PARTS; ++i) o += o_s[i][col];
    o *= L == 0.f ? 0.f : 1.f / L;
    stg8(p.ctx + row * DL + 4 * col, u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])});
    if (col == 0) p.lse[row] = L == 0.f ? -INFINITY : (M + fast_log2(L)) * kLn2;
  }
}

// ------------------------------------------------------------------------------------------------ host

// Slots of the ring in 4 bits: as many as fit, 8 at most; with keys of their own 4, or 3 where 4 leave no room for the heads' (more than 14
// of d_latent 384, 10 of 512).
template <int DL>
constexpr int slots4() {
  using C = Pd4<DL, true, 3>;
  return std::min(8, (C::LIMIT - C::SX) / C::SLOT);
}
// Runs: a workgroup for each place that the card has (LDS bounds them), no more than there can be tiles.
template <class C>
int runs_of(int64_t B, int64_t n_hg, int64_t capacity) {
  const int64_t places = 256 * std::max(1, std::min(2, 160 * 1024 / C::LDS));
  const int64_t line = B * n_hg * ((capacity + C::TT - 1) / C::TT + C::COST);  // (below 2^30)
  return (int)std::max<int64_t>(1, std::min(places, (line + C::LEAST - 1) / C::LEAST));
}
// f.take<kernel's constants>() for the kernel that serves the layout
template <int DL, bool SHARED, class F>
auto by_kernel(const mla_paged_cache& c, int64_t H, F&& f) {
  if (!c.scales) return f.template take<DL, SHARED, Pd16<DL, SHARED>>(paged_decode16_kernel<DL, SHARED>);
  if constexpr (SHARED) {
    constexpr int S = slots4<DL>();
    return f.template take<DL, SHARED, Pd4<DL, true, S>>(paged_decode4_kernel<DL, true, S>);
  } else {
    if constexpr (Pd4<DL, false, 4>::HEADS < 16) {
      if (std::min<int64_t>(H, 16) > Pd4<DL, false, 4>::HEADS)
        return f.template take<DL, SHARED, Pd4<DL, false, 3>>(paged_decode4_kernel<DL, false, 3>);
    }
    return f.template take<DL, SHARED, Pd4<DL, false, 4>>(paged_decode4_kernel<DL, false, 4>);
  }
}

template <class F>
auto by_layout(const mla_paged_cache& c, int64_t H, F&& f) {
  const bool shared = c.n_k_rope_heads == 1;
  switch (c.d_latent) {
    case 64: return shared ? by_kernel<64, true>(c, H, f) : by_kernel<64, false>(c, H, f);
    case 128: return shared ? by_kernel<128, true>(c, H, f) : by_kernel<128, false>(c, H, f);
    case 256: return shared ? by_kernel<256, true>(c, H, f) : by_kernel<256, false>(c, H, f);
    case 384: return shared ? by_kernel<384, true>(c, H, f) : by_kernel<384, false>(c, H, f);
    default: return shared ? by_kernel<512, true>(c, H, f) : by_kernel<512, false>(c, H, f);
  }
}
struct RunsOf {
  const mla_paged_decode_args& a;
  template <int DL, bool SHARED, class C, class K>
  int take(K) {
    return runs_of<C>(a.B, (a.H + 15) / 16, a.cache.table_pages * a.cache.page_size);
  }
};
struct LaunchOf {
  PagedDecodeParams& p;
  const char* op;
  hipStream_t st;
  template <int DL, bool SHARED, class C, class K>
  int take(K kernel) {
    kernel<<<dim3(p.runs), C::THREADS, 0, st>>>(p);
    MLA_TRY(launch_status(op));
    // (heads in a dimension of their own: a grid has less than 2^32 threads along each)
    paged_merge_kernel<DL, C><<<dim3((unsigned)p.B, (unsigned)p.H), 512, 0, st>>>(p);
    return launch_status(op);
  }
};

int decode_check(const mla_paged_decode_args* a, const char* op, PagedDecodeParams& p) {
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_CHECK(a->B >= 0 && a->B < (1 << 20) && a->H >= 1 && a->H <= 1024, MLA_ERR_INVALID_ARG, "%s: B %lld or H %lld is out of range", op,
            (long long)a->B, (long long)a->H);
  MLA_TRY(paged_setup(a->cache, op, a->B, p.c));
  MLA_CHECK(a->cache.table_pages * a->cache.page_size < (1ll << 28), MLA_ERR_INVALID_ARG, "%s: table_pages %lld is out of range", op,
            (long long)a->cache.table_pages);
  MLA_CHECK(a->B * ((a->H + 15) / 16) * (a->cache.table_pages * a->cache.page_size / 16 + 4) < (1ll << 30), MLA_ERR_INVALID_ARG,
            "%s: B %lld sequences of %lld pages are too many", op, (long long)a->B, (long long)a->cache.table_pages);
  MLA_CHECK(a->cache.n_k_rope_heads == 1 || a->cache.n_k_rope_heads == a->H, MLA_ERR_INVALID_ARG,
            "%s: n_k_rope_heads must be 1 or H (%lld)", op, (long long)a->H);
  return MLA_OK;
}
size_t parts_bytes(int runs, int64_t DL) { return (size_t)2 * runs * 16 * ((size_t)DL + 2) * 4; }
size_t units_bytes(const mla_paged_decode_args& a) { return (size_t)a.B * ((a.H + 15) / 16) * 4; }

}  // namespace mla

using namespace mla;

extern "C" size_t mla_paged_decode_workspace_bytes(const mla_paged_decode_args* a) {
  PagedDecodeParams p;
  if (decode_check(a, "mla_paged_decode_workspace_bytes", p) != MLA_OK || a->B == 0) return 0;
  return parts_bytes(by_layout(a->cache, a->H, RunsOf{*a}), a->cache.d_latent) + units_bytes(*a);
}

extern "C" int mla_paged_decode(const mla_paged_decode_args* a, void* stream) {
  const char* op = "mla_paged_decode";
  PagedDecodeParams p;
  MLA_TRY(decode_check(a, op, p));
  MLA_TRY(check_scale(op, a->scale));
  if (a->B == 0) return MLA_OK;
  MLA_CHECK(a->q_lat && a->q_rope && a->seq_lens && a->ctx && a->lse, MLA_ERR_INVALID_ARG, "%s: null pointer", op);
  MLA_CHECK((((uintptr_t)a->q_lat | (uintptr_t)a->q_rope | (uintptr_t)a->ctx) & 15) == 0 && (((uintptr_t)a->seq_lens | (uintptr_t)a->lse) & 3) == 0,
            MLA_ERR_INVALID_ARG, "%s: a pointer is not aligned", op);
  const int64_t st[] = {a->q_lat_sb, a->q_lat_sh, a->q_rope_sb, a->q_rope_sh};
  for (int64_t s : st) MLA_CHECK(s >= 0 && (s & 7) == 0, MLA_ERR_INVALID_ARG, "%s: strides must be non-negative multiples of 8", op);
  const size_t need = mla_paged_decode_workspace_bytes(a);
  MLA_CHECK(a->workspace && ((uintptr_t)a->workspace & 255) == 0 && a->workspace_bytes >= need, MLA_ERR_WORKSPACE,
            "%s: needs %zu bytes of 256-byte aligned workspace", op, need);
  p.q_lat = (const bf16*)a->q_lat;
  p.q_rope = (const bf16*)a->q_rope;
  p.seq_lens = a->seq_lens;
  p.ctx = (bf16*)a->ctx;
  p.lse = a->lse;
  p.B = (int)a->B;
  p.H = (int)a->H;
  p.n_hg = (int)((a->H + 15) / 16);
  p.pieces = p.c.size / 16;
  p.piece_magic = p.pieces == 1 ? 0 : (uint32_t)(((1ull << 32) + p.pieces - 1) / p.pieces);
  p.q_lat_sb = a->q_lat_sb;
  p.q_lat_sh = a->q_lat_sh;
  p.q_rope_sb = a->q_rope_sb;
  p.q_rope_sh = a->q_rope_sh;
  p.scale_log2 = a->scale * kLog2e;
  p.runs = by_layout(a->cache, a->H, RunsOf{*a});
  p.part_o = (float*)a->workspace;
  p.part_ml = p.part_o + (size_t)2 * p.runs * 16 * a->cache.d_latent;
  p.units = (int32_t*)(p.part_ml + (size_t)2 * p.runs * 16 * 2);
  return by_layout(a->cache, a->H, LaunchOf{p, op, (hipStream_t)stream});
}
