// Drawing one token for each row of logits: temperature, top-k, top-p, min-p and the draw from a given number (gfx950).
//
// A row's bytes are little (131 KB of 32768 fp32 logits); what bounds it is a workgroup's passes over it one after the other, and in
// those the weights (30 instructions each).  Measured (kernel trace): one row of 32768 bf16, top_k 50, top_p 0.95: 7.9 us; 256 rows of
// 32768 fp32 (34 MB), each with settings of its own: 34, which is the slowest row's time.  Of that row's 70000 cycles 7000 are the load,
// 20000 each of two passes over its weights (top_p over a flat row: most of it is kept), 16000 what lies between them.
#include <cmath>
#include <cstddef>
#include <type_traits>

#include "mla_common.h"

namespace mla {

constexpr int kSmThreads = 1024;
constexpr int kSmMaxV = 1 << 19;  // 2^19 weights of up to 2^44 add up to 2^63 at most: unsigned 64 bits hold it
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmBins = 2048, kSmPerNat = 64;  // 32 nats: what lies lower weighs less than half of 2^-44
constexpr int kSmRuns = kSmMaxV / 256 + kSmThreads / 64;
constexpr int kSmList = 512;
constexpr float kSmMost = 3.402823466e38f;
constexpr double kSmOne = 17592186044416.0;  // 2^44: the largest weight

struct SampleParams {
  const void* logits;
  const float *u, *temperature_rows, *top_p_rows, *min_p_rows;
  const int32_t* top_k_rows;
  int64_t* tokens;
  float* logprobs;
  int64_t stride;
  int V;
  float temperature, top_p, min_p;
  int top_k;
};

// A float's place in the order of values: NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t sm_key(float x) {
  const uint32_t b = __float_as_uint(x != x ? -INFINITY : x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

typedef unsigned long long u64;
#define SM_INLINE __attribute__((always_inline))  // a call would put what its lambda refers to into memory

// 2^(44 + i / 32)
__constant__ const double kSmTable[32] = {
    17592186044416.0, 17977404757381.453, 18371058661769.06, 18773332464219.316, 19184414915921.48, 19604498901177.664,
    20033781527906.22, 20472464220126.88, 20920752812471.082, 21378857646761.793, 21846993670708.133, 22325380538761.176,
    22814242715178.152, 23313809579343.508, 23824315533396.16, 24346000112213.52, 24879108095803.8, 25423889624159.453,
    25980600314625.527, 26549501381838.074, 27130859760288.855, 27724948229573.895, 28332045542384.562, 28952436555301.363,
    29586412362451.676, 30234270432094.277, 30896314746194.61, 31572855943056.41, 32264211463076.527, 32970705697691.37,
    33692670141584.85, 34430443548229.25,
};

// 2^y for y <= 0 in whole steps of 2^-44: 2^(n / 32) from a table times 2^(r / 32), |r| <= 1/2, as 1 + r q(r) with q the interpolation of
// degree 3 at the Chebyshev nodes: within 1.6e-13, in fp64 throughout (a token whose number falls that near a border could come out
// as its neighbour).  The additions of 1.5 2^52 and 2^52 round to whole numbers and leave them in the low bits: fp64 additions and
// products run at the full rate, conversions and exponent operations do not.
constexpr u64 kSmBias = 0x433ull << 52;
struct SmWeight {
  double w;  // in units of 2^-44, before the rounding
  u64 bits;  // kSmBias + the weight: sums of n of them less n kSmBias are the weights' (modulo 2^64)
  __device__ u64 whole() const { return bits & 0xfffffffffffffull; }
};
__device__ __forceinline__ SmWeight sm_weight(double d, double per32, const double* table) {
  const double t = fma(d, per32, 6755399441055744.0), r = fma(d, per32, -(t - 6755399441055744.0));
  const unsigned n = (unsigned)__double_as_longlong(t);
  const double c = table[n & 31];
  double q = 9.172598566029335e-09;
  q = fma(q, r, 1.6938609067364198e-06);
  q = fma(q, r, 0.00023459619820112603);
  q = fma(q, r, 0.021660849392187844);
  const double e = fma(c * r, q, c);
  const double w = __hiloint2double(__double2hiint(e) + (int)((n & ~31u) << 15), __double2loint(e));
  return {w, (u64)__double_as_longlong(w + 4503599627370496.0)};
}

// What the passes over a row share.
struct SmShared {
  u64 mass[kSmRuns];  // (of the bins: kSmBins)
  unsigned count[kSmBins];
  u64 order[kSmList];  // (key, ~index) of the list's tokens
  double table[32];
  u64 part[2][kSmWaves];
  float top[kSmWaves];
  unsigned low[kSmWaves];
  unsigned n, at, found_bin;
  u64 above;
};

// v + what the lanes before it hold, by DPP: rows of 16 (and, WHOLE, then the rows' ends)
template <bool WHOLE>
__device__ __forceinline__ unsigned sm_scan32(unsigned v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
  if (WHOLE) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // lane 15 of rows 0 and 2 into the next ones
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);  // lane 31 into rows 2 and 3
  }
  return v;
}
// 64 bits in pieces of 25, whose sums stay below 2^31: one instruction a step and piece, and no carries
template <bool WHOLE = true>
__device__ __forceinline__ u64 sm_wave_scan(u64 v) {
  const unsigned m = (1u << 25) - 1;
  const u64 lo = sm_scan32<WHOLE>((unsigned)v & m), mid = sm_scan32<WHOLE>((unsigned)(v >> 25) & m);
  return lo + (mid << 25) + ((u64)sm_scan32<WHOLE>((unsigned)(v >> 50)) << 50);
}
__device__ __forceinline__ u64 sm_lane(u64 v, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, lane);
}
__device__ __forceinline__ u64 sm_last(u64 v) { return sm_lane(v, 63); }
// the lanes' sum, of numbers below 2^52: two pieces whose sums fit 32 bits
__device__ __forceinline__ u64 sm_wave_sum(u64 v) {
  const unsigned lo = sm_scan32<true>((unsigned)v & ((1u << 26) - 1)), hi = sm_scan32<true>((unsigned)(v >> 26));
  return (unsigned)__builtin_amdgcn_readlane((int)lo, 63) + ((u64)(unsigned)__builtin_amdgcn_readlane((int)hi, 63) << 26);
}
// Sums of the threads up to and with this one, and of all; integers, so in any order.  `turn` says which half of `part` is free.
__device__ __forceinline__ u64 sm_scan(u64 v, SmShared& s, int& turn, u64& total) {
  v = sm_wave_scan(v);
  u64* part = s.part[turn];
  turn ^= 1;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((threadIdx.x & 63) == 63) part[w] = v;
  __syncthreads();
  const u64 p = sm_wave_scan<false>(part[threadIdx.x & (kSmWaves - 1)]);  // a row of 16 lanes scans the waves' sums
  total = sm_lane(p, kSmWaves - 1);
  return v + (w ? sm_lane(p, w - 1) : 0);
}
// the same of counts: 32 bits
__device__ __forceinline__ unsigned sm_scan_count(unsigned v, SmShared& s, int& turn, unsigned& total) {
  v = sm_scan32<true>(v);
  u64* part = s.part[turn];
  turn ^= 1;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((threadIdx.x & 63) == 63) part[w] = v;
  __syncthreads();
  const unsigned p = sm_scan32<false>((unsigned)part[threadIdx.x & (kSmWaves - 1)]);
  total = (unsigned)__builtin_amdgcn_readlane((int)p, kSmWaves - 1);
  return v + (w ? (unsigned)__builtin_amdgcn_readlane((int)p, w - 1) : 0);
}
__device__ __forceinline__ u64 sm_sum(u64 v, SmShared& s, int& turn) {
  u64 total;
  sm_scan(v, s, turn, total);
  return total;
}
// One step of a sorting network in a wave: lane t and lane t ^ J take the larger and the smaller of their values.  Nothing goes through
// LDS: quads are permuted, halves of rows mirrored, rows rotated and exchanged.
template <int CTRL>
__device__ __forceinline__ u64 sm_moved(u64 v) {
  return (u64)(unsigned)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, false) << 32 |
         (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, 0xf, 0xf, false);
}
template <int J>
__device__ __forceinline__ u64 sm_step(u64 v, bool larger) {
  u64 o;
  if constexpr (J >= 16) {  // (which of the two is whose does not matter)
    const auto lo = J == 32 ? __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false)
                            : __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
    const auto hi = J == 32 ? __builtin_amdgcn_permlane32_swap((unsigned)(v >> 32), (unsigned)(v >> 32), false, false)
                            : __builtin_amdgcn_permlane16_swap((unsigned)(v >> 32), (unsigned)(v >> 32), false, false);
    v = (u64)hi[0] << 32 | lo[0];
    o = (u64)hi[1] << 32 | lo[1];
  } else if constexpr (J == 8) {
    o = sm_moved<0x128>(v);  // row_ror 8
  } else if constexpr (J == 4) {
    o = sm_moved<0x141>(sm_moved<0x1b>(v));  // xor 3, then row_half_mirror: xor 7
  } else {
    o = sm_moved<J == 2 ? 0x4e : 0xb1>(v);
  }
  return larger == (v > o) ? v : o;
}
// the steps J, J / 2 .. 1 of the part that ends in runs of k
template <int J>
__device__ __forceinline__ u64 sm_steps(u64 v, int t, int k) {
  v = sm_step<J>(v, ((t & J) == 0) == ((t & k) == 0));
  if constexpr (J > 1) v = sm_steps<J / 2>(v, t, k);
  return v;
}
// a wave's 64 values in order, the largest in lane 0 (in lane 63 where t has bit 6 set)
__device__ __forceinline__ u64 sm_wave_sort(u64 v, int t) {
  v = sm_steps<1>(v, t, 2);
  v = sm_steps<2>(v, t, 4);
  v = sm_steps<4>(v, t, 8);
  v = sm_steps<8>(v, t, 16);
  v = sm_steps<16>(v, t, 32);
  return sm_steps<32>(v, t, 64);
}
// Sorts the list's n <= kSmList entries, the largest first; thread t gets the t-th (0 past the end).
__device__ __forceinline__ u64 sm_sort(SmShared& s, int n) {
  const int t = threadIdx.x;
  __syncthreads();
  u64 v = t < n ? s.order[t] : 0;
  int size = 64;  // (n <= kSmList: the threads past it only wait)
  while (size < n) size <<= 1;
  const bool in = (t & ~63) < size;  // (whole waves)
  if (in) v = sm_wave_sort(v, t);
#pragma unroll 1
  for (int k = 128; k <= size; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j >= 64; j >>= 1) {
      __syncthreads();
      if (in) s.order[t] = v;
      __syncthreads();
      const u64 o = in ? s.order[t ^ j] : 0;
      v = (((t & j) == 0) == ((t & k) == 0)) == (v > o) ? v : o;
    }
    if (in) v = sm_steps<32>(v, t, k);
  }
  __syncthreads();
  if (in) s.order[t] = v;
  __syncthreads();
  return t < n ? v : 0;
}

// One workgroup a row, which it keeps in LDS as fp32 (CH > 0: up to 4096 CH logits) or reads again in each pass (CH = 0).
//
// Nothing is sorted but short lists.  Logits fall into bins of 1 / 64 nat below the largest; what lies 32 nats below it weighs
// nothing.  The bin in which the top_k-th logit or the top_p share of the weight lies is found from the bins' counts or sums, and
// only that bin's tokens are listed and put in order.  With top_k up to kSmList all that is left is such a list, and weights are
// computed for it alone; one wave takes the usual short one to its end.  Bins that hold more than a list (equal logits, a high
// temperature) are cut by bisection over the values instead.  Each line runs once, so a pass is a small loop: unrolled whole, most
// of the time went into fetching instructions.  (Bisections over the whole row in place of bins: 467 us for one row, 807 for the 256.)
//
// A row that fits is kept in LDS: 36 us for the 256 rows where reading it again took 60.  Sums are of whole numbers, so atomics and
// scans may come in any order.
template <typename T, int CH>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleParams a) {
  __shared__ SmShared s;
  __shared__ f32x4 xs[CH > 0 ? CH * kSmThreads : 1];  // the row
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), V = a.V;
  const T* row = (const T*)a.logits + b * a.stride;
  float temperature = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const float top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const float p_min = a.min_p_rows ? a.min_p_rows[b] : a.min_p, min_p = p_min > 0.f ? fminf(p_min, 1.f) : 0.f;
  int top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const float u = fminf(fmaxf(a.u[b], 0.f), 1.f);
  if (!(temperature > 0.f) || top_p <= 0.f) top_k = 1;  // the largest alone (a NaN too)
  int turn = 0;

  // quad q of a thread: 4 logits from index (kSmThreads q + tid) 4 - head on, aligned as one; -inf for what is out of the row
  const int head = (int)((uintptr_t)row / sizeof(T) & 3);
  const int quads = CH > 0 ? CH : (V + head + 4 * kSmThreads - 1) / (4 * kSmThreads);
  bool all_or_nothing = false;
  auto load = [&](int q) SM_INLINE {
    const int i0 = (q * kSmThreads + tid) * 4 - head;
    f32x4 v;
    if (i0 >= 0 && i0 + 4 <= V) {
      if constexpr (sizeof(T) == 4) {
        v = *reinterpret_cast<const f32x4*>(row + i0);
      } else {
        const u32x2 r = ldg8(row + i0);
        v = f32x4{lo_bf16(r[0]), hi_bf16(r[0]), lo_bf16(r[1]), hi_bf16(r[1])};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i0 + e >= 0 && i0 + e < V ? (float)row[i0 + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] == v[e] ? v[e] + 0.f : -INFINITY;
    if (CH == 0 && all_or_nothing) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
    }
    return v;
  };
  auto at = [&](int q) SM_INLINE {
    if constexpr (CH > 0)
      return xs[q * kSmThreads + tid];
    else
      return load(q);
  };
  auto index = [&](int q, int e) { return (q * kSmThreads + tid) * 4 - head + e; };
  // f(value, index) of every logit of the thread
  auto each = [&](auto&& f) SM_INLINE {
#pragma unroll 1
    for (int q = 0; q < quads; ++q) {
      const f32x4 v = at(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(v[e], index(q, e));
    }
  };

  auto top_of = [](f32x4 v) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); };
  float own = -INFINITY;
  float quad_top[CH > 0 ? CH : 1];  // the largest of each of the thread's quads
  if constexpr (CH > 0) {
#pragma unroll
    for (int q0 = 0; q0 < CH; q0 += 8) {
      f32x4 v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q0 + q < CH) v[q] = load(q0 + q);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q0 + q < CH) {
          xs[(q0 + q) * kSmThreads + tid] = v[q];
          own = fmaxf(own, quad_top[q0 + q] = top_of(v[q]));
        }
    }
  } else {
    each([&](float v, int) { own = fmaxf(own, v); });
  }
  if (tid < 32) s.table[tid] = kSmTable[tid];
  s.count[tid] = s.count[tid + kSmThreads] = 0;
  if (tid == 0) s.found_bin = kSmBins;
  float big = own;
#pragma unroll
  for (int m = 8; m; m >>= 1) big = fmaxf(big, wave_shfl_xor(big, m));
  big = xor32_max(xor16_max(big));
  if (lane == 0) s.top[wave] = big;
  __syncthreads();
  big = s.top[lane & (kSmWaves - 1)];
#pragma unroll
  for (int m = 8; m; m >>= 1) big = fmaxf(big, wave_shfl_xor(big, m));
  if (big == -INFINITY) {
    if (tid == 0) {
      a.tokens[b] = -1;
      a.logprobs[b] = -INFINITY;
    }
    return;
  }
  if (top_k == 1) {
    unsigned low = 0x7fffffffu;
    if (own == big) each([&](float v, int i) { low = (v == big) & ((unsigned)i < low) ? (unsigned)i : low; });
#pragma unroll
    for (int m = 32; m; m >>= 1) low = min(low, (unsigned)__shfl_xor((int)low, m, 64));
    if (lane == 0) s.low[wave] = low;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kSmWaves; ++i) low = min(low, s.low[i]);
      a.tokens[b] = low;
      a.logprobs[b] = 0.f;
    }
    return;
  }
  if (big == INFINITY) {  // infinities share all the weight: 0 beside -inf
    all_or_nothing = true;
    big = 0.f;
    own = own == INFINITY ? 0.f : -INFINITY;
    if constexpr (CH > 0) {
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        f32x4& x = xs[q * kSmThreads + tid];
        quad_top[q] = quad_top[q] == INFINITY ? 0.f : -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = x[e] == INFINITY ? 0.f : -INFINITY;
      }
    }
  }
  const double t = fmin((double)temperature, 1e300);  // (an infinite one: all weights of finite logits 1)
  const double xmax = (double)big, rate = 1.0 / t, per32 = 46.16624130844683 * rate;  // 32 log2 e
  const double least_d = -33.0 * t;                                                   // weighs nothing
  const double least = (double)min_p * kSmOne;
  const float half_big = 0.5f * big, bins_t = 2.f * fminf((float)kSmPerNat / temperature, 1e30f);
  auto weight = [&](float v) SM_INLINE {
    SmWeight w = sm_weight(fmax((double)v - xmax, least_d), per32, s.table);
    asm volatile("" : "+v"(w.bits));  // not put under the condition of its use: a branch for each logit, each waiting for the table
    return w;
  };
  // a logit's distance from the largest in bins; a bin is its whole part, the last one takes all beyond.  By halves: two logits can be
  // further apart than fp32's largest number.  (A -inf at an infinite temperature is a NaN, which no comparison lets in.)
  auto distance = [&](float v) { return fmaf(v, -0.5f, half_big) * bins_t; };
  auto bin_of = [&](float v) { return (int)fminf(distance(v), (float)(kSmBins - 1)); };

  // what is kept: values of `cut` and more, from index `bound` on only those of `above_cut`, the next value, and more; never a -inf
  float cut = -kSmMost, above_cut = sm_value(sm_key(-kSmMost) + 1);
  int bound = V;
  auto is_kept = [&](float v, int i) SM_INLINE {
    const float least_here = i < bound ? +cut : +above_cut;
    return v >= least_here;
  };
  // a quad with -inf for what is not; `bound` lies in few of them
  auto kept_quad = [&](int q) SM_INLINE {
    f32x4 v = at(q);
    const int i0 = index(q, 0);
    const float least_here = i0 < bound ? +cut : +above_cut;
    if (__ballot((i0 < bound) & (bound < i0 + 4))) {
#pragma unroll
      for (int e = 1; e < 4; ++e) v[e] = is_kept(v[e], i0 + e) ? v[e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] >= least_here ? v[e] : -INFINITY;
    return v;
  };
  auto cut_at_key = [&](unsigned key) {
    cut = sm_value(key);
    above_cut = sm_value(key + 1);
  };
  auto cut_at = [&](u64 last) {  // the last one kept
    cut_at_key((unsigned)(last >> 32));
    bound = (int)~(unsigned)last + 1;
  };
  // g(j, k) of the thread's logits whose bits are set in `bits` (bit j: place j & 3 of quad j / 4), the k-th of all threads'; their number
  auto number = [&](unsigned bits, unsigned most, auto&& g) SM_INLINE {
    unsigned n;
    unsigned k = sm_scan_count(__popc(bits), s, turn, n) - __popc(bits);
    for (; bits && k < most; bits &= bits - 1) g(__ffs(bits) - 1, k++);
    __syncthreads();
    return n;
  };
  auto place = [&](int j) { return ((j >> 2) * kSmThreads + tid) * 4 + (j & 3); };  // of logit j in xs: its index + head
  auto entry = [&](float v, int i) { return (u64)sm_key(v) << 32 | ~(unsigned)i; };
  // lists the tokens that `f` says, of quads whose largest value `any` lets in; their number, which may be more than the list takes.
  // f gets the value, the index and the thread's number for it.
  auto list = [&](auto&& any, auto&& f) SM_INLINE {
    if constexpr (CH > 0) {
      unsigned hot = 0, bits = 0;
#pragma unroll
      for (int q = 0; q < CH; ++q) hot |= (unsigned)any(quad_top[q]) << q;
      for (; hot; hot &= hot - 1) {
        const int q = __ffs(hot) - 1;
        const f32x4 v = at(q);
#pragma unroll
        for (int e = 0; e < 4; ++e) bits |= (unsigned)f(v[e], index(q, e), 4 * q + e) << (4 * q + e);
      }
      return (int)number(bits, kSmList,
                         [&](int j, unsigned k) { s.order[k] = entry(reinterpret_cast<const float*>(xs)[place(j)], place(j) - head); });
    } else {
      if (tid == 0) s.n = 0;
      __syncthreads();
#pragma unroll 1
      for (int q = 0; q < quads; ++q) {
        const f32x4 v = at(q);
        if (any(top_of(v))) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (f(v[e], index(q, e), 0)) {
              const unsigned k = atomicAdd(&s.n, 1u);
              if (k < kSmList) s.order[k] = entry(v[e], index(q, e));
            }
        }
      }
      __syncthreads();
      return (int)s.n;
    }
  };
  // the bound that leaves the first r of the kept tokens equal to `cut`
  auto bound_of = [&](u64 r) SM_INLINE {
    int lo = 0;
#pragma unroll 1
    for (int bit = kSmMaxV; bit; bit >>= 1) {
      if (lo + bit > bound) continue;
      u64 n = 0;
      each([&](float v, int i) { n += (v == cut) & (i < lo + bit); });
      if (sm_sum(n, s, turn) <= r) lo += bit;
    }
    return lo;
  };
  // the bin at which the bins' numbers add up to what `need` makes of their sum, and what lies above it, in s.found_bin (left alone if
  // none) and s.above
  auto find = [&](u64 n0, u64 n1, auto&& need) SM_INLINE {
    u64 all;
    const u64 before = sm_scan(n0 + n1, s, turn, all) - n0 - n1, n = need(all);
    if (before < n && n <= before + n0 + n1) {
      const bool second = before + n0 < n;
      s.found_bin = 2 * tid + second;
      s.above = before + (second ? n0 : 0);
    }
    __syncthreads();
  };
  // the draw: the first sum above `aim` is the token's.  Where it ends up is one thread's `hit`.
  auto aim_of = [&](u64 total) { return min((u64)((double)u * (double)total), total - 1); };
  bool hit = false;
  int token = 0;
  float value = 0.f;
  double log_total = 0.0;
  u64 total = 0;

  int n_list = -1;  // a list of all that is kept, in order: thread t has entry t in `mine`
  bool in_one_wave = false;
  u64 mine = 0;
  if (top_k > 0 && top_k < V) {
    // the bin of the top_k-th of the threads' largest: as many logits at least lie in it and above
    if (top_k <= kSmThreads / 2) {
      const int bin = bin_of(own);
      if (bin < kSmBins - 1) atomicAdd(&s.count[bin], 1u);
      __syncthreads();
      find(s.count[2 * tid], s.count[2 * tid + 1], [&](u64) { return (u64)top_k; });
      if (s.found_bin < kSmBins) {
        const float end = (float)(s.found_bin + 1);
        auto near = [&](float v, int = 0, int = 0) { return distance(v) < end; };
        n_list = list(near, near);
        in_one_wave = n_list <= 64;
        if (n_list > kSmList) n_list = -1;
      }
    }
    if (n_list < 0) {
      __syncthreads();
      s.count[tid] = s.count[tid + kSmThreads] = 0;
      if (tid == 0) s.found_bin = kSmBins;
      __syncthreads();
      each([&](float v, int) {
        const int bin = bin_of(v);
        if (bin < kSmBins - 1) atomicAdd(&s.count[bin], 1u);
      });
      __syncthreads();
      find(s.count[2 * tid], s.count[2 * tid + 1], [&](u64) { return (u64)top_k; });
      const int bin = s.found_bin;
      if (bin < kSmBins) {  // (else fewer than top_k weigh anything)
        const int above = (int)s.above, in = s.count[bin];
        const bool all = above + in <= kSmList;
        const float from = all ? 0.f : (float)bin, end = (float)(bin + 1);
        if (in <= kSmList) {
          const int n = list([&](float v) { return distance(v) < end; },
                             [&](float v, int, int) { return (distance(v) >= from) & (distance(v) < end); });
          if (all) {
            n_list = n;
          } else {
            sm_sort(s, n);
            cut_at(s.order[top_k - above - 1]);
          }
        } else {
          unsigned t = 0;  // the top_k-th key
#pragma unroll 1
          for (unsigned bit = 1u << 31; bit; bit >>= 1) {
            u64 n = 0;
            each([&](float v, int) { n += sm_key(v) >= (t | bit); });
            if (sm_sum(n, s, turn) >= (u64)top_k) t |= bit;
          }
          u64 n = 0;
          each([&](float v, int) { n += sm_key(v) > t; });
          n = sm_sum(n, s, turn);
          cut_at_key(t);
          bound = bound_of(top_k - n);
        }
        if (n_list < 0 && top_k <= kSmList) {
          __syncthreads();
          n_list = list([&](float v) { return v >= cut; }, [&](float v, int i, int) { return is_kept(v, i); });
        }
      }
    }
    if (n_list >= 0 && !in_one_wave) {
      mine = sm_sort(s, n_list);
      n_list = min(n_list, top_k);
    }
  }

  if (in_one_wave) {
    // a lane an entry: in order for top_k and top_p, then by index (~index: the larger is the earlier) for the draw
    if (wave != 0) return;
    mine = sm_wave_sort(lane < n_list ? s.order[lane] : 0, lane);
    const SmWeight w = weight(sm_value((unsigned)(mine >> 32)));
    u64 whole = lane < min(n_list, top_k) ? w.whole() : 0;
    if (top_p < 1.f) {
      const u64 upto = sm_wave_scan(whole), target = (u64)ceil((double)top_p * (double)sm_last(upto));
      whole = lane > 0 && upto - whole >= target ? 0 : whole;
    }
    whole = w.w < least ? 0 : whole;
    total = sm_last(sm_wave_scan(whole));
    log_total = log((double)total / kSmOne);
    const u64 aim = aim_of(total), by_index = sm_wave_sort(mine << 32 | (unsigned)lane, lane);
    const int from = (int)(unsigned)by_index;
    whole = (u64)(unsigned)__shfl((int)(whole >> 32), from, 64) << 32 | (unsigned)__shfl((int)(unsigned)whole, from, 64);
    const u64 upto = sm_wave_scan(whole);
    hit = aim < upto && upto - whole <= aim;
    token = (int)~(unsigned)(by_index >> 32);
    value = sm_value((unsigned)__shfl((int)(mine >> 32), from, 64));
  } else if (n_list >= 0) {
    value = sm_value((unsigned)(mine >> 32));
    token = (int)~(unsigned)mine;
    const SmWeight w = weight(value);
    u64 whole = tid < n_list ? w.whole() : 0;
    if (top_p < 1.f) {
      const u64 upto = sm_scan(whole, s, turn, total);
      const u64 target = (u64)ceil((double)top_p * (double)total);
      if (tid > 0 && upto - whole >= target) whole = 0;
    }
    if (w.w < least) whole = 0;
    // the vocabulary in kSmThreads runs, of which the list's tokens fill a few
    int shift = 0;
    while ((V - 1) >> shift >= kSmThreads) ++shift;
    __syncthreads();
    s.mass[tid] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    if (whole) atomicAdd(&s.mass[token >> shift], whole);
    __syncthreads();
    const u64 run = s.mass[tid], upto = sm_scan(run, s, turn, total);
    const u64 aim = aim_of(total);
    if (upto > aim && upto - run <= aim) {
      s.at = tid;
      s.above = upto - run;
    }
    __syncthreads();
    const bool in = whole && (unsigned)(token >> shift) == s.at;
    if (in) {
      const unsigned k = atomicAdd(&s.n, 1u);
      s.order[k] = (u64)token;
      s.mass[k] = whole;
    }
    __syncthreads();
    if (in) {
      u64 sum = s.above;
      for (unsigned k = 0; k < s.n; ++k) sum += (int)s.order[k] < token ? s.mass[k] : 0;
      hit = sum <= aim && aim < sum + whole;
    }
  } else {
    // The whole row: its weights by bin for top_p, and again (there are no registers for 32 of them a thread) for the draw.
    unsigned above_bits = 0, in_bits = 0;  // (CH > 0) the thread's logits, a bit each: what lies above top_p's bin, and in it
    if (top_p < 1.f) {
      __syncthreads();
      s.mass[tid] = s.mass[tid + kSmThreads] = 0;
      if (tid == 0) s.found_bin = kSmBins;
      __syncthreads();
#pragma unroll 1
      for (int q = 0; q < quads; ++q) {
        const f32x4 v = kept_quad(q);
        u64 whole[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) whole[e] = weight(v[e]).whole();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = distance(v[e]);
          if (d < (float)(kSmBins - 1)) atomicAdd(&s.mass[(int)d], whole[e]);
        }
      }
      __syncthreads();
      u64 target;
      find(s.mass[2 * tid], s.mass[2 * tid + 1], [&](u64 sum) { return target = max((u64)ceil((double)top_p * (double)sum), (u64)1); });
      const float from = (float)s.found_bin, end = (float)(s.found_bin + 1);
      const u64 above = s.above;
      const int n = list([&](float v) { return distance(v) < end; },
                         [&](float v, int i, int j) {
                           const float d = distance(v);
                           const bool k = (d < end) & is_kept(v, i), in = k & (d >= from);
                           if (CH > 0) {
                             above_bits |= (unsigned)(k & !in) << j;
                             in_bits |= (unsigned)in << j;
                           }
                           return in;
                         });
      if (n <= 64) {
        if (wave == 0) {
          mine = sm_wave_sort(lane < n ? s.order[lane] : 0, lane);
          const SmWeight x = weight(sm_value((unsigned)(mine >> 32)));
          const u64 whole = lane < n ? x.whole() : 0, upto = above + sm_wave_scan(whole);
          // the last with less than the target before it: with its own weight it is reached
          if (upto - whole < target && upto >= target) s.order[kSmList - 1] = mine;
        }
        __syncthreads();
        cut_at(s.order[kSmList - 1]);
      } else if (n <= kSmList) {
        mine = sm_sort(s, n);
        const u64 w = weight(sm_value((unsigned)(mine >> 32))).whole(), mw = tid < n ? w : 0;
        const u64 ahead = sm_scan(mw, s, turn, total) - mw + above;
        const u64 last = sm_sum(tid < n && ahead < target, s, turn);
        cut_at(s.order[last - 1]);
      } else {
        auto mass_above = [&](unsigned t) SM_INLINE {
          u64 m = 0;
          each([&](float v, int i) {
            const u64 w = weight(v).whole();
            m += (sm_key(v) > t) & is_kept(v, i) ? w : 0;
          });
          return sm_sum(m, s, turn);
        };
        unsigned t = 0;  // the smallest key with less than the target above it
#pragma unroll 1
        for (unsigned bit = 1u << 31; bit; bit >>= 1)
          if (mass_above(t + bit - 1) >= target) t += bit;
        const u64 ahead = mass_above(t), w = weight(sm_value(t)).whole();
        if (sm_value(t) > cut) {
          cut_at_key(t);
          bound = V;
        }
        bound = bound_of(w ? (target - ahead + w - 1) / w : V);
      }
    }

    // The draw: runs of 256 indices, a wave's quad each.  Where the row is kept in LDS and few of it are left, their indices are listed
    // (where the counts and the list were) and only they are weighed again.
    // the weights of a quad and kSmBias each, and their sum
    u64 w[4];
    auto quad_weights = [&](int q) SM_INLINE {
      const f32x4 v = kept_quad(q);
      SmWeight x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = (x[e] = weight(v[e])).bits;
      if (least > 0) {
        asm volatile("");  // (a branch: most rows have none)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = x[e].w < least ? kSmBias : w[e];
      }
      return w[0] + w[1] + w[2] + w[3] - 4 * kSmBias;
    };
    __syncthreads();
    for (int i = tid; i < kSmRuns; i += kSmThreads) s.mass[i] = 0;
    __syncthreads();
    bool few = false;
    if constexpr (CH > 0) {
      unsigned short* at_of = reinterpret_cast<unsigned short*>(s.count);  // (places in xs)
      constexpr unsigned kFew = (sizeof(s.count) + sizeof(s.order)) / 2;
      static_assert(offsetof(SmShared, order) == offsetof(SmShared, count) + sizeof(s.count) && CH <= 8, "");
      unsigned n_kept = kFew + 1;
      if (top_p < 1.f) {
        unsigned kept = above_bits;
        for (unsigned m = in_bits; m; m &= m - 1) {
          const int i = place(__ffs(m) - 1);
          if (is_kept(reinterpret_cast<const float*>(xs)[i], i - head)) kept |= m & -m;
        }
        n_kept = number(kept, kFew, [&](int j, unsigned k) { at_of[k] = (unsigned short)place(j); });
      }
      few = n_kept <= kFew;
      if (few) {
#pragma unroll 1
        for (unsigned k = tid; k < n_kept; k += kSmThreads) {
          const unsigned i = at_of[k];
          const SmWeight w = weight(reinterpret_cast<const float*>(xs)[i]);
          if (!(w.w < least) && w.whole()) atomicAdd(&s.mass[i / 256], w.whole());
        }
      }
    }
    if (!few) {
#pragma unroll 1
      for (int q = 0; q < quads; ++q) {
        const u64 m = sm_wave_sum(quad_weights(q));
        if (lane == 0) s.mass[q * kSmWaves + wave] = m;
      }
    }
    __syncthreads();
    constexpr int PER = (kSmRuns + kSmThreads - 1) / kSmThreads;
    u64 runs[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += runs[k] = PER * tid + k < kSmRuns ? s.mass[PER * tid + k] : 0;
    u64 ahead = sm_scan(sum, s, turn, total) - sum;
    const u64 aim = aim_of(total);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (ahead <= aim && aim < ahead + runs[k]) {
        s.at = PER * tid + k;
        s.above = ahead;
      }
      ahead += runs[k];
    }
    __syncthreads();
    if ((int)s.at % kSmWaves != wave) return;
    const int q = s.at / kSmWaves;
    const f32x4 v = at(q);
    const u64 m = quad_weights(q);
    ahead = s.above + sm_wave_scan(m) - m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const u64 we = w[e] - kSmBias;
      if (ahead <= aim && aim < ahead + we) {
        hit = true;
        token = index(q, e);
        value = v[e];
      }
      ahead += we;
    }
  }
  if (hit) {
    a.tokens[b] = token;
    a.logprobs[b] = (float)(((double)value - xmax) * rate - (in_one_wave ? log_total : log((double)total / kSmOne)));
  }
}

template <typename T>
void sample_launch(const SampleParams& p, int64_t B, hipStream_t st) {
  const dim3 grid((unsigned)B);
  // A row may begin anywhere in a quad, unless all begin at its start.  8 quads a thread are what LDS takes; a short row is not worth
  // passes over as many, mostly empty ones; a longer one is read again in each pass.
  const bool aligned = (uintptr_t)p.logits % (4 * sizeof(T)) == 0 && (B == 1 || p.stride % 4 == 0);
  const int n = p.V + (aligned ? 0 : 3);
  if (n <= 8 * kSmThreads)
    sample_kernel<T, 2><<<grid, kSmThreads, 0, st>>>(p);
  else if (n <= 32 * kSmThreads)
    sample_kernel<T, 8><<<grid, kSmThreads, 0, st>>>(p);
  else
    sample_kernel<T, 0><<<grid, kSmThreads, 0, st>>>(p);
}

}  // namespace mla

using namespace mla;

extern "C" int mla_sample(const mla_sample_args* a, void* stream) {
  const char* op = "mla_sample";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_CHECK(a->B >= 0 && a->B < (1ll << 32) / kSmThreads && a->V >= 1 && a->V <= kSmMaxV, MLA_ERR_INVALID_ARG,
            "%s: B %lld or V %lld is out of range (fewer than 2^22 rows, 1 .. 2^19 logits)", op, (long long)a->B, (long long)a->V);
  MLA_CHECK(a->dtype == MLA_DTYPE_BF16 || a->dtype == MLA_DTYPE_F32, MLA_ERR_UNSUPPORTED, "%s: logits must be bf16 or fp32", op);
  if (a->B == 0) return MLA_OK;
  MLA_CHECK(a->logits && a->u && a->tokens && a->logprobs, MLA_ERR_INVALID_ARG, "%s: null pointer", op);
  const int es = a->dtype == MLA_DTYPE_BF16 ? 2 : 4;
  MLA_CHECK((uintptr_t)a->logits % es == 0 && ((uintptr_t)a->tokens & 7) == 0, MLA_ERR_INVALID_ARG, "%s: a pointer is not aligned to its type",
            op);
  const void* words[] = {a->u, a->temperature_rows, a->top_k_rows, a->top_p_rows, a->min_p_rows, a->logprobs};
  for (const void* q : words) MLA_CHECK(((uintptr_t)q & 3) == 0, MLA_ERR_INVALID_ARG, "%s: a pointer is not aligned to its type", op);
  MLA_CHECK(a->B == 1 || a->stride >= 0, MLA_ERR_INVALID_ARG, "%s: stride is negative", op);
  MLA_CHECK((a->temperature_rows || !std::isnan(a->temperature)) && (a->top_p_rows || !std::isnan(a->top_p)) &&
                (a->min_p_rows || !std::isnan(a->min_p)),
            MLA_ERR_INVALID_ARG, "%s: a setting is NaN", op);
  const SampleParams p = {a->logits, a->u,      a->temperature_rows, a->top_p_rows, a->min_p_rows, a->top_k_rows, a->tokens, a->logprobs,
                          a->stride, (int)a->V, a->temperature,      a->top_p,      a->min_p,      a->top_k};
  if (a->dtype == MLA_DTYPE_BF16)
    sample_launch<bf16>(p, a->B, (hipStream_t)stream);
  else
    sample_launch<float>(p, a->B, (hipStream_t)stream);
  return launch_status(op);
}
