// Drawing one token for each row of logits: temperature, top-k, top-p, min-p and the draw from a given number (gfx950).
#include <cmath>

#include "mla_common.h"

namespace mla {

constexpr int kSmThreads = 1024;
constexpr int kSmMaxV = 1 << 19;  // 2^19 weights of up to 2^44 add up below 2^63
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmBins = 2048, kSmPerNat = 64;
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
struct SmWeight {
  double w;  // in units of 2^-44, before the rounding
  u64 whole;
};
__device__ __forceinline__ SmWeight sm_weight(double d, double per32, const double* table) {
  const double t = fma(d, per32, 6755399441055744.0), r = fma(d, per32, -(t - 6755399441055744.0));
  const int n = (int)(unsigned)__double_as_longlong(t);
  const double c = table[n & 31];
  double q = 9.172598566029335e-09;
  q = fma(q, r, 1.6938609067364198e-06);
  q = fma(q, r, 0.00023459619820112603);
  q = fma(q, r, 0.021660849392187844);
  const double e = fma(c * r, q, c);
  const double w = __longlong_as_double(__double_as_longlong(e) + ((long long)(n >> 5) << 52));
  return {w, (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull};
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
__device__ __forceinline__ u64 sm_sum(u64 v, SmShared& s, int& turn) {
  u64 total;
  sm_scan(v, s, turn, total);
  return total;
}
// Sorts the list's n <= kSmList entries, the largest first; thread t gets the t-th (0 past the end).
__device__ __forceinline__ u64 sm_sort(SmShared& s, int n) {
  const int t = threadIdx.x;
  __syncthreads();
  u64 v = t < n ? s.order[t] : 0;
  int size = 64;  // (n <= kSmList: the threads past it only wait)
  while (size < n) size <<= 1;
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j; j >>= 1) {
      u64 o;
      if (j < 64) {
        if ((t & ~63) >= size) continue;  // (whole waves)
        o = __shfl_xor(v, j, 64);
      } else {
        __syncthreads();
        if (t < kSmList) s.order[t] = v;
        __syncthreads();
        o = s.order[(t ^ j) & (kSmList - 1)];
      }
      const bool larger = ((t & j) == 0) == ((t & k) == 0);  // this place takes the larger of the two
      v = larger == (v > o) ? v : o;
    }
  }
  __syncthreads();
  if (t < kSmList) s.order[t] = v;
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
// of the time went into fetching instructions.
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
  temperature = fminf(temperature, kSmMost);
  int turn = 0;

  // quad q of a thread: 4 logits from index (kSmThreads q + tid) 4 - head on, aligned as one; -inf for what is out of the row
  const int head = (int)((uintptr_t)row / sizeof(T) & 3);
  const int quads = CH > 0 ? CH : (V + head + 4 * kSmThreads - 1) / (4 * kSmThreads);
  bool all_or_nothing = false;
  auto load = [&](int q) {
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
  auto at = [&](int q) {
    if constexpr (CH > 0)
      return xs[q * kSmThreads + tid];
    else
      return load(q);
  };
  auto index = [&](int q, int e) { return (q * kSmThreads + tid) * 4 - head + e; };
  // f(value, index) of every logit of the thread
  auto each = [&](auto&& f) {
#pragma unroll 1
    for (int q = 0; q < quads; ++q) {
      const f32x4 v = at(q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(v[e], index(q, e));
    }
  };

  float own = -INFINITY;
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
          own = fmaxf(own, fmaxf(fmaxf(v[q][0], v[q][1]), fmaxf(v[q][2], v[q][3])));
        }
    }
  } else {
    each([&](float v, int) { own = fmaxf(own, v); });
  }
  if (tid < 32) s.table[tid] = kSmTable[tid];
  s.count[tid] = s.count[tid + kSmThreads] = 0;
  if (tid == 0) s.n = 0, s.found_bin = kSmBins;
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
#pragma unroll 1
      for (int q = 0; q < CH; ++q) {
        f32x4& x = xs[q * kSmThreads + tid];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = x[e] == INFINITY ? 0.f : -INFINITY;
      }
    }
  }
  const double xmax = (double)big, per32 = 46.16624130844683 / (double)temperature;  // 32 log2 e
  const double least_d = -33.0 * (double)temperature;                                // weighs nothing
  const double least = (double)min_p * kSmOne;
  const float bins_t = fminf((float)kSmPerNat / temperature, 1e30f);
  auto weight = [&](float v) {
    SmWeight w = sm_weight(fmax((double)v - xmax, least_d), per32, s.table);
    asm volatile("" : "+v"(w.whole));  // not put under the condition of its use: a branch for each logit, each waiting for the table
    return w;
  };
  // a logit's distance from the largest in bins; a bin is its whole part, the last one takes all beyond
  auto distance = [&](float v) { return (big - v) * bins_t; };
  auto bin_of = [&](float v) { return (int)fminf(distance(v), (float)(kSmBins - 1)); };

  // what is kept: values above `cut`, and of those equal to it the ones below index `bound`; never a -inf
  float cut = -kSmMost;
  int bound = V;
  auto is_kept = [&](float v, int i) { return (v > cut) | ((v == cut) & (i < bound)); };
  auto cut_at = [&](u64 last) {  // the last one kept
    cut = sm_value((unsigned)(last >> 32));
    bound = (int)~(unsigned)last + 1;
  };
  // lists the tokens that `f` says (s.n is 0 before); their number, which may be more than the list takes
  auto list = [&](auto&& f) {
    each([&](float v, int i) {
      if (f(v, i)) {
        const unsigned k = atomicAdd(&s.n, 1u);
        if (k < kSmList) s.order[k] = (u64)sm_key(v) << 32 | ~(unsigned)i;
      }
    });
    __syncthreads();
    return (int)s.n;
  };
  // the bound that leaves the first r of the kept tokens equal to `cut`
  auto bound_of = [&](u64 r) {
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
  // the bin at which the bins' numbers add up to `need`, and what lies above it, in s.found_bin (left alone if none) and s.above
  auto find = [&](u64 n0, u64 n1, u64 need) {
    u64 total;
    const u64 before = sm_scan(n0 + n1, s, turn, total) - n0 - n1;
    if (before < need && need <= before + n0 + n1) {
      const bool second = before + n0 < need;
      s.found_bin = 2 * tid + second;
      s.above = before + (second ? n0 : 0);
    }
    __syncthreads();
  };
  // One wave and a short list: its entries, two a lane, their weights, and of each its place and the weight before it, by a pass over
  // the others.
  u64 o[2], ow[2], before[2];
  double owd[2];
  int rank[2];
  auto ranks = [&](int n) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = lane + 64 * k;
      o[k] = t < n ? s.order[t] : 0;
      const SmWeight x = weight(sm_value((unsigned)(o[k] >> 32)));
      ow[k] = t < n ? x.whole : 0;
      owd[k] = x.w;
      s.mass[t] = ow[k];
      rank[k] = 0;
      before[k] = 0;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const u64 oj = s.order[j], wj = s.mass[j];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k == 1 && n <= 64) continue;
        rank[k] += oj > o[k];
        before[k] += oj > o[k] ? wj : 0;
      }
    }
  };

  // the draw: the first sum above `aim` is the token's.  Where it ends up is one thread's `hit`.
  auto aim_of = [&](u64 total) { return min((u64)((double)u * (double)total), total - 1); };
  bool hit = false;
  int token = 0;
  float value = 0.f;
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
      find(s.count[2 * tid], s.count[2 * tid + 1], top_k);
      if (s.found_bin < kSmBins) {
        const float end = (float)(s.found_bin + 1);
        n_list = list([&](float v, int) { return distance(v) < end; });
        in_one_wave = n_list <= 128;
        if (n_list > kSmList) n_list = -1;
      }
    }
    if (n_list < 0) {
      __syncthreads();
      s.count[tid] = s.count[tid + kSmThreads] = 0;
      if (tid == 0) s.n = 0, s.found_bin = kSmBins;
      __syncthreads();
      each([&](float v, int) {
        const int bin = bin_of(v);
        if (bin < kSmBins - 1) atomicAdd(&s.count[bin], 1u);
      });
      __syncthreads();
      find(s.count[2 * tid], s.count[2 * tid + 1], top_k);
      const int bin = s.found_bin;
      if (bin < kSmBins) {  // (else fewer than top_k weigh anything)
        const int above = (int)s.above, in = s.count[bin];
        const bool all = above + in <= kSmList;
        const float from = all ? 0.f : (float)bin, end = (float)(bin + 1);
        if (in <= kSmList) {
          const int n = list([&](float v, int) { return (distance(v) >= from) & (distance(v) < end); });
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
          cut = sm_value(t);
          bound = bound_of(top_k - n);
        }
        if (n_list < 0 && top_k <= kSmList) {
          __syncthreads();
          if (tid == 0) s.n = 0;
          __syncthreads();
          n_list = list([&](float v, int i) { return is_kept(v, i); });
        }
      }
    }
    if (n_list >= 0 && !in_one_wave) {
      mine = sm_sort(s, n_list);
      n_list = min(n_list, top_k);
    }
  }

  if (in_one_wave) {
    if (wave != 0) return;
    ranks(n_list);
#pragma unroll
    for (int k = 0; k < 2; ++k) ow[k] = rank[k] >= top_k ? 0 : ow[k];
    if (top_p < 1.f) {
      const u64 target = (u64)ceil((double)top_p * (double)sm_last(sm_wave_scan(ow[0] + ow[1])));
#pragma unroll
      for (int k = 0; k < 2; ++k) ow[k] = rank[k] > 0 && before[k] >= target ? 0 : ow[k];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      ow[k] = owd[k] < least ? 0 : ow[k];
      s.mass[lane + 64 * k] = ow[k];
      before[k] = 0;
    }
    total = sm_last(sm_wave_scan(ow[0] + ow[1]));
    const u64 aim = aim_of(total);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 4
    for (int j = 0; j < n_list; ++j) {
      const unsigned ij = (unsigned)s.order[j];
      const u64 wj = s.mass[j];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (k == 0 || n_list > 64) before[k] += ij > (unsigned)o[k] ? wj : 0;  // (~index: the larger is the earlier)
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (before[k] <= aim && aim < before[k] + ow[k]) {
        hit = true;
        token = (int)~(unsigned)o[k];
        value = sm_value((unsigned)(o[k] >> 32));
      }
  } else if (n_list >= 0) {
    value = sm_value((unsigned)(mine >> 32));
    token = (int)~(unsigned)mine;
    SmWeight w = weight(value);
    if (tid >= n_list) w = {0.0, 0};
    if (top_p < 1.f) {
      const u64 upto = sm_scan(w.whole, s, turn, total);
      const u64 target = (u64)ceil((double)top_p * (double)total);
      if (tid > 0 && upto - w.whole >= target) w.whole = 0;
    }
    if (w.w < least) w.whole = 0;
    // the vocabulary in kSmThreads runs, of which the list's tokens fill a few
    int shift = 0;
    while ((V - 1) >> shift >= kSmThreads) ++shift;
    __syncthreads();
    s.mass[tid] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    if (w.whole) atomicAdd(&s.mass[token >> shift], w.whole);
    __syncthreads();
    const u64 run = s.mass[tid], upto = sm_scan(run, s, turn, total);
    const u64 aim = aim_of(total);
    if (upto > aim && upto - run <= aim) {
      s.at = tid;
      s.above = upto - run;
    }
    __syncthreads();
    const bool in = w.whole && (unsigned)(token >> shift) == s.at;
    if (in) {
      const unsigned k = atomicAdd(&s.n, 1u);
      s.order[k] = (u64)token;
      s.mass[k] = w.whole;
    }
    __syncthreads();
    if (in) {
      u64 sum = s.above;
      for (unsigned k = 0; k < s.n; ++k) sum += (int)s.order[k] < token ? s.mass[k] : 0;
      hit = sum <= aim && aim < sum + w.whole;
    }
  } else {
    // The whole row: its weights by bin for top_p, and again (there are no registers for 32 of them a thread) for the draw.
    if (top_p < 1.f) {
      __syncthreads();
      s.mass[tid] = s.mass[tid + kSmThreads] = 0;
      if (tid == 0) s.n = 0, s.found_bin = kSmBins;
      u64 own_sum = 0;
      __syncthreads();
      each([&](float v, int i) {
        u64 w = weight(v).whole;
        w = is_kept(v, i) ? w : 0;
        own_sum += w;
        if (w) atomicAdd(&s.mass[bin_of(v)], w);
      });
      const u64 sum = sm_sum(own_sum, s, turn);
      const u64 target = max((u64)ceil((double)top_p * (double)sum), (u64)1);
      find(s.mass[2 * tid], s.mass[2 * tid + 1], target);
      const float from = (float)s.found_bin, end = (float)(s.found_bin + 1);
      const u64 above = s.above;
      const int n = list([&](float v, int i) { return (distance(v) >= from) & (distance(v) < end) & is_kept(v, i); });
      if (n <= 128) {
        if (wave == 0) {
          ranks(n);
          // the last with less than the target before it: with its own weight it is reached
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (before[k] + above < target && before[k] + above + ow[k] >= target) s.order[kSmList - 1] = o[k];
        }
        __syncthreads();
        cut_at(s.order[kSmList - 1]);
      } else if (n <= kSmList) {
        mine = sm_sort(s, n);
        const u64 w = weight(sm_value((unsigned)(mine >> 32))).whole, mw = tid < n ? w : 0;
        const u64 ahead = sm_scan(mw, s, turn, total) - mw + above;
        const u64 last = sm_sum(tid < n && ahead < target, s, turn);
        cut_at(s.order[last - 1]);
      } else {
        auto mass_above = [&](unsigned t) {
          u64 m = 0;
          each([&](float v, int i) {
            const u64 w = weight(v).whole;
            m += (sm_key(v) > t) & is_kept(v, i) ? w : 0;
          });
          return sm_sum(m, s, turn);
        };
        unsigned t = 0;  // the smallest key with less than the target above it
#pragma unroll 1
        for (unsigned bit = 1u << 31; bit; bit >>= 1)
          if (mass_above(t + bit - 1) >= target) t += bit;
        const u64 ahead = mass_above(t), w = weight(sm_value(t)).whole;
        if (sm_value(t) > cut) {
          cut = sm_value(t);
          bound = V;
        }
        bound = bound_of(w ? (target - ahead + w - 1) / w : V);
      }
    }

    // the draw: runs of 256 indices, a wave's quad each
    auto final_weight = [&](float v, int i) -> u64 {
      const SmWeight w = weight(v);
      return is_kept(v, i) & !(w.w < least) ? w.whole : 0;
    };
    __syncthreads();
    for (int i = tid; i < kSmRuns; i += kSmThreads) s.mass[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int q = 0; q < quads; ++q) {
      const f32x4 v = at(q);
      u64 m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) m += final_weight(v[e], index(q, e));
      m = sm_last(sm_wave_scan(m));
      if (lane == 0) s.mass[q * kSmWaves + wave] = m;
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
    u64 w[4], m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) m += w[e] = final_weight(v[e], index(q, e));
    ahead = s.above + sm_wave_scan(m) - m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (ahead <= aim && aim < ahead + w[e]) {
        hit = true;
        token = index(q, e);
        value = v[e];
      }
      ahead += w[e];
    }
  }
  if (hit) {
    a.tokens[b] = token;
    a.logprobs[b] = (float)(((double)value - xmax) / (double)temperature - log((double)total / kSmOne));
  }
}

template <typename T>
void sample_launch(const SampleParams& p, int64_t B, hipStream_t st) {
  const dim3 grid((unsigned)B);
  // a row may begin anywhere in a quad, unless all begin at its start
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
  MLA_CHECK(a->B >= 0 && a->B < (1ll << 31) && a->V >= 1 && a->V <= kSmMaxV, MLA_ERR_INVALID_ARG,
            "%s: B %lld or V %lld is out of range (1 .. 2^19 logits)", op, (long long)a->B, (long long)a->V);
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
