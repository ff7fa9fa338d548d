// Drawing one token for each row of logits: temperature, top-k, top-p, min-p and the draw from a given number (gfx950).
#include <cmath>

#include "rope_append.h"

namespace mla {

constexpr int kSmThreads = 1024;
constexpr int kSmMaxV = 1 << 19;  // 2^19 weights of up to 2^44 add up below 2^63
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmBins = 2 * kSmThreads, kSmPerNat = 64;
constexpr int kSmList = kSmThreads;
constexpr double kSmOne = 17592186044416.0;  // 2^44: the largest weight
constexpr unsigned long long kSmWhole = 1ull << 44;

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

// 2^y for y <= 0 in whole steps of 2^-44; 0 below 2^-46 (and for a NaN).  2^f of |f| <= 1/2 by interpolation at the nine Chebyshev nodes:
// within 1.1e-12 of it, fp64 throughout (a token whose number falls that near a border could come out as its neighbour).
struct SmWeight {
  double w;  // before the rounding
  u64 whole;
};
__device__ __forceinline__ SmWeight sm_weight(double y) {
  const double n = rint(y), f = y - n;
  double e = 1.3255224878668817e-06;
  e = fma(e, f, 1.5310079402249296e-05);
  e = fma(e, f, 0.00015403455852453838);
  e = fma(e, f, 0.0013333450568000645);
  e = fma(e, f, 0.009618129159402558);
  e = fma(e, f, 0.05550410941205933);
  e = fma(e, f, 0.2402265069581299);
  e = fma(e, f, 0.6931471805459335);
  e = fma(e, f, 1.0);
  if (!(y > -46.0)) return {0.0, 0};
  e = ldexp(e, (int)n);
  // e 2^44 + 2^52 has the rounded number in its mantissa
  const double s = e * kSmOne + 4503599627370496.0;
  return {e, (u64)__double_as_longlong(s) & 0xfffffffffffffull};
}

// What the passes over a row share.
struct SmShared {
  u64 mass[kSmBins];  // also the runs of the draw
  unsigned count[kSmBins];
  u64 order[kSmList];   // (key, ~index) of the list's tokens
  u64 part[kSmWaves];
  unsigned top[kSmWaves], low[kSmWaves];
  unsigned n, at, found_bin;
  u64 above;
};

__device__ __forceinline__ u64 sm_shfl_up(u64 v, int m) { return __shfl_up(v, m, 64); }
// sums of the threads up to and with this one, and of all; integers, so in any order
__device__ __forceinline__ u64 sm_scan(u64 v, u64* part, u64& total) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const u64 o = sm_shfl_up(v, m);
    v += lane >= m ? o : 0;
  }
  __syncthreads();  // part is free
  if (lane == 63) part[threadIdx.x >> 6] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < kSmWaves; ++i) {
    v += i < (int)(threadIdx.x >> 6) ? part[i] : 0;
    total += part[i];
  }
  return v;
}
__device__ __forceinline__ u64 sm_sum(u64 v, u64* part) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int i = 0; i < kSmWaves; ++i) s += part[i];
  return s;
}
// Sorts the list's n <= kSmList entries, the largest first; thread t gets the t-th (0 past the end).
__device__ __forceinline__ u64 sm_sort(SmShared& s, int n) {
  const int t = threadIdx.x;
  __syncthreads();
  u64 v = t < n ? s.order[t] : 0;
  int size = 64;
  while (size < n) size <<= 1;
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j; j >>= 1) {
      u64 o;
      if (j < 64) {
        if ((t & ~63) >= size) continue;  // (whole waves)
        o = __shfl_xor(v, j, 64);
      } else {
        __syncthreads();
        s.order[t] = v;
        __syncthreads();
        o = s.order[t ^ j];
      }
      const bool larger = ((t & j) == 0) == ((t & k) == 0);  // this place takes the larger of the two
      v = larger == (v > o) ? v : o;
    }
  }
  __syncthreads();
  s.order[t] = v;
  __syncthreads();
  return t < n ? v : 0;
}

// One workgroup a row, which its threads keep in registers (CH > 0: 8 CH logits each) or read again in each pass (CH = 0).
//
// Nothing is sorted but short lists.  Logits fall into bins of 1 / 64 nat below the largest; what lies 32 nats below it weighs
// nothing.  The bin in which the top_k-th logit or the top_p share of the weight lies is found from the bins' counts or sums, and
// only that bin's tokens are listed and sorted.  With top_k up to 1024 all that is left is such a list, and weights are computed for
// it alone.  Bins that hold more than a list (equal logits, a high temperature) are cut by bisection over the values instead.
template <typename T, int CH>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleParams a) {
  __shared__ SmShared s;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, V = a.V;
  const T* row = (const T*)a.logits + b * a.stride;
  const float temperature = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const float top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const float min_p = fminf(a.min_p_rows ? a.min_p_rows[b] : a.min_p, 1.f);
  int top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  if (!(temperature > 0.f) || top_p <= 0.f) top_k = 1;  // the largest alone

  // chunk j of a thread: 8 logits from index (1024 j + tid) 8 - head on, 16-byte aligned
  const int head = (int)(((uintptr_t)row & 15) / sizeof(T));
  const int chunks = (V + head + 8 * kSmThreads - 1) / (8 * kSmThreads);
  auto load = [&](int j, float (&v)[8]) {
    const int i0 = (j * kSmThreads + tid) * 8 - head;
    if (i0 >= 0 && i0 + 8 <= V) {
      RopeIO<T>::load8(row + i0, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i0 + e >= 0 && i0 + e < V ? (float)row[i0 + e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] == v[e] ? v[e] + 0.f : -INFINITY;
  };
  constexpr int KEPT = CH > 0 ? CH : 1;
  float kept[KEPT][8];
  // f(value, index) of every logit of the thread (index -1 or V and more: none, its value -inf)
  auto each_read = [&](auto&& f) {
    for (int j = 0; j < chunks; ++j) {
      float v[8];
      load(j, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) f(v[e], (j * kSmThreads + tid) * 8 - head + e);
    }
  };
  auto each = [&](auto&& f) {
    if constexpr (CH > 0) {
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        // one logit at a time, and nothing kept of it between the passes: the registers go to the logits
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          asm volatile("" : "+v"(kept[j][e]));
          f(kept[j][e], (j * kSmThreads + tid) * 8 - head + e);
          if (e & 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      each_read(f);
    }
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int j = 0; j < CH; ++j) load(j, kept[j]);
  }
  float big = -INFINITY;
  each([&](float v, int) { big = fmaxf(big, v); });
#pragma unroll
  for (int m = 32; m; m >>= 1) big = fmaxf(big, wave_shfl_xor(big, m));
  if (lane == 0) s.top[tid >> 6] = __float_as_uint(big);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSmWaves; ++i) big = fmaxf(big, __uint_as_float(s.top[i]));
  if (big == -INFINITY) {
    if (tid == 0) {
      a.tokens[b] = -1;
      a.logprobs[b] = -INFINITY;
    }
    return;
  }
  if (top_k == 1) {
    unsigned low = 0x7fffffffu;
    each([&](float v, int i) { low = v == big && (unsigned)i < low ? (unsigned)i : low; });
#pragma unroll
    for (int m = 32; m; m >>= 1) low = min(low, (unsigned)__shfl_xor((int)low, m, 64));
    if (lane == 0) s.low[tid >> 6] = low;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kSmWaves; ++i) low = min(low, s.low[i]);
      a.tokens[b] = low;
      a.logprobs[b] = 0.f;
    }
    return;
  }
  const double xmax = (double)big, per_t = 1.4426950408889634 / (double)temperature;
  const float bins_t = fminf((float)kSmPerNat / temperature, 1e30f);
  auto weight = [&](float v) -> SmWeight {
    if (v == big) return {1.0, kSmWhole};
    return sm_weight(v == -INFINITY ? -INFINITY : ((double)v - xmax) * per_t);
  };
  auto bin_of = [&](float v) { return v == big ? 0 : (int)fminf((big - v) * bins_t, (float)(kSmBins - 1)); };

  // what is kept: values above `cut`, and of those equal to it the ones below index `bound` (a -inf weighs nothing in any case)
  float cut = -INFINITY;
  int bound = V;
  auto is_kept = [&](float v, int i) { return v > cut || (v == cut && i < bound); };
  auto cut_at = [&](u64 last) {  // the last one kept
    cut = sm_value((unsigned)(last >> 32));
    bound = (int)~(unsigned)last + 1;
  };
  // lists the tokens that `f` says; their number, which may be more than the list takes
  auto list = [&](auto&& f) {
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    each([&](float v, int i) {
      if (f(v, i)) {
        const unsigned at = atomicAdd(&s.n, 1u);
        if (at < kSmList) s.order[at] = (u64)sm_key(v) << 32 | ~(unsigned)i;
      }
    });
    __syncthreads();
    return (int)s.n;
  };
  // the bound that leaves the first r of the kept keys equal to `cut`
  auto bound_of = [&](u64 r) {
    int lo = 0;
    for (int bit = kSmMaxV; bit; bit >>= 1) {
      if (lo + bit > bound) continue;
      u64 n = 0;
      each_read([&](float v, int i) { n += v == cut && i < lo + bit; });
      if (sm_sum(n, s.part) <= r) lo += bit;
    }
    return lo;
  };
  // the bin at which the scanned numbers (two a thread) reach `need`, and what lies above it, in s.found_bin and s.above
  auto find = [&](u64 n0, u64 n1, u64 need, u64& total) {
    const u64 upto = sm_scan(n0 + n1, s.part, total);
    if (tid == 0) s.found_bin = kSmBins;
    __syncthreads();
    const u64 before = upto - n0 - n1;
    if (before < need && need <= before + n0) {
      s.found_bin = 2 * tid;
      s.above = before;
    } else if (before + n0 < need && need <= upto) {
      s.found_bin = 2 * tid + 1;
      s.above = before + n0;
    }
    __syncthreads();
  };

  int n_list = -1;  // a list of all that is kept, sorted: thread t has entry t in `mine`
  u64 mine = 0;
  if (top_k > 0 && top_k < V) {
    __syncthreads();
    s.count[tid] = s.count[tid + kSmThreads] = 0;
    __syncthreads();
    each([&](float v, int) {
      const int bin = bin_of(v);
      if (bin < kSmBins - 1) atomicAdd(&s.count[bin], 1u);
    });
    __syncthreads();
    u64 total;
    find(s.count[2 * tid], s.count[2 * tid + 1], top_k, total);
    const int bin = s.found_bin;
    if (bin < kSmBins) {  // (else fewer than top_k weigh anything)
      const int above = (int)s.above, in = s.count[bin];
      if (above + in <= kSmList) {
        n_list = list([&](float v, int) { return bin_of(v) <= bin; });
        mine = sm_sort(s, n_list);
        cut_at(s.order[top_k - 1]);
      } else if (in <= kSmList) {
        const int n = list([&](float v, int) { return bin_of(v) == bin; });
        sm_sort(s, n);
        cut_at(s.order[top_k - above - 1]);
      } else {
        unsigned t = 0;  // the top_k-th key
        for (unsigned bit = 1u << 31; bit; bit >>= 1) {
          u64 n = 0;
          each_read([&](float v, int) { n += sm_key(v) >= (t | bit); });
          if (sm_sum(n, s.part) >= (u64)top_k) t |= bit;
        }
        u64 n = 0;
        each_read([&](float v, int) { n += sm_key(v) > t; });
        n = sm_sum(n, s.part);
        cut = sm_value(t);
        bound = bound_of(top_k - n);
      }
      if (n_list < 0 && top_k <= kSmList) {
        n_list = list([&](float v, int i) { return is_kept(v, i); });
        mine = sm_sort(s, n_list);
      }
      n_list = min(n_list, top_k);
    }
  }

  const float u = fminf(fmaxf(a.u[b], 0.f), 1.f);
  // the draw's number among `total`, and the answer
  auto aim_of = [&](u64 total) { return min((u64)((double)u * (double)total), total - 1); };
  auto answer = [&](int i, float v, u64 total) {
    a.tokens[b] = i;
    const double e = v == big ? 0.0 : ((double)v - xmax) / (double)temperature;
    a.logprobs[b] = (float)(e - log((double)total / kSmOne));
  };

  if (n_list >= 0) {
    const float v = sm_value((unsigned)(mine >> 32));
    const int i = (int)~(unsigned)mine;
    SmWeight w = {0.0, 0};
    if (tid < n_list) w = weight(v);
    if (top_p < 1.f) {
      u64 total;
      const u64 upto = sm_scan(w.whole, s.part, total);
      const u64 target = (u64)ceil((double)top_p * (double)total);
      if (tid > 0 && upto - w.whole >= target) w = {0.0, 0};
    }
    if (w.w < (double)min_p) w.whole = 0;
    // the draw: the vocabulary in 1024 runs, of which the list's tokens fill a few
    int shift = 0;
    while ((V - 1) >> shift >= kSmThreads) ++shift;
    __syncthreads();
    s.mass[tid] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    if (w.whole) atomicAdd(&s.mass[i >> shift], w.whole);
    __syncthreads();
    u64 total;
    const u64 run = s.mass[tid], upto = sm_scan(run, s.part, total);
    const u64 aim = aim_of(total);
    if (upto > aim && upto - run <= aim) {
      s.at = tid;
      s.above = upto - run;
    }
    __syncthreads();
    const bool in = w.whole && (unsigned)(i >> shift) == s.at;
    if (in) {
      const unsigned at = atomicAdd(&s.n, 1u);
      s.order[at] = (u64)i;
      s.mass[at] = w.whole;
    }
    __syncthreads();
    if (in) {
      u64 before = s.above;
      for (unsigned k = 0; k < s.n; ++k) before += (int)s.order[k] < i ? s.mass[k] : 0;
      if (before <= aim && before + w.whole > aim) answer(i, v, total);
    }
    return;
  }

  if (top_p < 1.f) {
    __syncthreads();
    s.mass[tid] = s.mass[tid + kSmThreads] = 0;
    __syncthreads();
    each([&](float v, int i) {
      const int bin = bin_of(v);
      if (bin < kSmBins - 1 && is_kept(v, i)) atomicAdd(&s.mass[bin], weight(v).whole);
    });
    __syncthreads();
    u64 total;
    const u64 n0 = s.mass[2 * tid], n1 = s.mass[2 * tid + 1];
    sm_scan(n0 + n1, s.part, total);
    const u64 target = max((u64)ceil((double)top_p * (double)total), (u64)1);
    find(n0, n1, target, total);
    const int bin = s.found_bin;
    const u64 above = s.above;
    const int n = list([&](float v, int i) { return bin_of(v) == bin && is_kept(v, i); });
    if (n <= kSmList) {
      mine = sm_sort(s, n);
      const u64 w = tid < n ? weight(sm_value((unsigned)(mine >> 32))).whole : 0;
      const u64 before = sm_scan(w, s.part, total) - w + above;
      // the last with less than the target before it
      const bool in = tid < n && before < target;
      const u64 last = sm_sum(in, s.part);
      cut_at(s.order[last - 1]);
    } else {
      auto mass_above = [&](unsigned t) {
        u64 m = 0;
        each_read([&](float v, int i) {
          if (sm_key(v) > t && is_kept(v, i)) m += weight(v).whole;
        });
        return sm_sum(m, s.part);
      };
      unsigned t = 0;  // the smallest key with less than the target above it
      for (unsigned bit = 1u << 31; bit; bit >>= 1)
        if (mass_above(t + bit - 1) >= target) t += bit;
      const u64 before = mass_above(t), w = weight(sm_value(t)).whole;
      if (sm_value(t) > cut) {
        cut = sm_value(t);
        bound = V;
      }
      bound = bound_of(w ? (target - before + w - 1) / w : V);
    }
  }

  // the draw over the whole row: runs of 512 indices, a wave's chunk each
  __syncthreads();
  auto final_weight = [&](float v, int i) -> u64 {
    if (!is_kept(v, i)) return 0;
    const SmWeight w = weight(v);
    return w.w < (double)min_p ? 0 : w.whole;
  };
  auto run_of = [&](int j, const float (&v)[8]) {
    u64 m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m += final_weight(v[e], (j * kSmThreads + tid) * 8 - head + e);
      if (e & 1) __builtin_amdgcn_sched_barrier(0);
    }
    return m;
  };
  s.mass[tid] = 0;
  __syncthreads();
  auto sum_run = [&](int j, const float (&v)[8]) {
    u64 m = run_of(j, v);
#pragma unroll
    for (int x = 32; x; x >>= 1) m += __shfl_xor(m, x, 64);
    if (lane == 0) s.mass[j * kSmWaves + (tid >> 6)] = m;
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int j = 0; j < CH; ++j) sum_run(j, kept[j]);
  } else {
    for (int j = 0; j < chunks; ++j) {
      float v[8];
      load(j, v);
      sum_run(j, v);
    }
  }
  __syncthreads();
  u64 total;
  const u64 run = s.mass[tid], upto = sm_scan(run, s.part, total);
  const u64 aim = aim_of(total);
  if (upto > aim && upto - run <= aim) {
    s.at = tid;
    s.above = upto - run;
  }
  __syncthreads();
  const int j = s.at / kSmWaves;
  if ((int)s.at % kSmWaves != tid >> 6) return;
  float v[8];
  if constexpr (CH > 0) {
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k == j ? kept[k][e] : v[e];
  } else {
    load(j, v);
  }
  u64 m = run_of(j, v), sum = m;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) {
    const u64 o = sm_shfl_up(sum, x);
    sum += lane >= x ? o : 0;
  }
  sum += s.above;
  if (sum > aim && sum - m <= aim) {
    u64 before = sum - m;
    bool done = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = (j * kSmThreads + tid) * 8 - head + e;
      before += final_weight(v[e], i);
      if (!done && before > aim) {
        answer(i, v[e], total);
        done = true;
      }
    }
  }
}

template <typename T>
void sample_launch(const SampleParams& p, int64_t B, hipStream_t st) {
  const dim3 grid((unsigned)B);
  // a row may begin anywhere in 16 bytes, unless all begin at their start
  const bool aligned = ((uintptr_t)p.logits & 15) == 0 && (B == 1 || p.stride * sizeof(T) % 16 == 0);
  const int n = p.V + (aligned ? 0 : 16 / (int)sizeof(T) - 1);
  if (n <= 8 * kSmThreads)
    sample_kernel<T, 1><<<grid, kSmThreads, 0, st>>>(p);
  else if (n <= 16 * kSmThreads)
    sample_kernel<T, 2><<<grid, kSmThreads, 0, st>>>(p);
  else if (n <= 32 * kSmThreads)
    sample_kernel<T, 4><<<grid, kSmThreads, 0, st>>>(p);
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
