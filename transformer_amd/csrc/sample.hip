// Drawing one token for each row of logits: temperature, top-k, top-p, min-p and the draw from a given number (gfx950).
#include <cmath>

#include "mla_common.h"

namespace mla {

constexpr int kSmThreads = 1024;
constexpr int kSmMaxV = 1 << 19;  // 2^19 weights of up to 2^44 add up below 2^63

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

// a sum over the workgroup, the same in every thread (integers: in any order)
__device__ __forceinline__ uint64_t sm_sum(uint64_t v, uint64_t* lds) {
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t s = 0;
  for (int i = 0; i < kSmThreads / 64; ++i) s += lds[i];
  return s;
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleParams a) {
  __shared__ uint64_t lds[kSmThreads / 64];
  __shared__ uint32_t top_s[kSmThreads / 64];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, V = a.V;
  const T* x = (const T*)a.logits + b * a.stride;
  const float temperature = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const float top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const float min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  const int top_k = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const bool greedy = !(temperature > 0.f);

  uint32_t top = 0;
  for (int i = tid; i < V; i += kSmThreads) top = max(top, sm_key((float)x[i]));
  for (int m = 32; m; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, 64));
  if ((tid & 63) == 0) top_s[tid >> 6] = top;
  __syncthreads();
  for (int i = 0; i < kSmThreads / 64; ++i) top = max(top, top_s[i]);
  const double xmax = (double)sm_value(top);
  if (xmax == -INFINITY) {
    if (tid == 0) {
      a.tokens[b] = -1;
      a.logprobs[b] = -INFINITY;
    }
    return;
  }
  auto weight = [&](uint32_t key) -> double {
    if (key == top) return 1.0;
    const float v = sm_value(key);
    return v == -INFINITY || greedy ? 0.0 : exp(((double)v - xmax) / (double)temperature);
  };
  auto whole = [&](double w) { return (uint64_t)(w * 17592186044416.0); };  // 2^44

  // what is kept: keys above `cut`, and those equal to it below index `bound`
  uint32_t cut = 0;
  int bound = V;
  auto kept = [&](uint32_t key, int i) { return key > cut || (key == cut && i < bound); };
  // the bound that leaves `r` of the keys equal to `cut` that are kept now
  auto bound_of = [&](uint64_t r) {
    int lo = 0;  // the largest index bound with at most r of them
    for (int bit = 1 << 19; bit; bit >>= 1) {
      if (lo + bit > bound) continue;
      uint64_t n = 0;
      for (int i = tid; i < lo + bit; i += kSmThreads) n += sm_key((float)x[i]) == cut;
      if (sm_sum(n, lds) <= r) lo += bit;
    }
    return lo;
  };

  const int64_t k = greedy ? 1 : top_k;
  if (k > 0 && k < V) {
    uint32_t t = 0;
    for (uint32_t bit = 1u << 31; bit; bit >>= 1) {
      uint64_t n = 0;
      for (int i = tid; i < V; i += kSmThreads) n += sm_key((float)x[i]) >= (t | bit);
      if (sm_sum(n, lds) >= (uint64_t)k) t |= bit;
    }
    uint64_t above = 0;
    for (int i = tid; i < V; i += kSmThreads) above += sm_key((float)x[i]) > t;
    above = sm_sum(above, lds);
    cut = t;
    bound = bound_of(k - above);
  }
  auto mass_above = [&](uint32_t t) {  // of the kept ones
    uint64_t s = 0;
    for (int i = tid; i < V; i += kSmThreads) {
      const uint32_t key = sm_key((float)x[i]);
      if (key > t && kept(key, i)) s += whole(weight(key));
    }
    return sm_sum(s, lds);
  };
  if (top_p < 1.f) {
    uint64_t total = mass_above(cut);
    uint64_t ties = 0;
    for (int i = tid; i < V; i += kSmThreads) ties += sm_key((float)x[i]) == cut && i < bound;
    total += sm_sum(ties, lds) * whole(weight(cut));
    const uint64_t target = top_p > 0.f ? (uint64_t)ceil((double)top_p * (double)total) : 0;  // kept while the sum before is below
    uint32_t t = 0;  // the smallest with a sum above it that is below the target
    for (uint32_t bit = 1u << 31; bit; bit >>= 1)
      if (mass_above(t + bit - 1) >= target && t + bit - 1 < top) t += bit;
    if (target == 0) t = top;
    const uint64_t before = mass_above(t), w = whole(weight(t));
    if (t > cut) {
      cut = t;
      bound = V;
    }
    if (t == cut) {
      const uint64_t r = target == 0 ? 1 : w ? (target - before + w - 1) / w : V;
      bound = bound_of(r);
    }
  }
  auto final_weight = [&](int i) -> uint64_t {
    const uint32_t key = sm_key((float)x[i]);
    if (!kept(key, i)) return 0;
    const double w = weight(key);
    return w < fmin((double)min_p, 1.0) ? 0 : whole(w);
  };
  // the draw: each thread a run of the vocabulary
  const int per = (V + kSmThreads - 1) / kSmThreads, i0 = min(tid * per, V), i1 = min(i0 + per, V);
  uint64_t mine = 0;
  for (int i = i0; i < i1; ++i) mine += final_weight(i);
  uint64_t upto = mine;
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t o = __shfl_up(upto, m, 64);
    if ((tid & 63) >= m) upto += o;
  }
  __syncthreads();
  if ((tid & 63) == 63) lds[tid >> 6] = upto;
  __syncthreads();
  uint64_t total = 0;
  for (int i = 0; i < kSmThreads / 64; ++i) {
    if (i < tid >> 6) upto += lds[i];
    total += lds[i];
  }
  const float u = a.u[b];
  const double at = fmin(fmax((double)u, 0.0), 1.0) * (double)total;
  const uint64_t aim = min((uint64_t)at, total - 1);  // the first sum above it
  if (upto > aim && upto - mine <= aim) {
    uint64_t s = upto - mine;
    int i = i0;
    for (; i < i1 - 1; ++i) {
      s += final_weight(i);
      if (s > aim) break;
    }
    a.tokens[b] = i;
    const float v = sm_value(sm_key((float)x[i]));
    const double e = greedy || (double)v == xmax ? 0.0 : ((double)v - xmax) / (double)temperature;
    a.logprobs[b] = (float)(e - log((double)total / 17592186044416.0));
  }
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
    sample_kernel<bf16><<<dim3((unsigned)a->B), kSmThreads, 0, (hipStream_t)stream>>>(p);
  else
    sample_kernel<float><<<dim3((unsigned)a->B), kSmThreads, 0, (hipStream_t)stream>>>(p);
  return launch_status(op);
}
