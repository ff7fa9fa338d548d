// The norm of many gradients taken together, and their clipping by it (gfx950): the training step's clip_grad_norm_
// (train.py:454) in two passes, with no host synchronisation and no tensor of its own per gradient.
//
// HBM bound: every gradient is read for the norm, then read and written for the factor.  The tensors' addresses travel in the
// kernel arguments, kGnTensors a launch; a tensor is cut into chunks of 64 KiB, which the workgroups take in turn.  Squares are
// summed in fp64 (the conversions and products run under the loads), so that no finite gradient overflows, each workgroup's sum
// goes to the workspace and every workgroup of the second pass adds them in the same order: results repeat bit for bit.
// The second pass walks the chunks backwards: what the first one read last is still in the last-level cache.
// 1228 million fp32 gradients in 338 tensors (4.9 GB, three launches a pass): norm 876 us, 5.6 TB/s, factor 1912 us, 5.1 TB/s, what
// a large copy reaches; twice the grid, eight loads in flight and stores past the caches changed nothing.  50 tensors of 4
// million: 7 and 12 us (chunks of 16 KiB: 2 us less at 1 million elements, 3 more at 8).
#include <algorithm>
#include <cmath>
#include <vector>

#include "mla_common.h"

namespace mla {

constexpr int kGnTensors = 128;      // of a launch (3 KiB of arguments)
constexpr int kGnVecs = 4096;        // 16-byte vectors of a chunk
constexpr int kGnGrid = 1024;        // workgroups of a launch, at most
constexpr int kGnThreads = 256;
constexpr int64_t kGnMaxTensors = 1 << 20;

struct GnTable {
  void* ptr[kGnTensors];
  int64_t n[kGnTensors];
  int first[kGnTensors + 1];  // first chunk
  unsigned char bf16s[kGnTensors];
  int count;
};

struct GnChunk {
  unsigned char* base;  // of the tensor's aligned body
  int64_t v0, v1;       // its vectors
  int head, tail;       // elements before the body and behind it, where the chunk is the first or the last
  int64_t body;         // vectors of the whole body
  bool is_bf16;
};

inline __host__ __device__ int gn_head(uintptr_t p, int64_t n, int es) {
  const int64_t h = (int64_t)((16 - (p & 15)) & 15) / es;
  return (int)(h < n ? h : n);
}

__device__ __forceinline__ GnChunk gn_chunk(const GnTable& t, int k, int c) {
  GnChunk r;
  r.is_bf16 = t.bf16s[k] != 0;
  const int es = r.is_bf16 ? 2 : 4, ve = 16 / es;
  const int64_t n = t.n[k];
  const int head = gn_head((uintptr_t)t.ptr[k], n, es);
  r.base = (unsigned char*)t.ptr[k] + (int64_t)head * es;
  r.body = (n - head) / ve;
  r.v0 = (int64_t)(c - t.first[k]) * kGnVecs;
  r.v1 = r.v0 + kGnVecs < r.body ? r.v0 + kGnVecs : r.body;
  r.head = c == t.first[k] ? head : 0;
  r.tail = c + 1 == t.first[k + 1] ? (int)(n - head - r.body * ve) : 0;
  return r;
}

// the tensor of chunk c: the last k with first[k] <= c (tensors without elements have no chunk)
__device__ __forceinline__ int gn_find(const GnTable& t, int c) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

// values of a 16-byte vector, and of an element
template <class F>
__device__ __forceinline__ void gn_values(const u32x4& v, bool is_bf16, F&& f) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (is_bf16) {
      f(lo_bf16(v[e]));
      f(hi_bf16(v[e]));
    } else {
      f(__uint_as_float(v[e]));
    }
  }
}
__device__ __forceinline__ float gn_element(const unsigned char* p, bool is_bf16) {
  return is_bf16 ? bf16_bits_to_f32(*(const unsigned short*)p) : *(const float*)p;
}

// sum, or the larger of the two where a NaN wins
template <bool MAX>
__device__ __forceinline__ double gn_join(double a, double b) {
  if (!MAX) return a + b;
  return b > a || b != b ? b : a;
}
template <bool MAX>
__device__ __forceinline__ double gn_take(double a, float x) {
  if (!MAX) return __builtin_fma((double)x, (double)x, a);
  return gn_join<true>(a, (double)fabsf(x));
}

// the workgroup's values joined in a fixed order; every thread gets the result
template <bool MAX>
__device__ __forceinline__ double gn_block(double v) {
  __shared__ double wave[kGnThreads / 64];
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) v = gn_join<MAX>(v, __shfl_xor(v, s, 64));
  if ((threadIdx.x & 63) == 0) wave[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = wave[0];
#pragma unroll
  for (int w = 1; w < kGnThreads / 64; ++w) r = gn_join<MAX>(r, wave[w]);
  return r;
}

template <bool MAX>
__global__ __launch_bounds__(kGnThreads) void grad_norm_kernel(GnTable t, double* part) {
  const int tid = threadIdx.x, chunks = t.first[t.count];
  double acc = 0.0;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const GnChunk k = gn_chunk(t, gn_find(t, c), c);
    const int es = k.is_bf16 ? 2 : 4;
    int64_t v = k.v0 + tid;
    for (; v + 3 * kGnThreads < k.v1; v += 4 * kGnThreads) {  // four loads in flight
      u32x4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = ldg16(k.base + (v + e * kGnThreads) * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) gn_values(x[e], k.is_bf16, [&](float f) { acc = gn_take<MAX>(acc, f); });
    }
    for (; v < k.v1; v += kGnThreads) gn_values(ldg16(k.base + v * 16), k.is_bf16, [&](float f) { acc = gn_take<MAX>(acc, f); });
    if (tid < k.head) acc = gn_take<MAX>(acc, gn_element(k.base - (int64_t)(tid + 1) * es, k.is_bf16));
    if (tid < k.tail) acc = gn_take<MAX>(acc, gn_element(k.base + k.body * 16 + (int64_t)tid * es, k.is_bf16));
  }
  acc = gn_block<MAX>(acc);
  if (tid == 0) part[blockIdx.x] = acc;
}

// The norm from the n parts, in every workgroup alike; then this launch's chunks are multiplied by the factor (a launch
// without tensors only stores the norm).
template <bool MAX>
__global__ __launch_bounds__(kGnThreads) void grad_scale_kernel(GnTable t, const double* part, int n, float max_norm,
                                                                float* norm_out) {
  const int tid = threadIdx.x, chunks = t.first[t.count];
  double acc = 0.0;
  for (int i = tid; i < n; i += kGnThreads) acc = gn_join<MAX>(acc, part[i]);
  acc = gn_block<MAX>(acc);
  const double norm = MAX ? acc : sqrt(acc);
  if (norm_out && blockIdx.x == 0 && tid == 0) *norm_out = (float)norm;
  const double f64 = (double)max_norm / (norm + 1e-6);
  const float f = (float)(f64 > 1.0 ? 1.0 : f64);  // (a NaN stays one)
  for (int r = blockIdx.x; r < chunks; r += gridDim.x) {
    const int c = chunks - 1 - r;
    const GnChunk k = gn_chunk(t, gn_find(t, c), c);
    const int es = k.is_bf16 ? 2 : 4;
    auto scaled = [&](u32x4 x) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = k.is_bf16 ? pack_bf16x2(lo_bf16(x[e]) * f, hi_bf16(x[e]) * f) : __float_as_uint(__uint_as_float(x[e]) * f);
      return x;
    };
    auto element = [&](unsigned char* at) {
      const float x = gn_element(at, k.is_bf16) * f;
      if (k.is_bf16) *(bf16*)at = (bf16)x;
      else *(float*)at = x;
    };
    int64_t v = k.v0 + tid;
    for (; v + 3 * kGnThreads < k.v1; v += 4 * kGnThreads) {
      u32x4 x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = ldg16(k.base + (v + e * kGnThreads) * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) stg16(k.base + (v + e * kGnThreads) * 16, scaled(x[e]));
    }
    for (; v < k.v1; v += kGnThreads) stg16(k.base + v * 16, scaled(ldg16(k.base + v * 16)));
    if (tid < k.head) element(k.base - (int64_t)(tid + 1) * es);
    if (tid < k.tail) element(k.base + k.body * 16 + (int64_t)tid * es);
  }
}

// one launch's tensors from `at` on (those without elements are left out); returns the next tensor
static int64_t gn_fill(const mla_grad_norm_args* a, int64_t at, GnTable& t) {
  t.count = 0;
  t.first[0] = 0;
  while (at < a->n_tensors && t.count < kGnTensors) {
    const int64_t n = a->numels[at];
    const bool b = a->dtypes[at] == MLA_DTYPE_BF16;
    if (n > 0) {
      const int es = b ? 2 : 4;
      const int64_t body = (n - gn_head((uintptr_t)a->ptrs[at], n, es)) / (16 / es);
      const int64_t chunks = std::max<int64_t>(1, (body + kGnVecs - 1) / kGnVecs);
      t.ptr[t.count] = a->ptrs[at];
      t.n[t.count] = n;
      t.bf16s[t.count] = b;
      t.first[t.count + 1] = t.first[t.count] + (int)chunks;
      ++t.count;
    }
    ++at;
  }
  return at;
}

static int gn_grid(const GnTable& t) { return std::min(t.first[t.count], kGnGrid); }

static int gn_sizes(const char* op, const mla_grad_norm_args* a) {
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_CHECK(a->n_tensors >= 0 && a->n_tensors < kGnMaxTensors, MLA_ERR_INVALID_ARG, "%s: %lld tensors", op, (long long)a->n_tensors);
  MLA_CHECK(a->n_tensors == 0 || (a->ptrs && a->numels && a->dtypes), MLA_ERR_INVALID_ARG, "%s: null table", op);
  for (int64_t i = 0; i < a->n_tensors; ++i) {
    MLA_CHECK(a->dtypes[i] == MLA_DTYPE_F32 || a->dtypes[i] == MLA_DTYPE_BF16, MLA_ERR_UNSUPPORTED, "%s: dtype of tensor %lld",
              op, (long long)i);
    MLA_CHECK(a->numels[i] >= 0 && a->numels[i] < (1ll << 36), MLA_ERR_INVALID_ARG, "%s: size of tensor %lld", op, (long long)i);
    const uintptr_t es = a->dtypes[i] == MLA_DTYPE_BF16 ? 2 : 4;
    MLA_CHECK(a->numels[i] == 0 || (a->ptrs[i] && (uintptr_t)a->ptrs[i] % es == 0), MLA_ERR_INVALID_ARG,
              "%s: tensor %lld must be aligned to its elements", op, (long long)i);
  }
  return MLA_OK;
}

static int gn_check(const char* op, const mla_grad_norm_args* a) {
  MLA_TRY(gn_sizes(op, a));
  MLA_CHECK(a->norm && ((uintptr_t)a->norm & 3) == 0, MLA_ERR_INVALID_ARG, "%s: norm must be given, 4-byte aligned", op);
  const size_t need = mla_grad_norm_workspace_bytes(a);
  MLA_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace & 15) == 0), MLA_ERR_WORKSPACE,
            "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", op, need, a->workspace_bytes);
  return MLA_OK;
}

// two workgroups that write the same element would race: tensors given twice or overlapping are refused
static int gn_check_apart(const char* op, const mla_grad_norm_args* a) {
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  for (int64_t i = 0; i < a->n_tensors; ++i)
    if (a->numels[i] > 0) {
      const uintptr_t b = (uintptr_t)a->ptrs[i];
      r.emplace_back(b, b + (uintptr_t)a->numels[i] * (a->dtypes[i] == MLA_DTYPE_BF16 ? 2 : 4));
    }
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    MLA_CHECK(r[i - 1].second <= r[i].first, MLA_ERR_INVALID_ARG, "%s: two tensors overlap", op);
  return MLA_OK;
}

template <bool MAX>
static int gn_run(const char* op, const mla_grad_norm_args* a, bool clip, hipStream_t s) {
  double* const part = (double*)a->workspace;
  int n = 0;
  std::vector<GnTable> tables;
  for (int64_t at = 0; at < a->n_tensors;) {
    tables.emplace_back();
    GnTable& t = tables.back();
    at = gn_fill(a, at, t);
    if (t.count == 0) {
      tables.pop_back();
      continue;
    }
    grad_norm_kernel<MAX><<<dim3((unsigned)gn_grid(t)), dim3(kGnThreads), 0, s>>>(t, part + n);
    MLA_TRY(launch_status(op));
    n += gn_grid(t);
  }
  if (!clip || tables.empty()) {
    GnTable none;
    none.count = 0;
    none.first[0] = 0;
    grad_scale_kernel<MAX><<<dim3(1), dim3(kGnThreads), 0, s>>>(none, part, n, 0.f, a->norm);
    return launch_status(op);
  }
  for (size_t i = tables.size(); i-- > 0;) {  // backwards, as their chunks
    grad_scale_kernel<MAX><<<dim3((unsigned)gn_grid(tables[i])), dim3(kGnThreads), 0, s>>>(
        tables[i], part, n, a->max_norm, i + 1 == tables.size() ? a->norm : nullptr);
    MLA_TRY(launch_status(op));
  }
  return MLA_OK;
}

// no C++ exception leaves a C entry point
template <class F>
static int gn_guarded(const char* op, F&& f) {
  try {
    return f();
  } catch (...) {
    set_error("%s: out of host memory", op);
    return MLA_ERR_WORKSPACE;
  }
}

}  // namespace mla

using namespace mla;

extern "C" size_t mla_grad_norm_workspace_bytes(const mla_grad_norm_args* a) {
  if (!a || a->n_tensors <= 0 || a->n_tensors >= kGnMaxTensors) return 0;
  return (size_t)((a->n_tensors + kGnTensors - 1) / kGnTensors) * kGnGrid * sizeof(double);
}

extern "C" int mla_grad_norm(const mla_grad_norm_args* a, void* stream) {
  const char* op = "mla_grad_norm";
  return gn_guarded(op, [&]() -> int {
    MLA_TRY(gn_check(op, a));
    return a->norm_is_max ? gn_run<true>(op, a, false, (hipStream_t)stream) : gn_run<false>(op, a, false, (hipStream_t)stream);
  });
}

extern "C" int mla_grad_clip(const mla_grad_norm_args* a, void* stream) {
  const char* op = "mla_grad_clip";
  return gn_guarded(op, [&]() -> int {
    MLA_TRY(gn_check(op, a));
    MLA_CHECK(a->max_norm >= 0.f, MLA_ERR_INVALID_ARG, "%s: max_norm must be at least 0", op);
    MLA_TRY(gn_check_apart(op, a));
    return a->norm_is_max ? gn_run<true>(op, a, true, (hipStream_t)stream) : gn_run<false>(op, a, true, (hipStream_t)stream);
  });
}
