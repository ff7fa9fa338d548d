// Absorbed latent decode over a paged cache in 16 or 4 bits (gfx950): one query token a sequence.
#include "paged.h"

namespace mla {

struct PagedDecodeParams {
  PagedParams c;
  const bf16 *q_lat, *q_rope;
  const int32_t* seq_lens;
  bf16* ctx;
  float* lse;
  int H, Hr, DL;
  int64_t q_lat_sb, q_lat_sh, q_rope_sb, q_rope_sh;
  float scale_log2;
};

// One workgroup a head of a sequence; its waves take the tokens in turn, a lane DL / 64 of the latent's values and one of the key's.
template <bool FOUR>
__global__ __launch_bounds__(256) void paged_decode_kernel(PagedDecodeParams a) {
  __shared__ float m_s[4], l_s[4], o_s[4][512];
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n = a.DL / 64;
  float q[8], o[8], v[8];
  for (int i = 0; i < n; ++i) {
    q[i] = (float)a.q_lat[b * a.q_lat_sb + h * a.q_lat_sh + 64 * i + lane];
    o[i] = 0.f;
  }
  const float qr = (float)a.q_rope[b * a.q_rope_sb + h * a.q_rope_sh + lane];
  const int64_t len = min((int64_t)max(a.seq_lens[b], 0), (int64_t)a.c.table_pages * a.c.size);
  float m = -INFINITY, l = 0.f;
  const int kr = a.DL + (a.Hr > 1 ? 64 * h : 0);
  for (int64_t t = w; t < len; t += 4) {
    const int id = page_of(a.c, b, t / a.c.size);
    if (id < 0) continue;
    const int slot = (int)(t % a.c.size);
    const unsigned char* row = a.c.pages + id * a.c.page_stride + (int64_t)slot * a.c.row_bytes;
    auto value = [&](int col) {
      if (!FOUR) return (float)reinterpret_cast<const bf16*>(row)[col];
      const int byte = row[col >> 1];
      return (float)((col & 1 ? byte >> 4 : byte & 15) - 8) *
             (float)a.c.scales[id * a.c.scale_stride + (col >> 6) * a.c.size + slot];
    };
    float s = qr * value(kr + lane);
    for (int i = 0; i < n; ++i) {
      v[i] = value(64 * i + lane);
      s += q[i] * v[i];
    }
    for (int x = 32; x; x >>= 1) s += wave_shfl_xor(s, x);
    s *= a.scale_log2;
    const float m_new = fmaxf(m, s), r = m == -INFINITY ? 0.f : fast_exp2(m - m_new), p = fast_exp2(s - m_new);
    m = m_new;
    l = l * r + p;
    for (int i = 0; i < n; ++i) o[i] = o[i] * r + p * v[i];
  }
  if (lane == 0) {
    m_s[w] = m;
    l_s[w] = l;
  }
  for (int i = 0; i < n; ++i) o_s[w][64 * i + lane] = o[i];
  __syncthreads();
  const float M = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
  float L = 0.f, f[4];
  for (int i = 0; i < 4; ++i) {
    f[i] = M == -INFINITY ? 0.f : fast_exp2(m_s[i] - M);
    L += f[i] * l_s[i];
  }
  for (int c = threadIdx.x; c < a.DL; c += 256) {
    const float s = f[0] * o_s[0][c] + f[1] * o_s[1][c] + f[2] * o_s[2][c] + f[3] * o_s[3][c];
    a.ctx[(int64_t)blockIdx.x * a.DL + c] = (bf16)(L > 0.f ? s / L : 0.f);
  }
  if (threadIdx.x == 0) a.lse[blockIdx.x] = L > 0.f ? (M + fast_log2(L)) * kLn2 : -INFINITY;
}

}  // namespace mla

using namespace mla;

extern "C" size_t mla_paged_decode_workspace_bytes(const mla_paged_decode_args* a) {
  return 0;
}

extern "C" int mla_paged_decode(const mla_paged_decode_args* a, void* stream) {
  const char* op = "mla_paged_decode";
  MLA_CHECK(a, MLA_ERR_INVALID_ARG, "%s: null args", op);
  MLA_CHECK(a->B >= 0 && a->B < (1 << 20) && a->H >= 1 && a->H <= 1024, MLA_ERR_INVALID_ARG, "%s: B %lld or H %lld is out of range", op,
            (long long)a->B, (long long)a->H);
  PagedDecodeParams p;
  MLA_TRY(paged_setup(a->cache, op, a->B, p.c));
  MLA_CHECK(a->cache.n_k_rope_heads == 1 || a->cache.n_k_rope_heads == a->H, MLA_ERR_INVALID_ARG,
            "%s: n_k_rope_heads must be 1 or H (%lld)", op, (long long)a->H);
  MLA_TRY(check_scale(op, a->scale));
  if (a->B == 0) return MLA_OK;
  MLA_CHECK(a->q_lat && a->q_rope && a->seq_lens && a->ctx && a->lse, MLA_ERR_INVALID_ARG, "%s: null pointer", op);
  MLA_CHECK((((uintptr_t)a->q_lat | (uintptr_t)a->q_rope | (uintptr_t)a->ctx) & 15) == 0 && (((uintptr_t)a->seq_lens | (uintptr_t)a->lse) & 3) == 0,
            MLA_ERR_INVALID_ARG, "%s: a pointer is not aligned", op);
  const int64_t st[] = {a->q_lat_sb, a->q_lat_sh, a->q_rope_sb, a->q_rope_sh};
  for (int64_t s : st) MLA_CHECK(s >= 0 && (s & 7) == 0, MLA_ERR_INVALID_ARG, "%s: strides must be non-negative multiples of 8", op);
  p.q_lat = (const bf16*)a->q_lat;
  p.q_rope = (const bf16*)a->q_rope;
  p.seq_lens = a->seq_lens;
  p.ctx = (bf16*)a->ctx;
  p.lse = a->lse;
  p.H = (int)a->H;
  p.Hr = (int)a->cache.n_k_rope_heads;
  p.DL = (int)a->cache.d_latent;
  p.q_lat_sb = a->q_lat_sb;
  p.q_lat_sh = a->q_lat_sh;
  p.q_rope_sb = a->q_rope_sb;
  p.q_rope_sh = a->q_rope_sh;
  p.scale_log2 = a->scale * kLog2e;
  const dim3 grid((unsigned)(a->B * a->H));
  if (p.c.scales)
    paged_decode_kernel<true><<<grid, 256, 0, (hipStream_t)stream>>>(p);
  else
    paged_decode_kernel<false><<<grid, 256, 0, (hipStream_t)stream>>>(p);
  return launch_status(op);
}
