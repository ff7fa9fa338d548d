// Activations of the linear layers' epilogues, their slopes, and the pre-activations that a backward keeps.
#pragma once

#include "mla_common.h"

namespace mla {

// 1 / (1 + e^-x): 0 and 1 at the ends (2^inf = inf, 1 / inf = 0)
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + fast_exp2(-x * kLog2e)); }

// 0.5 (1 + tanh v) = sigmoid(2 v) with v = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kGelu2c = 1.5957691216057308f, kGeluCube = 0.044715f;

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == MLA_ACT_SILU) return z * sigmoid(z);
  if (ACT == MLA_ACT_GELU_TANH) return z * sigmoid(kGelu2c * (z + kGeluCube * z * z * z));
  if (ACT == MLA_ACT_RELU) return z < 0.f ? 0.f : z;  // (a NaN stays one)
  return z;
}

// value and slope together (they share the sigmoid)
template <int ACT>
__device__ __forceinline__ void act_both(float z, float& value, float& slope) {
  if (ACT == MLA_ACT_SILU) {
    const float s = sigmoid(z);
    value = z * s;
    slope = s * (1.f + z * (1.f - s));
  } else if (ACT == MLA_ACT_GELU_TANH) {
    const float z2 = fminf(z * z, 1e30f);  // (the slope's 0 times an infinity would be a NaN)
    const float s = sigmoid(kGelu2c * (z + kGeluCube * z * z2));
    value = z * s;
    slope = s + z * s * (1.f - s) * (kGelu2c * (1.f + 3.f * kGeluCube * z2));
  } else if (ACT == MLA_ACT_RELU) {
    value = z < 0.f ? 0.f : z;
    slope = z > 0.f ? 1.f : 0.f;
  } else {
    value = z;
    slope = 1.f;
  }
}

// Pre-activations kept for a backward: the upper 24 bits of the fp32 value (cut, not rounded: off by less than 2^-15 of it, a
// hundredth of the bf16 rounding of what is computed from it, for no instruction), as a 32 x 32 block's accumulators lie in the
// lanes (32 m x 32 n, see gemm_core.h): 2 x 16 bytes of upper halves and 16 bytes of the next 8 bits per lane, 3 KiB a block.
// Written and read by whole 1 KiB runs straight from registers.  In bf16 they would cost 2 KiB and their rounding would add
// to that of the gradients computed from them: an rms error of 1.7 to 2 times a single rounding's instead of 1.4.
constexpr int kSavedBlock = 3 << 10;

__device__ __forceinline__ void saved_store(unsigned char* block, int lane, const f32x16& v) {
  u32x4 hi[2], lo;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    hi[k >> 2][k & 3] = __builtin_amdgcn_perm(__float_as_uint(v[2 * k + 1]), __float_as_uint(v[2 * k]), 0x07060302u);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k]), 0x0c0c0501u);
    const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(v[4 * k + 3]), __float_as_uint(v[4 * k + 2]), 0x0c0c0501u);
    lo[k] = a | (b << 16);
  }
  __builtin_nontemporal_store(hi[0], (u32x4*)(block + lane * 16));
  __builtin_nontemporal_store(hi[1], (u32x4*)(block + 1024 + lane * 16));
  __builtin_nontemporal_store(lo, (u32x4*)(block + 2048 + lane * 16));
}

struct SavedRegs {
  u32x4 hi[2], lo;
};
__device__ __forceinline__ SavedRegs saved_load(const unsigned char* block, int lane) {
  return SavedRegs{{__builtin_nontemporal_load((const u32x4*)(block + lane * 16)),
                    __builtin_nontemporal_load((const u32x4*)(block + 1024 + lane * 16))},
                   __builtin_nontemporal_load((const u32x4*)(block + 2048 + lane * 16))};
}
__device__ __forceinline__ float saved_value(const SavedRegs& r, int e) {
  const uint32_t h = r.hi[e >> 3][(e >> 1) & 3], l = r.lo[e >> 2];
  const uint32_t top = (e & 1) ? (h & 0xffff0000u) : (h << 16);
  return __uint_as_float(top | (((l >> (8 * (e & 3))) & 255u) << 8));
}

}  // namespace mla
