// Shared by the sources of the 4-bit weights.
#pragma once

#include "kad_common.h"

namespace kad_q4 {

// columns of a weight, so that offsets within a row of blocks stay in 32 bits
constexpr int kMaxK = 1 << 20;
// rows of a weight
constexpr int kMaxN = 1 << 26;

// the value of a scale's byte: 2^(byte - 127), NaN for 255
__device__ __forceinline__ float scale_value(uint32_t byte) {
  if (byte == 255u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(byte ? byte << 23 : 1u << 22);
}

// the 8 codes of a word as floats
__device__ __forceinline__ void codes_to_float(uint32_t w, float* f) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2);
  const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
  f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1];
  f[4] = c[0], f[5] = c[1], f[6] = d[0], f[7] = d[1];
}

}  // namespace kad_q4
