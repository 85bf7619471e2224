// Quantisation of one block of 32 values to 4-bit floats (see mx.hip).
#pragma once

#include "common.hpp"

namespace trnblas {

// Scale byte of a block whose largest magnitude has these bits (as fp32):
// floor(log2) - 2 so that it lands in [4, 8), not below 2^-127; infinities and
// NaN give 255.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// 2^-(byte - 127)
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __builtin_bit_cast(float, (254u - byte) << 23); }

// Eight values times inv (exact but for results far below 0.25) to eight
// codes: the conversion rounds to nearest even and saturates at 6.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float inv) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0] * inv, v[1] * inv, 1.0f, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2] * inv, v[3] * inv, 1.0f, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4] * inv, v[5] * inv, 1.0f, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6] * inv, v[7] * inv, 1.0f, 3);
  return c;
}

}  // namespace trnblas
