// Device helpers for 4-bit weights (layout and values: fp4.hip).
#pragma once

#include "common.h"

namespace ttamd {

// 2^(byte - 127) of tile j of a lane's four exponent bytes; byte 255 gives the
// bits of an infinity, which the conversion takes for NaN.
__device__ __forceinline__ float fp4_scale(uint32_t bytes, int j) {
  return __uint_as_float((bytes >> (8 * j) & 0xffu) << 23);
}

// Eight codes (a dword, low half byte first) times their scale as eight bf16.
__device__ __forceinline__ uint4 fp4_bits(uint32_t q, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
  return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                    __builtin_bit_cast(uint32_t, d));
}
__device__ __forceinline__ bf16x8_t fp4_frag(uint32_t q, float scale) {
  return __builtin_bit_cast(bf16x8_t, fp4_bits(q, scale));
}

}  // namespace ttamd
