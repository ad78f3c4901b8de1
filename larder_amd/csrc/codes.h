// e4m3 codes with power-of-two scales: what the paged cache (rope.hip) and the norms' 8-bit rows (norm.hip) are written in.
#pragma once
#include "lmoe_common.h"

namespace lmoe {

// the least s >= -100 with m <= 448 2^s
__device__ __forceinline__ float scale_for(float m) {
  const uint32_t u = __float_as_uint(m);
  // m = (1 + f) 2^e with 448 = 1.75 2^8
  const int e = int(u >> 23) - 127, s = e - 8 + ((u & 0x7fffffu) > 0x600000u);
  return __uint_as_float(uint32_t(max(s, -100) + 127) << 23);
}

// four floats to e4m3 (nearest even; the values are within 448)
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}
// e4m3 codes 0, 1 (HI: 2, 3) of a word as floats
template <bool HI>
__device__ __forceinline__ float2 from_e4m3(uint32_t w) {
  const auto v = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), HI);
  return float2{v[0], v[1]};
}
__device__ __forceinline__ float finite_or_nan(float v) {
  return (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : v;
}

}  // namespace lmoe
