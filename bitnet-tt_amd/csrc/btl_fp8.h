// e4m3 codes (OCP: bias 7, largest 448, 0x7f is NaN) of rows with a power of
// two, on gfx950's conversions: two codes an instruction in either direction,
// the scale of the way back included.
#pragma once

#include "btl_common.h"

namespace btl {

// The factor of an exponent byte (e + 127, e in [-126, 127]).
__device__ __forceinline__ float exp_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The codes of y[0..7] * 2^e, each rounded to nearest even (2^e normal, and the
// products at most 448, so the scaling is exact and nothing saturates).
__device__ __forceinline__ uint2 to_e4m3(const float* y, int e) {
  const float f = exp_scale(e + 127);
  uint32_t r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * f, y[4 * i + 1] * f, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * f, y[4 * i + 3] * f, w, true);
    r[i] = (uint32_t)w;
  }
  return make_uint2(r[0], r[1]);
}

// Eight codes times scale (a power of two) as bf16.
__device__ __forceinline__ uint4 from_e4m3(uint2 c, float scale) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, scale, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, scale, true));
  return r;
}

}  // namespace btl
