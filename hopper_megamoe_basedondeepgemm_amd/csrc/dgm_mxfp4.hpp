// MXFP4 blocks: 32 values as E2M1 codes under one E8M0 scale. Shared by the kernels that write such rows.
#pragma once
#include "dgm_rows.hpp"

namespace dgm {

// Scale code of a block whose largest magnitude has these bits: e + 127 for the least power of two 2^e with
// max(amax, floor) <= 6 2^e (6 = 1.5 2^2, so the mantissa decides between exponent - 2 and - 1), at least 1; 255
// (E8M0's NaN) where the block holds an infinity or NaN. The maximum is one of integers, which keeps a NaN.
DGM_DEV uint32_t mx_scale_code(uint32_t amax_bits, uint32_t floor_bits) {
  const uint32_t b = amax_bits > floor_bits ? amax_bits : floor_bits;
  const int c = (int)((b + 0x3fffffu) >> 23) - 2;
  return amax_bits >= 0x7f800000u ? 255u : (uint32_t)(c < 1 ? 1 : c);
}
DGM_DEV uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
DGM_DEV uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
DGM_DEV uint32_t magnitude8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_u32(m, magnitude(v[i]));
  return m;
}
// Magnitudes of two 16-bit elements in a dword, and the larger of each half: bf16 and fp16 order as their bits do.
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
DGM_DEV uint32_t max_pairs(uint32_t m, uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, m), __builtin_bit_cast(us2, w & 0x7fff7fffu)));
}
// the fp32 bits of a 16-bit magnitude (an infinity or NaN stays one)
template <int T>
DGM_DEV uint32_t magnitude_bits(uint32_t half) {
  if constexpr (T == T_F16) return __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)half));
  else return half << 16;
}
// maximum over aligned groups of four lanes (all active), in each of them
DGM_DEV uint32_t max_u32_lanes4(uint32_t v) {
  v = max_u32(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));      // quad_perm [1,0,3,2]
  return max_u32(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
}

// E2M1 codes of eight values of a block with scale code `code`, two a byte, the first in the low half: the nearest
// code, midpoints to the smaller magnitude, no negative zero; a block of scale 255 has zeros. The conversion
// instruction rounds midpoints to even, so values are moved off them first. 16-bit sources (at most 11 significant
// bits) shrink by 2^-13: one on a midpoint (3 bits at most) falls below it, one beyond by at least 2^-11 of itself
// stays beyond. fp32 sources move one unit towards zero where their last 16 bits are zero, as a midpoint's are.
template <int T>
DGM_DEV uint32_t e2m1_codes8(const float* v, uint32_t code) {
#pragma clang fp contract(off)
  float q[8];
  const float inv = e8m0_inv(code);
  if constexpr (T != T_F32) {
    const float k = inv * (1.0f - 0x1p-13f);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] * k;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = __float_as_uint(v[i] * inv);
      const uint32_t m = u & 0x7fffffffu;
      q[i] = __uint_as_float(u - ((u & 0xffffu) == 0u && m != 0u ? 1u : 0u));
    }
  }
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[0], q[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[2], q[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[4], q[5], 1.0f, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, q[6], q[7], 1.0f, 3);
  const uint32_t some = (w | w >> 1 | w >> 2) & 0x11111111u;      // (codes that are not zero keep their sign)
  w &= 0x77777777u | some << 3;
  return code == 255u ? 0u : w;
}

}  // namespace dgm
