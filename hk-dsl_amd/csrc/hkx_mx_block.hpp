// A 32-column MX block held by the 4 threads of a quad, 8 fp32 values each: its largest magnitude, and
// its codes and E8M0 scale byte as MXFP4 or MXFP8. A block with an infinity or a NaN is NaN: scale 255,
// codes 0.
#pragma once

#include "hkx_device.hpp"

namespace hkx {

template <int CTRL>
HKX_DEV uint32_t quad_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}

// The bits of the block's largest magnitude (of whole quads): an infinity's or a NaN's are 0x7f800000 or more.
HKX_DEV uint32_t mx_block_top(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
  return quad_max<0x4e>(quad_max<0xb1>(top));  // quad_perm [1, 0, 3, 2], [2, 3, 0, 1]
}

// e = ceil(log2(top / 6)), at least -127. 6 is 1.5 2^2, e2m1's largest: the exponent field less 2, plus one
// where the mantissa is above 1.5.
HKX_DEV uint32_t mx4_block(const float (&v)[8], uint32_t top, uint32_t& codes) {
  codes = 0;
  if (top >= 0x7f800000u) return 255u;
  const uint32_t s = (uint32_t)max((int)((top + 0x3fffffu) >> 23) - 2, 0);
  const float f = __builtin_bit_cast(float, s << 23);  // (byte 0, 2^-127, too: the exponent field alone counts)
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], f, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], f, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], f, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], f, 3);
  return s;
}

// e = ceil(log2(top / 448)) of a top of 2^-126 or more, at least -127. 448 is 1.75 2^8, e4m3's largest.
HKX_DEV uint32_t mx8_block(const float (&v)[8], uint32_t top, u32x2& codes) {
  const bool bad = top >= 0x7f800000u;
  const int e = max((int)((max(top, 0x00800000u) + 0x1fffffu) >> 23) - 8, 0) - 127;
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    t[i] = bad ? 0.0f : __builtin_fminf(__builtin_fmaxf(__builtin_ldexpf(v[i], -e), -448.0f), 448.0f);
  codes = u32x2{cvt_e4m3x4(t[0], t[1], t[2], t[3]), cvt_e4m3x4(t[4], t[5], t[6], t[7])};
  return bad ? 255u : (uint32_t)(e + 127);
}

}  // namespace hkx
