// Quantising a block of the microscaled formats, shared by the appends (mi_mx.hip,
// which describes it, and mi_qk_norm.hip).
#pragma once

#include "mi_common.h"

namespace mi {

template <int KVT>
constexpr int kMxMaxExp = KVT == kKvMx8 ? 119 : 125;

// The scale byte of a block whose largest magnitude has these float bits.
template <int KVT>
MI_DEVICE uint32_t mx_scale_byte(uint32_t amax) {
  constexpr uint32_t kMantissa = KVT == kKvMx8 ? 0x680000u : 0x600000u;  // of T: 1.8125, 1.75
  constexpr int kExp = KVT == kKvMx8 ? 8 : 2;                            // T's exponent
  if (amax >= 0x7f800000u) return 255u;
  if (amax == 0) return 127u;
  // a subnormal a is below every 2^-126 T: it gets the least exponent
  const int e = (int)(amax >> 23) - kExp + ((amax & 0x7fffffu) > kMantissa ? 1 : 0);  // biased by 127
  return (uint32_t)min(max(e, 1), 127 + kMxMaxExp<KVT>);
}

// Eight elements of a block's four adjacent threads -> their codes and the block's scale byte.
template <int KVT>
MI_DEVICE uint32_t mx_encode8(float (&x)[8], uint32_t (&codes)[2]) {
  typedef __attribute__((ext_vector_type(2))) short s16x2;
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, bitcast<uint32_t>(x[i]) & 0x7fffffffu);  // floats order as ints, NaN on top
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xb1, 0xf, 0xf, false));  // quad_perm [1,0,3,2]
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4e, 0xf, 0xf, false));  // quad_perm [2,3,0,1]
  const uint32_t byte = mx_scale_byte<KVT>(a);
  const float scale = bitcast<float>(byte << 23);
  codes[0] = codes[1] = 0;
  if (byte == 255) return byte;
  if constexpr (KVT == kKvMx8) {
    if (byte == 127 + kMxMaxExp<KVT>) {  // the conversion gives NaN past 464 (e2m1's gives the largest code)
      const float top = 448.f * scale;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -top), top);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s16x2 w = {0, 0};
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i], x[4 * i + 1], scale, false);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i + 2], x[4 * i + 3], scale, true);
      codes[i] = bitcast<uint32_t>(w);
    }
  } else {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    codes[0] = w;
  }
  return byte;
}

}  // namespace mi
