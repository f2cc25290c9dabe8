// 4-bit rows of a paged context: E2M1 codes (magnitudes 0, 1/2, 1, 3/2, 2, 3, 4, 6), two a byte,
// element 2i in the low half of byte i, and a scale 2^(x - 127) as a byte x for every 32
// elements of a row.  gfx950 converts pairs of codes in one instruction, the scale with them.
#pragma once

#include "fmlm_common.h"

namespace fmlm {

constexpr int kFp4Block = 32;

FMLM_DEV float fp4_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// codes of byte SEL of c, times the scale (its exponent field), as a pair of T
template <typename T, int SEL>
FMLM_DEV uint32_t fp4_pair(uint32_t c, float scale) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, SEL));
}
// the eight values of four bytes
template <typename T>
FMLM_DEV u32x4 fp4_oct(uint32_t c, float scale) {
  return u32x4{fp4_pair<T, 0>(c, scale), fp4_pair<T, 1>(c, scale), fp4_pair<T, 2>(c, scale), fp4_pair<T, 3>(c, scale)};
}

}  // namespace fmlm
