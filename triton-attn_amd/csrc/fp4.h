// e2m1 codes of the 4-bit cache and their conversions, two codes an instruction: v_cvt_scalef32_pk divides (or
// multiplies) by the power of two in the scale's exponent, rounds to nearest even and saturates at 6; an exponent of 255
// makes every value NaN (checked on an MI355X: codes, scales, every 16-bit value).
#pragma once

#include "common.h"

namespace tattn {

template <typename T> struct Fp4;
template <> struct Fp4<f16> {
  static constexpr uint32_t kInf = 0x7c00, kTop = 127 + 13;  // 6 * 2^13 is finite, 4 * 2^14 is not
  static __device__ __forceinline__ uint32_t exponent(uint32_t mag) {  // fp32 bits of a magnitude
    return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(f16, (uint16_t)mag));
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t pack(uint32_t old, uint32_t two, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, two), scale, SEL);
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t unpack(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
  }
};
template <> struct Fp4<bf16> {
  static constexpr uint32_t kInf = 0x7f80, kTop = 127 + 125;
  static __device__ __forceinline__ uint32_t exponent(uint32_t mag) { return mag << 16; }
  template <int SEL>
  static __device__ __forceinline__ uint32_t pack(uint32_t old, uint32_t two, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, two), scale, SEL);
  }
  template <int SEL>
  static __device__ __forceinline__ uint32_t unpack(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  }
};

}  // namespace tattn
