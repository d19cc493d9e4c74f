// The number formats of a quantised cache and their conversions (gfx950).
//
// 32 neighbouring elements of a head share a scale 2^(byte - 127).  Elements: e4m3 (one byte, largest
// 448) or e2m1 (half a byte, the first of two in the low half, largest 6).  Scales are powers of two
// so that an element times its scale is exact in bf16 (4 bits of significand) and the conversions
// are one instruction for two elements, scale included; a scale that is not costs e4m3, a floating
// format itself, nothing.  Byte 255: a group that held an infinity or NaN; its elements are NaN.
#pragma once

#include "dsp_common.h"

namespace dsp_quant {

enum Format { kNone = 0, kFp8 = DSP_KV_FP8, kFp4 = DSP_KV_FP4 };
constexpr int kGroup = 32;
constexpr int kMinExp = -100, kMaxExp = 118;  // of a scale: products neither vanish nor overflow bf16
constexpr uint32_t kNanScale = 255;

// Bytes of n elements.
template <int kFmt>
constexpr int bytes(int n) {
  return kFmt == kFp8 ? n : n / 2;
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two elements of a word as a pair of 16-bit numbers (kF16: fp16, rounded to nearest, infinite past
// its range; else bf16, exact), element 2 * kPair first.  A scale of byte 255 gives NaN.
template <int kFmt, bool kF16, int kPair>
__device__ __forceinline__ uint32_t widen2(uint32_t word, float scale) {
  if constexpr (kFmt == kFp8) {
    if constexpr (kF16)
      return __builtin_bit_cast(uint32_t,
                                __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, kPair != 0));
    else
      return __builtin_bit_cast(uint32_t,
                                __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, kPair != 0));
  } else {
    if constexpr (kF16)
      return __builtin_bit_cast(uint32_t,
                                __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, kPair));
    else
      return __builtin_bit_cast(uint32_t,
                                __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, kPair));
  }
}

// kN elements from the words at w as kN / 2 words of pairs.
template <int kFmt, bool kF16, int kN>
__device__ __forceinline__ void widen(const uint32_t* w, float scale, uint32_t* out) {
  if constexpr (kFmt == kFp8) {
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      out[2 * i] = widen2<kFmt, kF16, 0>(w[i], scale);
      out[2 * i + 1] = widen2<kFmt, kF16, 1>(w[i], scale);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN / 8; ++i) {
      out[4 * i] = widen2<kFmt, kF16, 0>(w[i], scale);
      out[4 * i + 1] = widen2<kFmt, kF16, 1>(w[i], scale);
      out[4 * i + 2] = widen2<kFmt, kF16, 2>(w[i], scale);
      out[4 * i + 3] = widen2<kFmt, kF16, 3>(w[i], scale);
    }
  }
}

}  // namespace dsp_quant
