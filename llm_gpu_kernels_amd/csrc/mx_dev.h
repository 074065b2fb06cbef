// Microscaled elements: 32 neighbouring values of a row share a power of two.
//
//   value = element * 2^(scale - 127), elements e4m3 (8 bits) or e2m1 (4 bits, two in
//   a byte, the earlier in the low half), scale 8 bits; scale 255: all 32 are NaN.
//
// The scale is the smallest with which the largest of the 32 magnitudes is in the
// elements' range, so that no element saturates and each is off by half of its own
// step at most.  It ends where the largest element times it is the largest such
// product that is finite in the tokens' type (larger magnitudes saturate there), and
// at 2^-117, from where on every product is a normal bf16 number.  A block that holds
// an infinity or a NaN reads back as NaN.
//
// gfx950 converts both ways in single instructions, to nearest even; its decoders
// apply the scale exactly where the 16-bit type holds the product, which has 4 or 2 bits.
// It does for all that is made of bf16 tokens, and of fp16 ones: those are multiples of 2^-24,
// and so is one that is rounded to 4 or 2 bits or to an element's step above 2^-24.  Keys that
// are quantised from fp32 under scales below 2^-15 (fp8) or 2^-23 (fp4) may lie between
// fp16's smallest numbers: decoded to nearest even, off by 2^-25 (every element under every
// scale is tested).
#pragma once

#include "common.h"
#include "gqa_dev.h"

namespace moe {
namespace mx {

constexpr int kFp8 = 1, kFp4 = 2;  // KV_STORAGE_*
constexpr int kBlock = 32;         // values with one scale
constexpr int kFirstScale = 10;    // 2^-117
template <int FMT, bool F16>
constexpr int kLastScale = FMT == kFp8 ? (F16 ? 127 + 7 : 127 + 119) : (F16 ? 127 + 13 : 127 + 125);
template <int FMT>
__host__ __device__ constexpr int row_bytes(int d) { return FMT == 0 ? 2 * d : FMT == kFp8 ? d : d / 2; }

// The scale byte of a block whose largest magnitude has the fp32 bits `top`.
template <int FMT, bool F16>
__device__ __forceinline__ int scale_byte(uint32_t top) {
  const int e = (int)(top >> 23);
  if (e == 255) return 255;
  // 448 = 1.75 * 2^8, 6 = 1.5 * 2^2.
  const int over = (top & 0x7fffffu) > (FMT == kFp8 ? 0x600000u : 0x400000u);
  return min(max(e - (FMT == kFp8 ? 8 : 2) + over, kFirstScale), kLastScale<FMT, F16>);
}
// Larger of two magnitudes by their bits (NaN largest).
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
// The value of the lane next to this one (l ^ 1).
__device__ __forceinline__ uint32_t neighbour(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true);  // quad_perm 1 0 3 2
}

// Four fp32 values to elements under a scale byte: fp8 in four bytes, fp4 in the low two.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, int byte) {
#if defined(__HIP_DEVICE_COMPILE__)
  if (byte == 255) return 0u;
  const float inv = __uint_as_float((uint32_t)(254 - byte) << 23), most = FMT == kFp8 ? 448.f : 6.f;
  a = __builtin_amdgcn_fmed3f(a * inv, -most, most);
  b = __builtin_amdgcn_fmed3f(b * inv, -most, most);
  c = __builtin_amdgcn_fmed3f(c * inv, -most, most);
  d = __builtin_amdgcn_fmed3f(d * inv, -most, most);
  if constexpr (FMT == kFp8) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
  } else {
    const uint32_t lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, 1.0f, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, c, d, 1.0f, 1) & 0xffffu;
  }
#else
  return 0u;
#endif
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two neighbouring elements of a word, scaled, as two 16-bit numbers: fp8 half PART (0,
// 1) of the word, fp4 byte PART (0 to 3).
template <int FMT, bool F16, int PART>
__device__ __forceinline__ uint32_t decode2(uint32_t w, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (FMT == kFp8) {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, PART));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, PART));
  } else {
    if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, PART));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, PART));
  }
#else
  return w;
#endif
}
// Eight neighbouring elements: fp8 in two words, fp4 in the first.
template <int FMT, bool F16>
__device__ __forceinline__ u32x4 decode8(uint32_t w0, uint32_t w1, float scale) {
  if constexpr (FMT == kFp8)
    return u32x4{decode2<FMT, F16, 0>(w0, scale), decode2<FMT, F16, 1>(w0, scale), decode2<FMT, F16, 0>(w1, scale),
                 decode2<FMT, F16, 1>(w1, scale)};
  else
    return u32x4{decode2<FMT, F16, 0>(w0, scale), decode2<FMT, F16, 1>(w0, scale), decode2<FMT, F16, 2>(w0, scale),
                 decode2<FMT, F16, 3>(w0, scale)};
}

}  // namespace mx
}  // namespace moe
