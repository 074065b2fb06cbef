// Device helpers of the packed and paged attention kernels.
#pragma once

#include "common.h"

namespace moe {
namespace gqa {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#define GQA_AS_LDS __attribute__((address_space(3)))

constexpr float kLog2e = 1.4426950408889634f;
// A row's probabilities are 2^(s - m), s its scores in base 2; softmax does not depend
// on the reference m, so m may differ from the maximum, and O is rescaled only when a
// score passes limit(m).
//   bf16: m is a maximum so far and lags by at most kRescaleSlack: p <= 2^8.
//   fp16 has five bits of exponent: below 2^-14 p loses bits, below 2^-25 all of them,
// while the fp32 sum has it whole.  So m lies kF16Bias under a maximum and lags by at
// most kF16Slack, and the largest p lies in [2^11, 2^15]: those within 2^-25 of it
// are off by half a step, smaller ones by 2^-36 of it at most.  (With m at a maximum,
// what many keys add under one that has nearly all of the sum was lost: 18 below it
// in natural logarithms, most of it.)  That costs no time; 13 and 2 cost 5 to 8 % with
// heads of 64, since maxima rise by more than 2 here and there.  From 2^20 on a score is
// itself off by 2^-4 and more, and may pass m by more than limit(m) says: there m is a
// maximum, and follows every new one.
constexpr float kRescaleSlack = 8.f;
constexpr float kF16Bias = 11.f, kF16Slack = 4.f, kF16Exact = 1048576.f;
template <bool F16>
__device__ __forceinline__ float reference(float top) {
  if constexpr (F16) return top - (__builtin_fabsf(top) < kF16Exact ? kF16Bias : 0.f);
  else return top;
}
template <bool F16>
__device__ __forceinline__ float limit(float m) {
  if constexpr (F16) return m + (__builtin_fabsf(m) < kF16Exact ? kF16Bias + kF16Slack : 0.f);
  else return m + kRescaleSlack;
}
constexpr int kXcds = 8;

__device__ __forceinline__ int sgpr(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t sgpr64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return ((uint64_t)hi << 32) | lo;
}

// The two element types: F16 false is bf16, true is fp16.
template <bool F16>
__device__ __forceinline__ f32x4 mfma16x16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ f32x16 mfma32x32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}
// Two floats rounded to nearest even and packed.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    const f32x2_t v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  } else {
    return pack_bf16x2(lo, hi);
  }
}
template <bool F16>
__device__ __forceinline__ float to_f32(uint32_t bits16) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)bits16);
  else return bf16_bits_to_f32(bits16);
}

// A buffer of `bytes` bytes; loads past its end give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void *)sgpr64((uint64_t)base), (short)0, sgpr((int)bytes), 0x00020000);
}
// 16 bytes per lane straight into LDS, lane l's at dst + 16 l.  (The builtin is
// compiled in the device pass only: in the host pass a kernel that calls it
// loses its launch stub.)
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t rs, uint8_t *dst, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (GQA_AS_LDS void *)dst, 16, off, 0, 0, 0);
#endif
}
__device__ __forceinline__ uint32_t lds_addr(const uint8_t *p) {
  return (uint32_t)(uintptr_t)(const GQA_AS_LDS uint8_t *)p;
}
// Waits until at most N vector-memory operations of the wave are in flight.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}

// Over the four lanes l, l^16, l^32, l^48, in the same order on each (lane swaps
// of two copies leave every lane its own value and its partner's).
__device__ __forceinline__ float quad_max(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// An MFMA's results take up to 19 wait states, and across a branch the compiler can
// miss that they are not there yet.  Where they are read in another block than
// the MFMA's, mfma_settle() stands before, or two later MFMAs (each waits for the
// one before), and pin() keeps the reads behind that.
__device__ __forceinline__ void mfma_settle() { asm volatile("s_nop 15\n\ts_nop 3" ::: "memory"); }
__device__ __forceinline__ float pin(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

}  // namespace gqa
}  // namespace moe
