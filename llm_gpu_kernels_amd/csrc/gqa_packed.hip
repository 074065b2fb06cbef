// Causal attention of several packed prompts on gfx950.
#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_internal.h"

namespace moe {

namespace {

__device__ __forceinline__ float to_f32(uint16_t x, int dtype) {
  return dtype == GQA_FP16 ? (float)__builtin_bit_cast(_Float16, x) : bf16_bits_to_f32(x);
}
__device__ __forceinline__ uint16_t from_f32(float x, int dtype) {
  return dtype == GQA_FP16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : (uint16_t)f32_to_bf16_bits(x);
}

// One wave per token and query head, a key per lane and step.
__global__ __launch_bounds__(64) void gqa_packed_simple(GqaPackedArgs a) {
  __shared__ float qs[128], ps[64];
  const int t = blockIdx.x, head = blockIdx.y, kvh = head / (a.Hq / a.Hkv), lane = threadIdx.x;
  int s0 = -1;
  for (int s = 0; s < a.S; ++s) {
    const int b = a.starts[s], e = a.starts[s + 1];
    if ((b < 0 || e < b || e > a.N) && lane == 0) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
    if (t >= b && t < e) s0 = max(b, 0);
  }
  if (s0 < 0) return;
  for (int d = lane; d < a.D; d += 64) qs[d] = to_f32(a.q[t * a.q_stride + head * a.D + d], a.dtype);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int base = s0; base <= t; base += 64) {
    const int j = base + lane, n = min(64, t + 1 - base);
    float s = -INFINITY;
    if (lane < n) {
      const uint16_t *kp = a.k + j * a.k_stride + kvh * a.D;
      s = 0.f;
      for (int d = 0; d < a.D; ++d) s += qs[d] * to_f32(kp[d], a.dtype);
      s *= a.scale;
    }
    float mx = s;
    for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn, alpha = expf(m - ref);
    const float p = lane < n ? expf(s - ref) : 0.f;
    float sum = p;
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    __syncthreads();
    ps[lane] = p;
    __syncthreads();
    l = l * alpha + sum;
    m = mn;
    o0 *= alpha;
    o1 *= alpha;
    for (int i = 0; i < n; ++i) {
      const uint16_t *vp = a.v + (base + i) * a.v_stride + kvh * a.D;
      o0 += ps[i] * to_f32(vp[lane], a.dtype);
      if (a.D > 64) o1 += ps[i] * to_f32(vp[64 + lane], a.dtype);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t *op = a.out + ((int64_t)t * a.Hq + head) * a.D;
  op[lane] = from_f32(o0 * inv, a.dtype);
  if (a.D > 64) op[64 + lane] = from_f32(o1 * inv, a.dtype);
}

}  // namespace

hipError_t launch_gqa_packed(const GqaPackedArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(gqa_packed_simple, dim3(a.N, a.Hq), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace moe
