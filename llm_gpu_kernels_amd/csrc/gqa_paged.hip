// Attention of one new token per sequence over a paged cache on gfx950.
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

// One wave per sequence and query head, a key per lane and step.
__global__ __launch_bounds__(64) void gqa_paged_simple(GqaPagedArgs a) {
  __shared__ float qs[128], ps[64];
  __shared__ int64_t rows[64];
  const int b = blockIdx.x, head = blockIdx.y, kvh = head / (a.Hq / a.Hkv), lane = threadIdx.x;
  int len = a.lengths[b];
  if (len < 0 || len > a.M * a.page) {
    if (lane == 0) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
    len = max(0, min(len, a.M * a.page));
  }
  for (int d = lane; d < a.D; d += 64) qs[d] = to_f32(a.q[b * a.q_stride + head * a.D + d], a.dtype);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int base = 0; base < len; base += 64) {
    const int j = base + lane, n = min(64, len - base);
    float s = -INFINITY;
    int64_t vrow = -1;
    if (lane < n) {
      const int p = a.tables[b * a.table_stride + j / a.page], r = j % a.page;
      if (p < 0 || p >= a.P) {
        atomicOr(a.status, GQA_STATUS_BAD_PAGE);
      } else {
        const uint16_t *kp = a.k + p * a.k_page + kvh * a.k_head + r * a.k_row;
        vrow = p * a.v_page + kvh * a.v_head + r * a.v_row;
        s = 0.f;
        for (int d = 0; d < a.D; ++d) s += qs[d] * to_f32(kp[d], a.dtype);
        s *= a.scale;
      }
    }
    float mx = s;
    for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn, alpha = expf(m - ref);
    const float p = vrow >= 0 ? expf(s - ref) : 0.f;
    float sum = p;
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    __syncthreads();
    ps[lane] = p;
    rows[lane] = vrow;
    __syncthreads();
    l = l * alpha + sum;
    m = mn;
    o0 *= alpha;
    o1 *= alpha;
    for (int i = 0; i < n; ++i) {
      if (rows[i] < 0) continue;
      const uint16_t *vp = a.v + rows[i];
      o0 += ps[i] * to_f32(vp[lane], a.dtype);
      if (a.D > 64) o1 += ps[i] * to_f32(vp[64 + lane], a.dtype);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t *op = a.out + ((int64_t)b * a.Hq + head) * a.D;
  op[lane] = from_f32(o0 * inv, a.dtype);
  if (a.D > 64) op[64 + lane] = from_f32(o1 * inv, a.dtype);
}

__global__ void clear_word(uint32_t *w) { *w = 0; }

}  // namespace

hipError_t launch_gqa_paged(const GqaPagedArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(gqa_paged_simple, dim3(a.B, a.Hq), dim3(64), 0, s, a);
  return hipGetLastError();
}

hipError_t read_and_clear_status(uint32_t *status, uint32_t *flags, hipStream_t s) {
  hipError_t e = hipStreamSynchronize(s);
  if (e == hipSuccess) e = hipMemcpy(flags, status, sizeof(uint32_t), hipMemcpyDeviceToHost);
  if (e == hipSuccess && *flags) {
    hipLaunchKernelGGL(clear_word, dim3(1), dim3(1), 0, s, status);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace moe
