// Norms of queries and keys for each head and their rotation by position, in one pass,
// with the keys and values written to a cache (include/qk_mi355x.h has the formulas).
//
// Every byte is read and written once, so HBM bounds it; per element there are a few
// operations.  A workgroup has one token: its first wave computes the token's R/2 sines
// and cosines into LDS (the angle in 64 bits, in turns, so that far positions lose
// nothing, then half turns in fp32), and a head row is the work of D/8 lanes, 16 bytes
// each on either side.  Rows are independent: no barrier but the one for the angles.
#include "common.h"
#include "gqa_dev.h"
#include "mx_dev.h"
#include "qk_internal.h"
#include "../../include/kv_mi355x.h"

namespace moe {

namespace {

constexpr int kThreads = 256;

// How a lane finds the partner of an element: kHalves, R/2 dims away in whole groups of
// eight; kNeighbours, in the lane; kAny, R/2 dims away.
constexpr int kHalves = 0, kNeighbours = 1, kAny = 2;

__device__ __forceinline__ void angle(int position, float freq, float *c, float *s) {
  const double turns = (double)position * (double)freq * 0.15915494309189533577;
  sincospif(2.f * (float)(turns - rint(turns)), s, c);
}

// Sum over the D/8 lanes of a row, the same on each.
template <int D>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int o = 1; o < D / 8; o *= 2) x += __shfl_xor(x, o, kWave);
  return x;
}

// Eight values of a lane, a quarter of a block, to a cache row under the block's scale.
template <int FMT, bool F16>
__device__ __forceinline__ void put8(uint8_t *to, uint8_t *scale_to, const float (&y)[8], bool first) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = mx::larger(top, __float_as_uint(y[i]) & 0x7fffffffu);
  top = mx::larger(top, mx::neighbour(top));
  top = mx::larger(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4e, 0xf, 0xf, true));  // l ^ 2
  const int byte = mx::scale_byte<FMT, F16>(top);
  const uint32_t lo = mx::encode4<FMT>(y[0], y[1], y[2], y[3], byte), hi = mx::encode4<FMT>(y[4], y[5], y[6], y[7], byte);
  if constexpr (FMT == mx::kFp8) *(u32x2 *)to = u32x2{lo, hi};
  else *(uint32_t *)to = lo | hi << 16;
  if (first) *scale_to = (uint8_t)byte;
}

// FMT: how the cache holds its rows (0: 16 bits, or no cache).
template <int D, bool F16, int PAIRS, int FMT>
__global__ __launch_bounds__(kThreads) void qk_norm_rope(QkArgs a, int passes) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;  // lanes of a row, rows at a time
  __shared__ __attribute__((aligned(16))) float cosines[D / 2], sines[D / 2];
  __shared__ __attribute__((aligned(16))) float turned[PAIRS == kNeighbours ? 1 : kRows][D];
  const int t = blockIdx.x, c = threadIdx.x % kLanes, mine = threadIdx.x / kLanes;
  const int half = a.R / 2, rows = a.Hq + a.Hkv + (a.cached ? a.Hkv : 0);
  const int from = blockIdx.y * passes * kRows;
  int64_t slot = -1;
  if (a.cached) {
    slot = a.cache.slots[t];
    if (slot >= (int64_t)a.cache.pages * a.cache.page_size) slot = -1;
  }
  if ((int)threadIdx.x < half) angle(a.positions[t], a.inv_freq[threadIdx.x], cosines + threadIdx.x, sines + threadIdx.x);
  __syncthreads();
  for (int pass = 0; pass < passes; ++pass) {
    const int h = from + pass * kRows + mine;
    // Lanes without a row go along: rows are whole groups of lanes, and the others of a
    // wave shuffle with them.
    const bool live = h < rows, query = h < a.Hq, key = !query && h < a.Hq + a.Hkv;
    const int head = query ? h : key ? h - a.Hq : h - a.Hq - a.Hkv;
    const uint16_t *const x = (query ? a.q + t * a.q_stride : key ? a.k + t * a.k_stride : a.v + t * a.v_stride);
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (live) raw = *(const u32x4 *)(x + (int64_t)head * D + 8 * c);
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = gqa::to_f32<F16>(raw[i] & 0xffffu);
      y[2 * i + 1] = gqa::to_f32<F16>(raw[i] >> 16);
    }
    const void *const weight = query ? a.q_weight : key ? a.k_weight : nullptr;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(y[i], y[i], sum);
    sum = row_sum<D>(sum);
    if (weight) {
      const float scale = 1.0f / sqrtf(sum * (1.0f / D) + a.eps);
      float w[8];
      if (a.weights_fp32) {
        const f32x4 w0 = ((const f32x4 *)weight)[2 * c], w1 = ((const f32x4 *)weight)[2 * c + 1];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = i < 4 ? w0[i] : w1[i - 4];
      } else {
        const u32x4 wr = ((const u32x4 *)weight)[c];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = gqa::to_f32<F16>(i & 1 ? wr[i / 2] >> 16 : wr[i / 2] & 0xffffu);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * scale * w[i];
    }
    if constexpr (PAIRS == kNeighbours) {
      if (query || key) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = 4 * c + i;
          if (p >= half) continue;
          const float cs = cosines[p], sn = sines[p], l = y[2 * i], u = y[2 * i + 1];
          y[2 * i] = l * cs - u * sn;
          y[2 * i + 1] = u * cs + l * sn;
        }
      }
    } else {
      // The row's lanes are in one wave and in step: what they write they can read.
      float *const row = turned[mine];
#pragma unroll
      for (int i = 0; i < 8; ++i) row[8 * c + i] = y[i];
      __builtin_amdgcn_wave_barrier();
      if (query || key) {
        if constexpr (PAIRS == kHalves) {
          if (8 * c < a.R) {
            const bool low = 8 * c < half;
            const int p = low ? 8 * c : 8 * c - half, other = low ? 8 * c + half : p;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float cs = cosines[p + i], sn = sines[p + i], z = row[other + i];
              y[i] = low ? y[i] * cs - z * sn : y[i] * cs + z * sn;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = 8 * c + i;
            if (d >= a.R) continue;
            const bool low = d < half;
            const int p = low ? d : d - half;
            const float z = row[low ? d + half : p];
            y[i] = low ? y[i] * cosines[p] - z * sines[p] : y[i] * cosines[p] + z * sines[p];
          }
        }
      }
      __builtin_amdgcn_wave_barrier();  // read before the next pass writes
    }
    const u32x4 out = {gqa::pack2<F16>(y[0], y[1]), gqa::pack2<F16>(y[2], y[3]), gqa::pack2<F16>(y[4], y[5]),
                       gqa::pack2<F16>(y[6], y[7])};
    if (live && query) *(u32x4 *)(a.q_out + ((int64_t)t * a.Hq + head) * D + 8 * c) = out;
    if (live && key && a.k_out) *(u32x4 *)(a.k_out + ((int64_t)t * a.Hkv + head) * D + 8 * c) = out;
    if (live && !query && slot >= 0) {
      const KvState &s = a.cache;
      const int64_t at = ((int64_t)a.layer * s.pages + slot / s.page_size) * a.Hkv + head;
      const int row = (int)(slot % s.page_size);
      uint8_t *const to = (uint8_t *)(key ? s.k : s.v) + (at * s.page_size + row) * mx::row_bytes<FMT>(D) + mx::row_bytes<FMT>(8 * c);
      if constexpr (FMT == 0)
        // Values are copied: their bits stay, a NaN's too.
        *(u32x4 *)to = key ? out : raw;
      else
        put8<FMT, F16>(to, (key ? s.k_scales : s.v_scales) + (at * (D / mx::kBlock) + c / 4) * s.page_size + row, y,
                       c % 4 == 0);
    }
  }
}

template <int D, bool F16, int FMT>
hipError_t launch(const QkArgs &a, int cus, hipStream_t s) {
  constexpr int kRows = kThreads / (D / 8);
  const int rows = a.Hq + a.Hkv + (a.cached ? a.Hkv : 0), all = (rows + kRows - 1) / kRows;
  // A workgroup for every pass where those have a place on the chip at once (eight a CU),
  // else one for all of a token's, which computes its angles once.
  const int passes = (int64_t)a.N * all <= 8 * cus ? 1 : all;
  const dim3 grid(a.N, (all + passes - 1) / passes);
  if (a.interleaved) hipLaunchKernelGGL((qk_norm_rope<D, F16, kNeighbours, FMT>), grid, dim3(kThreads), 0, s, a, passes);
  else if (a.R % 16 == 0) hipLaunchKernelGGL((qk_norm_rope<D, F16, kHalves, FMT>), grid, dim3(kThreads), 0, s, a, passes);
  else hipLaunchKernelGGL((qk_norm_rope<D, F16, kAny, FMT>), grid, dim3(kThreads), 0, s, a, passes);
  return hipGetLastError();
}

template <int D, bool F16>
hipError_t launch(const QkArgs &a, int cus, hipStream_t s) {
  const int storage = a.cached ? a.cache.storage : KV_STORAGE_16BIT;
  if (storage == KV_STORAGE_MXFP8) return launch<D, F16, mx::kFp8>(a, cus, s);
  if (storage == KV_STORAGE_MXFP4) return launch<D, F16, mx::kFp4>(a, cus, s);
  return launch<D, F16, 0>(a, cus, s);
}

}  // namespace

hipError_t launch_qk_norm_rope(const QkArgs &a, int cus, hipStream_t s) {
  if (a.D == 128) return a.f16 ? launch<128, true>(a, cus, s) : launch<128, false>(a, cus, s);
  return a.f16 ? launch<64, true>(a, cus, s) : launch<64, false>(a, cus, s);
}

}  // namespace moe
