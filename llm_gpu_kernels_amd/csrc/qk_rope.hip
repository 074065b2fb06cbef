// Norms of queries and keys for each head and their rotation by position, in one pass,
// with the keys and values written to a cache (include/qk_mi355x.h has the formulas).
//
// Every byte is read and written once, so HBM bounds it; per element there are a few
// operations.  A wave has one token, or some of its heads: each lane computes one of the
// R/2 angles (in 64 bits, in turns, so that far positions lose nothing, then half turns
// in fp32), and takes from LDS the cosines and sines that its eight elements of every row
// meet.  A row is the work of D/8 lanes, 16 bytes each on either side; the sum of squares and
// the elements R/2 further come by lane exchanges within vector instructions.  No
// workgroup's waves wait for each other.
//
// Measured, a copy of 2 GiB running at 5.1 TB/s: 8191 tokens of 32 + 8 heads of 128 (168 MB)
// 33.8 us, 5.0 TB/s (a workgroup per token, its rows in LDS: 51; arguments, positions and weights
// loaded where they are used: 38.8); 2500 of 12 + 4 heads of 64 with their cache in eight bits
// 7.3; 16 tokens 3.6, the launch, a load and a chain of some hundred instructions.
#include "common.h"
#include "gqa_dev.h"
#include "mx_dev.h"
#include "qk_internal.h"
#include "../../include/kv_mi355x.h"

namespace moe {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;

// How a lane finds the partners of its elements: kNeighbours, in the lane; 1, 2, 4 or 8, so
// many lanes on (R/2 = 8 times that); kAny, R/2 elements on, through LDS.
constexpr int kNeighbours = 0, kAny = 16;

__device__ __forceinline__ void angle(int position, float freq, float *c, float *s) {
  const double turns = (double)position * (double)freq * 0.15915494309189533577;
  sincospif(2.f * (float)(turns - rint(turns)), s, c);
}

template <int CTRL, int BANKS = 0xf>
__device__ __forceinline__ float dpp(float old, float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), CTRL, 0xf, BANKS, false));
}
// The value of lane l ^ N of a row of sixteen lanes.
template <int N>
__device__ __forceinline__ float partner(float x) {
  if constexpr (N == 1) return dpp<0xb1>(x, x);        // quad_perm 1 0 3 2
  else if constexpr (N == 2) return dpp<0x4e>(x, x);   // quad_perm 2 3 0 1
  else if constexpr (N == 4) return dpp<0x114, 0xa>(dpp<0x104, 0x5>(x, x), x);  // row_shl:4, row_shr:4
  else return dpp<0x128>(x, x);                        // row_ror:8
}
// Sum over the D/8 lanes of a row, in the same order on each.
template <int D>
__device__ __forceinline__ float row_sum(float x) {
  if constexpr (D == 128) x += dpp<0x140>(x, x);  // row_mirror: lane 15 - l
  x += dpp<0x141>(x, x);                          // row_half_mirror: 7 - l
  x += partner<1>(x);
  return x + partner<2>(x);
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

// FMT: how the cache holds its rows (0: 16 bits, or no cache).  A token's rows of kRows heads
// are `passes` of them; `parts` waves have a token, `each` passes of them one.
template <int D, bool F16, int PAIRS, int FMT>
__global__ __launch_bounds__(kThreads) void qk_norm_rope(QkArgs a, int parts, int each) {
  constexpr int kLanes = D / 8, kRows = kWave / kLanes;  // lanes of a row, rows at a time
  __shared__ __attribute__((aligned(16))) float turn[kWaves][2][kWave];
  __shared__ __attribute__((aligned(16))) float lds_rows[kWaves][PAIRS == kAny ? kRows : 1][PAIRS == kAny ? D : 4];
  // The arguments at once, not line by line where they are used: a token takes no longer than that.
  asm volatile("" ::"s"(a.N), "s"(a.Hkv), "s"(a.R), "s"(a.weights_fp32), "s"(a.q), "s"(a.k), "s"(a.v), "s"(a.positions),
               "s"(a.inv_freq), "s"(a.q_weight), "s"(a.k_weight), "s"(a.q_out), "s"(a.k_out), "s"(a.q_stride), "s"(a.k_stride),
               "s"(a.v_stride), "s"(a.eps), "s"(a.cache.slots), "s"(parts), "s"(each));
  const int lane = threadIdx.x & 63, wave = gqa::sgpr(threadIdx.x >> 6), c = lane % kLanes, nth = lane / kLanes;
  const uint32_t unit = blockIdx.x * kWaves + wave;  // below 2^27
  const int t = gqa::sgpr((int)(unit / (uint32_t)parts)), part = gqa::sgpr((int)(unit - (uint32_t)(t * parts)));
  if (t >= a.N) return;
  const int half = a.R / 2, rows = a.Hq + a.Hkv + (a.cached ? a.Hkv : 0);
  const int from = part * each * kRows, to = min(rows, from + each * kRows);
  const uint16_t *const qp = a.q + t * a.q_stride, *const kp = a.k + t * a.k_stride, *const vp = a.v + t * a.v_stride;
  // The lane's elements of the row h, which is a query's, a key's or a value's.
  auto load = [&](int h) __attribute__((always_inline)) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (h < to) {
      const uint16_t *const p = h < a.Hq ? qp + (int64_t)h * D : h < a.Hq + a.Hkv ? kp + (int64_t)(h - a.Hq) * D
                                                                                : vp + (int64_t)(h - a.Hq - a.Hkv) * D;
      x = *(const u32x4 *)(p + 8 * c);
    }
    return x;
  };
  // Everything that is needed before the first row is loaded before the first wait.
  const int position = a.positions[t];
  const float freq = a.inv_freq[min(lane, half - 1)];
  u32x4 next = load(from + nth);
  u32x4 raw_q[2] = {}, raw_k[2] = {};
  auto fetch = [&](const void *w, u32x4 (&x)[2]) __attribute__((always_inline)) {
    if (!w) return;
    x[0] = ((const u32x4 *)w)[a.weights_fp32 ? 2 * c : c];
    if (a.weights_fp32) x[1] = ((const u32x4 *)w)[2 * c + 1];
  };
  fetch(a.q_weight, raw_q);
  fetch(a.k_weight, raw_k);
  // The token's page and row there; -1: none.  (A cache has at most 2^30 places.)
  int page = -1, page_row = 0;
  if (a.cached) {
    const int64_t slot = a.cache.slots[t];
    const bool in = slot >= 0 && slot < (int64_t)a.cache.pages * a.cache.page_size;
    const int place = gqa::sgpr(in ? (int)slot : -1);
    page = place < 0 ? -1 : place / a.cache.page_size;
    page_row = place - page * a.cache.page_size;
  }
  float wq[8], wk[8];
  if (lane < half) angle(position, freq, &turn[wave][0][lane], &turn[wave][1][lane]);
  auto weights = [&](const u32x4 (&r)[2], float (&x)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = a.weights_fp32 ? __uint_as_float(r[i / 4][i % 4]) : gqa::to_f32<F16>(i & 1 ? r[0][i / 2] >> 16 : r[0][i / 2] & 0xffffu);
  };
  weights(raw_q, wq);
  weights(raw_k, wk);
  __builtin_amdgcn_wave_barrier();  // a wave's LDS operations are in order
  // Of element 8 c + i: the cosine, the sine with its sign, and where its partner lies.
  // Neighbours: of the pair 4 c + i.
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < (PAIRS == kNeighbours ? 4 : 8); ++i) {
    const int d = 8 * c + i, p = PAIRS == kNeighbours ? 4 * c + i : d < half ? d : d - half;
    cs[i] = turn[wave][0][min(p, half - 1)];
    sn[i] = turn[wave][1][min(p, half - 1)];
    if (PAIRS != kNeighbours && d < half) sn[i] = -sn[i];
  }
  for (int h0 = from; h0 < to; h0 += kRows) {
    const int h = h0 + nth;
    const u32x4 raw = next;
    next = load(h + kRows);
    // Lanes without a row go along: the others of the wave exchange with them.
    const bool live = h < to, query = h < a.Hq, key = !query && h < a.Hq + a.Hkv;
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = gqa::to_f32<F16>(raw[i] & 0xffffu);
      y[2 * i + 1] = gqa::to_f32<F16>(raw[i] >> 16);
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(y[i], y[i], sum);
    sum = row_sum<D>(sum);
    if (query ? a.q_weight != nullptr : key && a.k_weight != nullptr) {
      const float scale = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * scale * (query ? wq[i] : wk[i]);
    }
    if constexpr (PAIRS == kNeighbours) {
      if (query || key) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float l = y[2 * i], u = y[2 * i + 1];
          const bool turns = 4 * c + i < half;
          y[2 * i] = turns ? l * cs[i] - u * sn[i] : l;
          y[2 * i + 1] = turns ? u * cs[i] + l * sn[i] : u;
        }
      }
    } else if constexpr (PAIRS == kAny) {
      float *const row = lds_rows[wave][nth];
#pragma unroll
      for (int i = 0; i < 8; ++i) row[8 * c + i] = y[i];
      __builtin_amdgcn_wave_barrier();
      if (query || key) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = 8 * c + i;
          if (d < a.R) y[i] = y[i] * cs[i] + row[d < half ? d + half : d - half] * sn[i];
        }
      }
      __builtin_amdgcn_wave_barrier();  // read before the next rows are written
    } else {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = partner<PAIRS>(y[i]);
      if ((query || key) && c < 2 * PAIRS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * cs[i] + z[i] * sn[i];
      }
    }
    const u32x4 out = {gqa::pack2<F16>(y[0], y[1]), gqa::pack2<F16>(y[2], y[3]), gqa::pack2<F16>(y[4], y[5]),
                       gqa::pack2<F16>(y[6], y[7])};
    if (live && query) *(u32x4 *)(a.q_out + ((int64_t)t * a.Hq + h) * D + 8 * c) = out;
    if (live && key && a.k_out) *(u32x4 *)(a.k_out + ((int64_t)t * a.Hkv + h - a.Hq) * D + 8 * c) = out;
    if (live && !query && page >= 0) {
      const KvState &s = a.cache;
      const int64_t at = ((int64_t)a.layer * s.pages + page) * a.Hkv + (key ? h - a.Hq : h - a.Hq - a.Hkv);
      uint8_t *const to_row = (uint8_t *)(key ? s.k : s.v) + (at * s.page_size + page_row) * mx::row_bytes<FMT>(D) + mx::row_bytes<FMT>(8 * c);
      if constexpr (FMT == 0)
        // Values are copied: their bits stay, a NaN's too.
        *(u32x4 *)to_row = key ? out : raw;
      else
        put8<FMT, F16>(to_row, (key ? s.k_scales : s.v_scales) + (at * (D / mx::kBlock) + c / 4) * s.page_size + page_row, y,
                       c % 4 == 0);
    }
  }
}

template <int D, bool F16, int FMT>
hipError_t launch(const QkArgs &a, int cus, hipStream_t s) {
  constexpr int kRows = kWave / (D / 8);
  const int rows = a.Hq + a.Hkv + (a.cached ? a.Hkv : 0), passes = (rows + kRows - 1) / kRows;
  // A token's passes are shared out over waves, each of which computes its angles: over as many
  // as 20 waves a CU allow (24 to 32 run at once, by the variant's registers; 1000 tokens of 32 + 8
  // heads of 128: 6.4 us, 7.5 with twice as many, 6.8 with 12 a CU), and where those are fewer, five
  // passes to a wave by itself, thirteen to two, 21 to three (from 2700 tokens on the best of one to
  // five waves a token, or mostly within 5 % of that).  In one wave, in two and in three, 3000 tokens:
  // 10 passes (32 + 8 of 128) 12.4, 11.4, 12.2 us, 12 (the same into eight bits) 15.6, 14.5, 15.6, 3 (12 + 4
  // of 64 into eight bits) 6.5, 7.0, 7.5; 6000: 27.2, 25.8, 25.3 and 31.0, 29.5, 30.0 and 9.6, 10.6, 11.7.
  // 7000 of 64 + 8, 18 passes, in one to five: 63.1, 53.6, 49.8, 49.3, 47.7; of 24 + 8, 8 passes, 27.1,
  // 24.0, 24.3; of 16 + 8, 6 passes, 19.1, 17.9; of 16 + 4, 5 passes, 13.6, 13.9, 15.3.
  const int64_t places = 20 * (int64_t)cus;
  // (Fewer than 2^26 waves in all: a grid has fewer than 2^32 threads, and N goes up to 2^24.)
  const int least = min(1 + (passes + 2) / 8, (1 << 25) / a.N), most = max(least, (int)(places / a.N));
  const int each = (passes + most - 1) / most;
  const int parts = (passes + each - 1) / each;
  const uint32_t grid = (uint32_t)(((int64_t)a.N * parts + kWaves - 1) / kWaves);
  auto go = [&](auto *kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, s, a, parts, each); };
  const int lanes = a.R / 16;
  if (a.interleaved) go(qk_norm_rope<D, F16, kNeighbours, FMT>);
  else if (a.R % 16 || (lanes & (lanes - 1))) go(qk_norm_rope<D, F16, kAny, FMT>);
  else if (lanes == 1) go(qk_norm_rope<D, F16, 1, FMT>);
  else if (lanes == 2) go(qk_norm_rope<D, F16, 2, FMT>);
  else if (lanes == 4) go(qk_norm_rope<D, F16, 4, FMT>);
  else go(qk_norm_rope<D, F16, D == 128 ? 8 : 4, FMT>);
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
