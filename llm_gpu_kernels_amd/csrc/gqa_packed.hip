// Causal attention of several packed prompts on gfx950.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j - max),
//   over the keys j of t's sequence up to t; head h reads KV head h / G.
//
// Long prompts are bound by the matrix cores, and next to them by the LDS: an
// MFMA operand read is used for as many query rows as the wave holds.  So a
// workgroup owns 256 query rows of one KV head (a sequence's tokens with their G
// heads side by side, row = token * G + head, whatever G is) and each of its
// four waves, one per SIMD, owns 64: two blocks of 32 that share every K and V
// operand.  With one wave per SIMD nothing else fills its pauses, so the wave
// overlaps its own work: per 32 keys
//   A: S^T = K Q^T of the next 32 keys (MFMA) beside the exponentials of these,
//   B: O^T += V^T P^T of these (MFMA) beside the sums and the next maxima,
// with the operands of each read from LDS one phase ahead.  A lane holds sixteen
// scores of one query per block (the partner lane l ^ 32 the other sixteen), so
// the online softmax is lane-local and P is the B operand of O^T as it lies.
//
// K and V come in stages of 64 keys, global -> LDS in whole rows (buffer loads
// with an LDS destination; keys behind the sequence's end read as zeros), three
// stages ahead in a ring of four, with one barrier per stage.
#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"

namespace moe {

using namespace gqa;

namespace {

constexpr int kTileRows = 256;  // query rows of a workgroup
constexpr int kWaves = 4;
constexpr int kStageKeys = 64;
constexpr int kSlots = 4;
constexpr int kWindow = 4;      // sequences per lane that a search looks at together
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Row i of a stage's K (V) tile holds its 16-byte chunk c at place c ^ swizzle(i):
// sixteen lanes that read one chunk of sixteen K rows, or two chunks of four V
// rows, then meet different bank groups.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swizzle_v(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

// 16 bytes per lane from a buffer straight into LDS at `dst` + 16 l.  As inline
// assembly (it has no output register): the compiler would make every later LDS
// read wait for all such loads in flight; the kernel waits with exact counts.
// (Nothing else in this kernel uses m0.)
__device__ __forceinline__ void load_lds(u32x4 rsrc, uint32_t dst, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(dst), "v"(off), "s"(rsrc)
               : "memory");
}
__device__ __forceinline__ u32x4 buffer_words(const void *base, uint32_t bytes) {
  const uint64_t b = sgpr64((uint64_t)base);
  return u32x4{(uint32_t)b, (uint32_t)(b >> 32) & 0xffffu, (uint32_t)sgpr((int)bytes), 0x00020000u};
}
__device__ __forceinline__ u32x4 lds_b128(uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
  return *(const GQA_AS_LDS u32x4 *)at;
#else
  return u32x4{at, 0u, 0u, 0u};
#endif
}
// Within each group of 16 lanes, lane 4a + b receives element b of the 8-byte
// rows addressed by lanes a, a + 4, a + 8, a + 12.
__device__ __forceinline__ u32x2 lds_tr16(uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((GQA_AS_LDS i16x4 *)at));
#else
  return u32x2{at, 0u};
#endif
}
// The value of this lane and of lane l ^ 32, in the same order on both.
__device__ __forceinline__ f32x2_t halves(float x) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f32x2_t{__uint_as_float(h[0]), __uint_as_float(h[1])};
}
// MFMA results stay in AGPRs and are read and written by these.  As plain
// arithmetic, the rare rescale of O would make the compiler move all of O to VGPRs
// and back at every step; and across a branch it can miss that an MFMA's result is
// not there yet (it takes up to 19 wait states for 16 passes).  Before the first
// read: acc_settle(), or two later MFMAs (each waits for the one before).
__device__ __forceinline__ float acc_read(float x) {
  float t;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(t) : "a"(x));
  return t;
}
__device__ __forceinline__ float acc_write(float t) {
  float x;
  asm volatile("v_accvgpr_write_b32 %0, %1" : "=a"(x) : "v"(t));
  return x;
}
__device__ __forceinline__ void acc_settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
template <bool F16>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

template <bool F16>
__device__ __forceinline__ float element(u32x4 x, int i) {
  return to_f32<F16>(i & 1 ? x[i / 2] >> 16 : x[i / 2] & 0xffffu);
}

// A workgroup's rows: tile `tile` (kTileRows query rows) of the sequence that
// starts at token `start` and has `len`.
struct Rows {
  int start, len, tile;
};

// The item-th tile of all sequences.  Up to 64 kWindow sequences: in descending
// number of 64-key stages (the longest start first), found by bisection over
// that number, with every wave counting for itself: a sequence of n tokens has
// T = ceil(n G / 256) tiles, tile t sees min(n, (256 t + 255) / G + 1) keys, so
// T - min(T, G s / 4) of them have more than s stages.  More sequences: in
// order, since no one tile weighs much there.  len 0: no such tile.
__device__ __forceinline__ Rows find_rows(const GqaPackedArgs &a, int G, int item) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.S; base += kWave * kWindow) {
    int b[kWindow], n[kWindow];
#pragma unroll
    for (int i = 0; i < kWindow; ++i) {
      const int s = base + kWave * i + lane;
      const int lo = s < a.S ? a.starts[s] : 0, hi = s < a.S ? a.starts[s + 1] : 0;
      b[i] = max(0, min(lo, a.N));
      n[i] = max(0, min(hi, a.N) - b[i]);
      if (lo < 0 || hi < lo || hi > a.N) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
    }
    auto tiles = [&](int i) { return (n[i] * G + kTileRows - 1) / kTileRows; };
    auto longer = [&](int i, int s) {
      const int T = tiles(i);
      return n[i] > kStageKeys * s ? T - min(T, G * s / 4) : 0;
    };
    static_assert(kTileRows == 4 * kStageKeys, "G s / 4 above");
    auto count = [&](int s) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kWindow; ++i) c += longer(i, s);
      return sgpr(wave_sum_i(c));
    };
    const bool sorted = a.S <= kWave * kWindow;
    const int total = count(0);
    if (item >= total) {
      if (sorted) break;
      item -= total;
      continue;
    }
    int above = 0, stages = 0;  // tiles with more stages; stages of this one (0: in order)
    if (sorted && a.S > 1) {
      int lo = 1, hi = (a.N + kStageKeys - 1) / kStageKeys;  // count(hi) is 0
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (count(mid) <= item) hi = mid;
        else lo = mid + 1;
      }
      stages = lo;
      above = count(lo);
    }
    // The (item - above)-th of the tiles of that class, in order.
    int left = item - above;
#pragma unroll
    for (int i = 0; i < kWindow; ++i) {
      const int rest = stages ? longer(i, stages) : 0, c = (stages ? longer(i, stages - 1) : tiles(i)) - rest;
      int incl = c;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(incl, o, kWave);
        if (lane >= o) incl += y;
      }
      const int here = __builtin_amdgcn_readlane(incl, 63);
      if (left < here) {
        const int at = sgpr(__builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > left)));
        const int nth = left - (__builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(c, at));
        const int T = __builtin_amdgcn_readlane(tiles(i), at) - __builtin_amdgcn_readlane(rest, at);
        return Rows{__builtin_amdgcn_readlane(b[i], at), __builtin_amdgcn_readlane(n[i], at), T - 1 - nth};
      }
      left -= here;
    }
    break;
  }
  return Rows{0, 0, 0};
}

// The 64 rows of a wave from row0 on, a row per lane and a key per step, in plain
// fp32: for waves that meet a V that only some of their rows see and that is not
// finite.  A key that a row does not see touches nothing of it.
template <int D, bool F16>
__device__ __forceinline__ void take_rows(const GqaPackedArgs &a, const Rows &w, int kvh, int row0, int tok_hi) {
  const int G = a.Hq / a.Hkv, rows = w.len * G;
  const int row = min(row0 + (int)(threadIdx.x & 63), rows - 1), tok = row / G, head = kvh * G + row % G;
  const uint16_t *const qp = a.q + (int64_t)(w.start + tok) * a.q_stride + (int64_t)head * D;
  u32x4 q[D / 8];
#pragma unroll
  for (int c = 0; c < D / 8; ++c) q[c] = *(const u32x4 *)(qp + 8 * c);
  float o[D], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < D; ++d) o[d] = 0.f;
  const float sl2 = a.scale * kLog2e;
#pragma clang loop unroll(disable)
  for (int key = 0; key <= tok_hi; ++key) {
    const uint16_t *const kp = a.k + (int64_t)(w.start + key) * a.k_stride + (int64_t)kvh * D;
    const uint16_t *const vp = a.v + (int64_t)(w.start + key) * a.v_stride + (int64_t)kvh * D;
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const u32x4 x = *(const u32x4 *)(kp + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        dot = __builtin_fmaf(element<F16>(q[c], i), element<F16>(x, i), dot);
    }
    const bool seen = key <= tok;
    const float sc = seen ? dot * sl2 : -INFINITY, m_new = fmaxf(m, sc), ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - ref), p = seen ? exp2f(sc - ref) : 0.f;
    m = m_new;
    l = l * alpha + p;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const u32x4 x = *(const u32x4 *)(vp + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __builtin_fmaf(p, element<F16>(x, i), o[8 * c + i] * alpha);
        o[8 * c + i] = seen ? y : o[8 * c + i];
      }
    }
  }
  if (row0 + (int)(threadIdx.x & 63) >= rows) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint32_t *const op = (uint32_t *)(a.out + ((int64_t)(w.start + tok) * a.Hq + head) * D);
#pragma unroll
  for (int d = 0; d < D; d += 2) op[d / 2] = pack2<F16>(o[d] * inv, o[d + 1] * inv);
}

template <int D, bool F16>
__global__ __launch_bounds__(64 * kWaves, 1) void gqa_packed_kernel(GqaPackedArgs a) {
  constexpr int kSteps = D / 16;                    // QK MFMAs per block and half stage
  constexpr int kDims = D / 32;                     // 32-dim tiles of O
  constexpr int kTile = kStageKeys * D * 2;         // bytes of a stage's K (or V)
  constexpr int kLoads = kTile / 1024 / kWaves;     // of K (or V) per wave and stage
  constexpr int kChunks = D / 8;                    // 16-byte chunks of a row
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = sgpr(threadIdx.x >> 6);
  const int G = a.Hq / a.Hkv;

  // Workgroups go round the eight XCDs; the tiles of one KV head stay on the
  // XCDs of its class, which share K and V through their L2.
  const int xcd = blockIdx.x % kXcds, slot8 = blockIdx.x / kXcds;
  const int classes = a.Hkv % 8 == 0 ? 8 : a.Hkv % 4 == 0 ? 4 : a.Hkv % 2 == 0 ? 2 : 1;
  const int in_class = slot8 * (kXcds / classes) + xcd / classes, per_class = a.Hkv / classes;
  const int kvh = sgpr(xcd % classes + classes * (in_class % per_class));
  const Rows w = find_rows(a, G, sgpr(in_class / per_class));
  if (w.len == 0) return;

  const int rows = w.len * G;                                           // of the sequence
  const int row0 = w.tile * kTileRows + 64 * wave;                      // of the wave
  const int keys = min(w.len, (w.tile * kTileRows + kTileRows - 1) / G + 1);  // that the workgroup sees
  const int stages = (keys + kStageKeys - 1) / kStageKeys;
  // The wave's half stages of 32 keys: all up to its last token's, the first
  // `full` of them seen by all of its tokens.
  const int tok_lo = row0 / G, tok_hi = min(w.len - 1, (row0 + 63) / G);
  const int nhalf = row0 < rows ? tok_hi / 32 + 1 : 0, full = (tok_lo + 1) / 32;

  // ---- loads ----
  const uint32_t lds0 = lds_addr(smem);
  const uint32_t ksb = (uint32_t)(2 * a.k_stride), vsb = (uint32_t)(2 * a.v_stride);
  const uint16_t *const k0 = a.k + (int64_t)w.start * a.k_stride + (int64_t)kvh * D;
  const uint16_t *const v0 = a.v + (int64_t)w.start * a.v_stride + (int64_t)kvh * D;
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int row = (64 * (wave * kLoads + j) + lane) / kChunks, place = lane % kChunks;
    k_off[j] = (uint32_t)row * ksb + 16 * (place ^ swizzle_k<D>(row));
    v_off[j] = (uint32_t)row * vsb + 16 * (place ^ swizzle_v<D>(row));
  }
  auto issue = [&](int st) __attribute__((always_inline)) {
    const int first = st * kStageKeys, n = min(kStageKeys, w.len - first);
    const u32x4 krs = buffer_words(k0 + (int64_t)first * a.k_stride, (uint32_t)(n - 1) * ksb + 2 * D);
    const u32x4 vrs = buffer_words(v0 + (int64_t)first * a.v_stride, (uint32_t)(n - 1) * vsb + 2 * D);
    const uint32_t dst = sgpr((int)(lds0 + (st % kSlots) * (2 * kTile) + wave * kLoads * 1024));
#pragma unroll
    for (int j = 0; j < kLoads; ++j) load_lds(krs, dst + j * 1024, k_off[j]);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) load_lds(vrs, dst + kTile + j * 1024, v_off[j]);
  };
  // Stage st is there for every wave, and every wave is done with stage st - 2,
  // whose slot takes stage st + 2.
  auto sync = [&](int st) __attribute__((always_inline)) {
    if (st + 1 < stages) wait_vmcnt<2 * kLoads>();
    else wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (st + 2 < stages) issue(st + 2);
  };
  issue(0);
  if (stages > 1) issue(1);

  // ---- operands ----
  u32x4 qf[2][kSteps];
  int lim[2];  // the lane's token per block: the last key that it sees
#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    const int row = min(row0 + 32 * blk + r, rows - 1), tok = row / G;
    lim[blk] = tok;
    const uint16_t *const qp = a.q + (int64_t)(w.start + tok) * a.q_stride + (int64_t)(kvh * G + row % G) * D + 8 * h;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) qf[blk][ks] = *(const u32x4 *)(qp + 16 * ks);
  }
  // K fragment ks: row r, chunk 2 ks + h.  V: the lane addresses dims 16 (gi % 2)
  // + 4 x .. of 32, key 4 h + c.
  const uint32_t k_at = (uint32_t)(r * 2 * D + 16 * (h ^ swizzle_k<D>(r)));
  const int v_key = 4 * h + ((lane >> 2) & 3), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = (uint32_t)(kTile + v_key * 2 * D + 16 * (v_chunk ^ swizzle_v<D>(v_key)) + 8 * (lane & 1));

  u32x4 kf[kSteps], vf[2][kDims];
  auto half_base = [&](int hf) { return lds0 + (uint32_t)((hf / 2) % kSlots * (2 * kTile) + (hf & 1) * (kTile / 2)); };
  auto read_k = [&](int hf) __attribute__((always_inline)) {
    const uint32_t at = half_base(hf) + k_at;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) kf[ks] = lds_b128(at ^ (32 * ks));
  };
  auto read_v = [&](int hf) __attribute__((always_inline)) {
    const uint32_t at = half_base(hf) + v_at;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < kDims; ++db) {
        const u32x2 lo = lds_tr16((at ^ (64 * db)) + j * 32 * D), hi = lds_tr16((at ^ (64 * db)) + j * 32 * D + 16 * D);
        vf[j][db] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
  };

  const float sl2 = a.scale * kLog2e;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};  // base-2 domain; l of this lane's keys
  f32x16 o[2][kDims];
#pragma unroll
  for (int blk = 0; blk < 2; ++blk)
#pragma unroll
    for (int db = 0; db < kDims; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[blk][db][i] = 0.f;

  float s[2][16], mx[2];  // raw scores of the half at hand, and their maxima
  f32x16 sn[2];           // the next half's
  // Pairs of scores (b, i), (b, i + 1): b = x / 8, i = 2 (x % 8), x = 0..15.
  auto take_next = [&](int x) __attribute__((always_inline)) {
    const int b = x / 8, i = 2 * (x % 8);
    s[b][i] = acc_read(sn[b][i]);
    s[b][i + 1] = acc_read(sn[b][i + 1]);
    mx[b] = fmaxf(fmaxf(s[b][i], s[b][i + 1]), i ? mx[b] : -INFINITY);
  };
  bool redo = false;
  sync(0);
  if (nhalf > 0) {
    read_k(0);
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sn[blk][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) sn[blk] = mfma32x32<F16>(kf[ks], qf[blk][ks], sn[blk]);
    }
    if (nhalf > 1) read_k(1);
    acc_settle();
#pragma unroll
    for (int x = 0; x < 16; ++x) take_next(x);
  }
  for (int hf = 0; hf < nhalf; ++hf) {
    const bool masked = hf >= full;
    if (masked) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const int last = lim[blk] - 32 * hf - 4 * h;
        mx[blk] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[blk][i] = 8 * (i >> 2) + (i & 3) <= last ? s[blk][i] : -INFINITY;
          mx[blk] = fmaxf(mx[blk], s[blk][i]);
        }
      }
    }
    const bool grow = mx[0] * sl2 > m_run[0] + kRescaleSlack || mx[1] * sl2 > m_run[1] + kRescaleSlack;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      acc_settle();
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        const f32x2_t both = halves(mx[blk] * sl2);
        const float m_new = fmaxf(m_run[blk], fmaxf(both[0], both[1]));
        const float alpha = __builtin_amdgcn_exp2f(m_run[blk] - (m_new == -INFINITY ? 0.f : m_new));
        l_run[blk] *= alpha;
        m_run[blk] = m_new;
#pragma unroll
        for (int db = 0; db < kDims; ++db)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[blk][db][i] = acc_write(acc_read(o[blk][db][i]) * alpha);
      }
    }
    const float neg_m[2] = {m_run[0] == -INFINITY ? 0.f : -m_run[0], m_run[1] == -INFINITY ? 0.f : -m_run[1]};
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) asm volatile("" : "+a"(qf[blk][ks]));  // Q stays in AGPRs

    // A: the next half's scores beside this one's exponentials.  (Behind the
    // wave's last half kf holds keys that nothing asks for.)
    read_v(hf);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int blk = 0; blk < 2; ++blk)
#pragma unroll
      for (int i = 0; i < 16; ++i) sn[blk][i] = 0.f;
    u32x4 pb[2][2];
#pragma unroll
    for (int m = 0; m < 2 * kSteps; ++m) {
      sn[m & 1] = mfma32x32<F16>(kf[m >> 1], qf[m & 1][m >> 1], sn[m & 1]);
#pragma unroll
      for (int x = 8 / kSteps * m; x < 8 / kSteps * (m + 1); ++x) {
        const int b = x / 8, i = 2 * (x % 8);
        float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], sl2, neg_m[b]));
        float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i + 1], sl2, neg_m[b]));
        // Probabilities in the type of V: half a step each, against fp32 sums of both.
        uint32_t w = pack2<F16>(p0, p1);
        asm volatile("" : "+v"(p0), "+v"(p1), "+v"(w));  // here, not where they are used
        s[b][i] = p0;
        s[b][i + 1] = p1;
        pb[b][i / 8][(i / 2) % 4] = w;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!(hf & 1) && hf / 2 + 1 < stages) sync(hf / 2 + 1);

    // B: O of this half beside its sums and the next half's maxima (from the
    // third MFMA on: the scores are there then).
    if (hf + 2 < nhalf) read_k(hf + 2);
    if (masked) {
      // A probability of 0 times a V that is not finite is NaN: rows before such a
      // V would not be what they are without it.
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int db = 0; db < kDims; ++db)
#pragma unroll
          for (int c = 0; c < 4; ++c) bad |= not_finite2<F16>(vf[j][db][c]);
      redo |= __builtin_amdgcn_ballot_w64(bad) != 0;
    }
    __builtin_amdgcn_sched_barrier(0);
    float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
    constexpr int kPv = 4 * kDims;
#pragma unroll
    for (int m = 0; m < kPv; ++m) {
      const int blk = m & 1, db = (m >> 1) % kDims, j = m / (2 * kDims);
      o[blk][db] = mfma32x32<F16>(vf[j][db], pb[blk][j], o[blk][db]);
#pragma unroll
      for (int x = m < 2 ? 0 : 16 * (m - 2) / (kPv - 2); x < (m < 2 ? 0 : 16 * (m - 1) / (kPv - 2)); ++x) {
        const int b = x / 8, i = 2 * (x % 8);
        sum[b][0] += s[b][i];
        sum[b][1] += s[b][i + 1];
        take_next(x);
        asm volatile("" : "+v"(sum[b][0]), "+v"(sum[b][1]), "+v"(mx[b]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) l_run[blk] += sum[blk][0] + sum[blk][1];
  }
  // The stages that other waves still read.
  for (int st = (nhalf + 1) / 2 + 1; st < stages; ++st) sync(st);
  if (__builtin_expect(redo, 0)) {
    take_rows<D, F16>(a, w, kvh, row0, tok_hi);
    return;
  }
  acc_settle();

#pragma unroll
  for (int blk = 0; blk < 2; ++blk) {
    const f32x2_t both = halves(l_run[blk]);
    const float L = both[0] + both[1], inv = L == 0.f ? 0.f : 1.0f / L;
    const int row = row0 + 32 * blk + r;
    if (row >= rows) continue;
    // Lane (r, h): dims 32 db + 8 q + 4 h + i of its row.
    uint16_t *const op = a.out + ((int64_t)(w.start + lim[blk]) * a.Hq + kvh * G + row % G) * D + 4 * h;
#pragma unroll
    for (int db = 0; db < kDims; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u32x2 v;
        v[0] = pack2<F16>(acc_read(o[blk][db][4 * q]) * inv, acc_read(o[blk][db][4 * q + 1]) * inv);
        v[1] = pack2<F16>(acc_read(o[blk][db][4 * q + 2]) * inv, acc_read(o[blk][db][4 * q + 3]) * inv);
        *(u32x2 *)(op + 32 * db + 8 * q) = v;
      }
  }
}

template <int D, bool F16>
hipError_t launch(const GqaPackedArgs &a, hipStream_t s) {
  auto k = gqa_packed_kernel<D, F16>;
  constexpr int lds = kSlots * 2 * kStageKeys * D * 2;
  static const bool attr = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds) ==
                           hipSuccess;
  if (!attr) return hipErrorInvalidValue;
  // Every sequence ends in at most one tile that is not full.
  const int64_t tiles = (int64_t)a.N * (a.Hq / a.Hkv) / kTileRows + (a.S < a.N ? a.S : a.N);
  const int classes = a.Hkv % 8 == 0 ? 8 : a.Hkv % 4 == 0 ? 4 : a.Hkv % 2 == 0 ? 2 : 1;
  const int64_t in_class = tiles * (a.Hkv / classes), per_xcd = (in_class + kXcds / classes - 1) / (kXcds / classes);
  hipLaunchKernelGGL(k, dim3((uint32_t)(per_xcd * kXcds)), dim3(64 * kWaves), lds, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_gqa_packed(const GqaPackedArgs &a, hipStream_t s) {
  if (a.D == 128) return a.dtype == GQA_FP16 ? launch<128, true>(a, s) : launch<128, false>(a, s);
  return a.dtype == GQA_FP16 ? launch<64, true>(a, s) : launch<64, false>(a, s);
}

}  // namespace moe
