// Causal attention of several packed prompts on gfx950.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j - max),
//   over the keys j of t's sequence up to t; head h reads KV head h / G.
//
// Long prompts are bound by the matrix cores and, next to them, by the issue of
// the softmax's vector instructions.  A workgroup owns 256 query rows of one KV
// head (a sequence's tokens with their G heads side by side, row = token * G +
// head, whatever G is), each of its eight waves, two per SIMD, 32 of them.  A wave
// overlaps its own work: per 32 keys
//   A: S^T = K Q^T of the next 32 keys (MFMA) beside the exponentials and sums of
//      these,
//   B: O^T += V^T P^T of these (MFMA) beside the next maxima,
// with the operands of each read from LDS one phase ahead.  A lane holds sixteen
// scores of one query (the partner lane l ^ 32 the other sixteen), so the online
// softmax is lane-local and P is the B operand of O^T as it lies.  (Four waves of
// 64 rows, one per SIMD, read half as much from LDS but cannot issue more than one
// instruction in four cycles: 1.03 PFLOP/s at 16384 tokens.)
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
constexpr int kWaves = 8;
constexpr int kWaveRows = 32;
constexpr int kStageKeys = 64;
constexpr int kSlots = 4;
constexpr int kWindow = 4;      // sequences per lane that a search looks at together
typedef short i16x4 __attribute__((ext_vector_type(4)));

// Row i of a stage's K (V) tile holds its 16-byte chunk c at place c ^ swizzle(i):
// sixteen lanes that read one chunk of sixteen K rows, or 32 lanes that read four
// chunks of four V rows, then meet sixteen different bank groups.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swizzle_v(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

// 16 bytes per lane from a buffer straight into LDS at `dst` + 16 l (load j 1024 j
// further).  As inline
// assembly (it has no output register): the compiler would make every later LDS
// read wait for all such loads in flight; the kernel waits with exact counts.
// (Nothing else in this kernel uses m0.)
template <int N>
__device__ __forceinline__ void load_lds(u32x4 rsrc, uint32_t dst, const uint32_t (&off)[N]) {
  static_assert(N == 1 || N == 2, "loads of a wave");
  if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
        :
        : "s"(dst), "v"(off[0]), "v"(off[1]), "s"(rsrc)
        : "memory", "scc");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(dst), "v"(off[0]), "s"(rsrc)
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
// An MFMA's results take up to 19 wait states, and across a branch the compiler can
// miss that they are not there yet.  Where they are read in another block than
// the MFMA's, mfma_settle() stands before, or two later MFMAs (each waits for the
// one before), and pin() keeps the reads behind that.
__device__ __forceinline__ void mfma_settle() { asm volatile("s_nop 15\n\ts_nop 3" ::: "memory"); }
__device__ __forceinline__ float pin(float x) {
  asm volatile("" : "+v"(x));
  return x;
}
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
      return wave_total(c);
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
      const int incl = wave_scan(c);
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

// The rows of a wave from row0 on, a row per pair of lanes l, l + 32 (each with half
// of the dims) and a key per step, in plain fp32: for waves that meet a V that only
// some of their rows see and that is not finite.  A key that a row does not see
// touches nothing of it.
template <int D, bool F16>
__device__ __forceinline__ void take_rows(const GqaPackedArgs &a, const Rows &w, int kvh, int row0, int tok_hi) {
  constexpr int kPart = D / 16;  // 16-byte chunks of a lane
  const int G = a.Hq / a.Hkv, rows = w.len * G, lane = threadIdx.x & 63;
  const int row = min(row0 + lane % kWaveRows, rows - 1), tok = row / G, head = kvh * G + row % G;
  const int first = lane / kWaveRows * (D / 2);  // of the lane's dims
  const uint16_t *const qp = a.q + (int64_t)(w.start + tok) * a.q_stride + (int64_t)head * D + first;
  u32x4 q[kPart];
#pragma unroll
  for (int c = 0; c < kPart; ++c) q[c] = *(const u32x4 *)(qp + 8 * c);
  float o[8 * kPart], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < 8 * kPart; ++d) o[d] = 0.f;
  const float sl2 = a.scale * kLog2e;
#pragma clang loop unroll(disable)
  for (int key = 0; key <= tok_hi; ++key) {
    const uint16_t *const kp = a.k + (int64_t)(w.start + key) * a.k_stride + (int64_t)kvh * D + first;
    const uint16_t *const vp = a.v + (int64_t)(w.start + key) * a.v_stride + (int64_t)kvh * D + first;
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < kPart; ++c) {
      const u32x4 x = *(const u32x4 *)(kp + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = __builtin_fmaf(element<F16>(q[c], i), element<F16>(x, i), dot);
    }
    const f32x2_t both = halves(dot);
    const bool seen = key <= tok;
    const float sc = seen ? (both[0] + both[1]) * sl2 : -INFINITY;
    const float m_new = fmaxf(m, sc), ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - ref), p = exp2f(sc - ref);
    m = seen ? m_new : m;
    l = seen ? l * alpha + p : l;
#pragma unroll
    for (int c = 0; c < kPart; ++c) {
      const u32x4 x = *(const u32x4 *)(vp + 8 * c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __builtin_fmaf(p, element<F16>(x, i), o[8 * c + i] * alpha);
        o[8 * c + i] = seen ? y : o[8 * c + i];
      }
    }
  }
  if (row0 + lane % kWaveRows >= rows) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint32_t *const op = (uint32_t *)(a.out + ((int64_t)(w.start + tok) * a.Hq + head) * D + first);
#pragma unroll
  for (int d = 0; d < 8 * kPart; d += 2) op[d / 2] = pack2<F16>(o[d] * inv, o[d + 1] * inv);
}

template <int D, bool F16>
__global__ __launch_bounds__(64 * kWaves, 2) void gqa_packed_kernel(GqaPackedArgs a) {
  constexpr int kSteps = D / 16;                    // QK MFMAs per half stage
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
  const int row0 = w.tile * kTileRows + kWaveRows * wave;                      // of the wave
  const int keys = min(w.len, (w.tile * kTileRows + kTileRows - 1) / G + 1);  // that the workgroup sees
  const int stages = (keys + kStageKeys - 1) / kStageKeys;
  // The wave's half stages of 32 keys: all up to its last token's, the first
  // `full` of them seen by all of its tokens.
  const int tok_lo = row0 / G, tok_hi = min(w.len - 1, (row0 + kWaveRows - 1) / G);
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
    load_lds(krs, dst, k_off);
    load_lds(vrs, dst + kTile, v_off);
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
  const int row = min(row0 + r, rows - 1), tok = row / G;  // the lane's; tok: the last key that it sees
  const int64_t at_q = (int64_t)(w.start + tok), head = kvh * G + row % G;
  u32x4 qf[kSteps];
#pragma unroll
  for (int ks = 0; ks < kSteps; ++ks) qf[ks] = *(const u32x4 *)(a.q + at_q * a.q_stride + head * D + 8 * h + 16 * ks);
  // K fragment ks: row r, chunk 2 ks + h.  V: the lane addresses dims 16 (gi % 2)
  // + 4 x .. of 32, key 4 h + c.
  const uint32_t k_at = (uint32_t)(r * 2 * D + 16 * (h ^ swizzle_k<D>(r)));
  const int v_key = 4 * h + ((lane >> 2) & 3), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = (uint32_t)(kTile + v_key * 2 * D + 16 * (v_chunk ^ swizzle_v<D>(v_key)) + 8 * (lane & 1));

  u32x4 kf[kSteps], vf[2][kDims];
  auto half_base = [&](int hf) { return lds0 + (uint32_t)((hf / 2) % kSlots * (2 * kTile) + (hf & 1) * (kTile / 2)); };
  // Operand reads, spread over the MFMAs before their use: all at once they would
  // not fit the registers, and the waves' bursts would wait for each other.
  auto read_k = [&](int hf, int ks) __attribute__((always_inline)) {
    kf[ks] = lds_b128((half_base(hf) + k_at) ^ (32 * ks));
  };
  auto read_v = [&](int hf, int j, int db) __attribute__((always_inline)) {
    const uint32_t at = ((half_base(hf) + v_at) ^ (64 * db)) + j * 32 * D;
    const u32x2 lo = lds_tr16(at), hi = lds_tr16(at + 16 * D);
    vf[j][db] = u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  const float sl2 = a.scale * kLog2e;
  float m_run = -INFINITY, l_run = 0.f;  // base-2 domain; l of this lane's keys
  f32x16 o[kDims], s0, s1;
#pragma unroll
  for (int db = 0; db < kDims; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float mx = -INFINITY;  // of the raw scores of the half at hand

  // One half: its scores in s; the next half's come into sn.
  // The second four waves, each beside one of the first on its SIMD, meet them at
  // the barrier a phase earlier in their own work, so that one's exponentials fall
  // beside the other's MFMAs.
  auto half = [&](int hf, f32x16 &s, f32x16 &sn) __attribute__((always_inline)) {
    if (wave >= kWaves / 2 && !(hf & 1) && hf / 2 + 1 < stages) sync(hf / 2 + 1);
    if (hf >= full) {
      const int last = tok - 32 * hf - 4 * h;
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = 8 * (i >> 2) + (i & 3) <= last ? s[i] : -INFINITY;
        mx = fmaxf(mx, s[i]);
      }
    }
    if (__builtin_amdgcn_ballot_w64(mx * sl2 > m_run + kRescaleSlack)) {
      mfma_settle();
      const f32x2_t both = halves(mx * sl2);
      const float m_new = fmaxf(m_run, fmaxf(both[0], both[1]));
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int db = 0; db < kDims; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = pin(o[db][i]) * alpha;
    }
    const float neg_m = m_run == -INFINITY ? 0.f : -m_run;

    // A: the next half's scores beside this one's exponentials.  (Behind the
    // wave's last half these are of rows in the ring that nothing asks for.)
#pragma unroll
    for (int ks = kSteps / 2; ks < kSteps; ++ks) read_k(hf + 1, ks);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) sn[i] = 0.f;
    u32x4 pb[2];
    float sum0 = 0.f, sum1 = 0.f, p0 = 0.f, p1 = 0.f;
    // Pair x of probabilities (in the type of V: half a step each, against fp32
    // sums of both) and of the sums; a pair later than its exponentials.
    auto take = [&](int x) __attribute__((always_inline)) {
      uint32_t w = pack2<F16>(p0, p1);
      sum0 += p0;
      sum1 += p1;
      asm volatile("" : "+v"(w), "+v"(sum0), "+v"(sum1));  // here, not where they are used
      pb[x / 4][x % 4] = w;
    };
    constexpr int kEach = 8 / kSteps;  // pairs of scores per MFMA
#pragma unroll
    for (int m = 0; m < kSteps; ++m) {
      sn = mfma32x32<F16>(kf[m], qf[m], sn);
#pragma unroll
      for (int x = kEach * m; x < kEach * (m + 1); ++x) {
        const float e0 = pin(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * x], sl2, neg_m)));
        const float e1 = pin(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * x + 1], sl2, neg_m)));
        if (x > 0) take(x - 1);
        p0 = e0;
        p1 = e1;
      }
      if (m == kSteps - 1) take(7);
      // V's first keys beside the first half of the MFMAs, the others (in the place
      // of K fragments that are done with) beside the second.
      if (m < kSteps / 2) read_v(hf, 0, m % kDims);
      else read_v(hf, 1, m % kDims);
      __builtin_amdgcn_sched_barrier(0);
    }
    l_run += sum0 + sum1;
    if (wave < kWaves / 2 && !(hf & 1) && hf / 2 + 1 < stages) sync(hf / 2 + 1);

    // B: O of this half beside the next half's maxima (from the third MFMA on: the
    // scores are there then).
    constexpr int kPv = 2 * kDims;
    mx = -INFINITY;
#pragma unroll
    for (int m = 0; m < kPv; ++m) {
      o[m % kDims] = mfma32x32<F16>(vf[m / kDims][m % kDims], pb[m / kDims], o[m % kDims]);
#pragma unroll
      for (int x = m < 2 ? 0 : 8 * (m - 2) / (kPv - 2); x < (m < 2 ? 0 : 8 * (m - 1) / (kPv - 2)); ++x) {
        sn[2 * x] = pin(sn[2 * x]);
        sn[2 * x + 1] = pin(sn[2 * x + 1]);
        mx = pin(fmaxf(fmaxf(sn[2 * x], sn[2 * x + 1]), mx));
      }
      if (m >= kDims) read_k(hf + 2, m - kDims);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  sync(0);
  if (nhalf > 0) {
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) read_k(0, ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) s0[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) s0 = mfma32x32<F16>(kf[ks], qf[ks], s0);
#pragma unroll
    for (int ks = 0; ks < kSteps / 2; ++ks) read_k(1, ks);
    mfma_settle();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s0[i] = pin(s0[i]);
      mx = fmaxf(mx, s0[i]);
    }
    for (int hf = 0; hf < nhalf; hf += 2) {
      half(hf, s0, s1);
      if (hf + 1 == nhalf) break;
      half(hf + 1, s1, s0);
    }
  }
  // The stages that other waves still read.
  for (int st = (nhalf + 1) / 2 + 1; st < stages; ++st) sync(st);
  mfma_settle();

  // In the masked halves a probability of 0 stood before values that the row does
  // not see, and 0 times one that is not finite is NaN.  Looked for only where O is
  // not finite; then the wave takes its rows again, slowly.
  float zero = 0.f;
#pragma unroll
  for (int db = 0; db < kDims; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      o[db][i] = pin(o[db][i]);
      zero = __builtin_fmaf(o[db][i], 0.f, zero);
    }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(zero != 0.f) != 0, 0)) {
    bool bad = false;
    for (int key = 32 * full + lane / kChunks; key < min(32 * nhalf, w.len); key += 64 / kChunks) {
      const u32x4 v = *(const u32x4 *)(v0 + (int64_t)key * a.v_stride + 8 * (lane % kChunks));
#pragma unroll
      for (int c = 0; c < 4; ++c) bad |= not_finite2<F16>(v[c]);
    }
    if (nhalf > 0 && __builtin_amdgcn_ballot_w64(bad)) {
      take_rows<D, F16>(a, w, kvh, row0, tok_hi);
      return;
    }
  }
  const f32x2_t both = halves(l_run);
  const float L = both[0] + both[1], inv = L == 0.f ? 0.f : 1.0f / L;
  // Lane (r, h): dims 32 db + 8 q + 4 h + i of its row.
  uint16_t *const op = a.out + (at_q * a.Hq + head) * D + 4 * h;
#pragma unroll
  for (int db = 0; db < kDims; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u32x2 v;
      v[0] = pack2<F16>(o[db][4 * q] * inv, o[db][4 * q + 1] * inv);
      v[1] = pack2<F16>(o[db][4 * q + 2] * inv, o[db][4 * q + 3] * inv);
      if (row0 + r < rows) *(u32x2 *)(op + 32 * db + 8 * q) = v;
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
