// Causal attention of several packed prompts on gfx950.
//
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j - max),
//   over the keys j of t's sequence up to t; head h reads KV head h / G.
//
// Long prompts are bound by the matrix cores and, next to them, by the issue of
// the softmax's vector instructions.  A workgroup owns 128 query rows of one KV
// head (a sequence's tokens with their G heads side by side, row = token * G +
// head, whatever G is), each of its four waves, one per SIMD, 32 of them; two
// workgroups (four with heads of 64) share a CU, so that one's exponentials, waits and ends fall beside the
// other's MFMAs.  A wave also overlaps its own work: per 32 keys
//   A: S^T = K Q^T of the next 32 keys (MFMA) beside the exponentials and sums of
//      these,
//   B: O^T += V^T P^T of these (MFMA) beside the next maxima,
// with the operands of each read from LDS one phase ahead.  A lane holds sixteen
// scores of one query (the partner lane l ^ 32 the other sixteen), so the online
// softmax is lane-local and P is the B operand of O^T as it lies.
//   Measured before, each against two workgroups of four waves as they were then: one
// workgroup of eight such waves per CU (16384 tokens 2.08 against 2.05 ms, 16 ragged
// prompts 114 against 100 us: nothing runs beside its start and end), and four waves
// of 64 rows, one per SIMD, that read half as much from LDS but issue at most one
// instruction in four cycles (2.13 ms).
//
// K and V come in stages of 32 keys, global -> LDS in whole rows (buffer loads with an
// LDS destination; keys behind the sequence's end read as zeros), three to four
// stages ahead in a ring of five, with one barrier per stage.
//
// Measured, 32 query heads of 128 on 8 KV heads, bf16: one prompt of 16384 tokens 2.0 to
// 2.15 ms by card, 1.02 to 1.10 PFLOP/s, the matrix cores 58 % busy (1.48 ms with
// inputs of 0: the card's power bounds the rest; a matrix product of 16384 cubed runs
// at 1.31 PFLOP/s, with inputs of 0 at 1.77); 16 prompts of 65 to 1134 tokens 83 us
// behind 5 for the list: the start and end of a tile, 5 us with one workgroup left
// beside it, and the longest tiles; four prompts of up to 48 tokens 6 us: launch and
// one round of loads.
#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"
#include "launch.h"

namespace moe {

using namespace gqa;

namespace {

constexpr int kWaveRows = 32;   // query rows of a wave
constexpr int kWaves = 4;
constexpr int kTileRows = kWaveRows * kWaves;  // of a workgroup
constexpr int kStageKeys = 32;
constexpr int kRing = 5;        // stages in LDS
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
template <int N>
__device__ __forceinline__ void load_lds(u32x4 rsrc, uint32_t dst, const uint32_t (&off)[N]) {
  static_assert(N == 1 || N == 2, "loads of a wave");
  if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
        :
        : "s"(dst), "v"(off[0]), "v"(off[1]), "s"(rsrc)
        : "memory", "scc", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(dst), "v"(off[0]), "s"(rsrc)
                 : "memory", "m0");
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
__device__ __forceinline__ void lds_write_b64(uint32_t at, u32x2 v) {
#if defined(__HIP_DEVICE_COMPILE__)
  *(GQA_AS_LDS u32x2 *)at = v;
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
template <bool F16>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}

template <bool F16>
__device__ __forceinline__ float element(u32x4 x, int i) {
  return to_f32<F16>(i & 1 ? x[i / 2] >> 16 : x[i / 2] & 0xffffu);
}

// A workgroup's rows: tile `tile` of the sequence that starts at token `start` and
// has `len`.
struct Rows {
  int start, len, tile, none;
};

// n / d for n < 2^26, d <= 64 and magic = ceil(2^32 / d).
__device__ __forceinline__ int quotient(int n, int d, uint32_t magic) {
  return d == 1 ? n : (int)__umulhi((uint32_t)n, magic);
}

// Bound s of the sequences as given, forced into [0, N].  Bounds are taken as the
// largest so far, so that sequences never overlap and there are no more tiles than
// the list has room for.
__device__ __forceinline__ int bound(const GqaPackedArgs &a, int s) { return max(0, min(a.starts[s], a.N)); }
// Reports bounds that are not what they are taken as.
__device__ __forceinline__ void check_bounds(const GqaPackedArgs &a, int s, const Rows &q) {
  if (a.starts[s] != q.start || a.starts[s + 1] != q.start + q.len) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
}
// The list of all sequences' tiles, those that see the most keys first
// (the last workgroups to run are short then).  One workgroup sorts them by counting
// in kClasses classes of equally many stages; the order within a class does not
// matter to any result.  A search of every workgroup for its own tile took 3 to 5 us
// of its 10 to 50.
constexpr int kPlanThreads = 512;   // (100 prompts of 64 tokens 35.5 us, 37.0 with 1024)
constexpr int kClasses = kPlanThreads;
constexpr int kPlanLds = 2048;  // sequences whose tile sums lie in LDS
__device__ __forceinline__ int plan_scan(int x, int *lds, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, incl = wave_scan(x);
  __syncthreads();  // the last scan's sums have been read
  if (lane == kWave - 1) lds[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    const int v = lds[w];
    before += w < wave ? v : 0;
    all += v;
  }
  *total = all;
  return before + incl - x;
}
// The largest of the earlier threads' numbers (not negative) and of all.
__device__ __forceinline__ int plan_max_scan(int x, int *lds, int *top) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, incl = wave_max_scan(x);
  __syncthreads();
  if (lane == kWave - 1) lds[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    const int v = lds[w];
    before = max(before, w < wave ? v : 0);
    all = max(all, v);
  }
  *top = all;
  return max(before, incl);
}
template <bool LDS>  // S <= kPlanLds
__global__ __launch_bounds__(kPlanThreads) void gqa_packed_plan(GqaPackedArgs a) {
  __shared__ int waves[kPlanThreads / kWave], count[kClasses], longest;
  // Tiles before a sequence, and the sequences' starts and lengths, [S] each.
  __shared__ int lds[3][LDS ? kPlanLds : 1];
  int *const sums = LDS ? lds[0] : a.tile_sums;
  int *const first = LDS ? lds[1] : a.tile_sums + a.S;
  int *const length = LDS ? lds[2] : a.tile_sums + 2 * a.S;
  const int tid = threadIdx.x;
  if (tid == 0) longest = 0;
  count[tid] = 0;
  int total = 0, top = 0, most_here = 0;
  for (int base = 0; base < a.S; base += kPlanThreads) {
    const int s = base + tid;
    int here, all;
    Rows q = {0, 0, 0, 0};
    q.start = max(top, plan_max_scan(s < a.S ? bound(a, s) : 0, waves, &here));
    if (s < a.S) {
      q.len = max(0, bound(a, s + 1) - q.start);
      check_bounds(a, s, q);
    }
    top = max(top, here);
    const int at = total + plan_scan((q.len * a.G + kTileRows - 1) / kTileRows, waves, &all);
    if (s < a.S) {
      sums[s] = at;
      first[s] = q.start;
      length[s] = q.len;
    }
    total += all;
    most_here = max(most_here, q.len);
  }
  if (most_here > 0) atomicMax(&longest, most_here);
  if (tid == 0) *a.num_tiles = total;
  __syncthreads();
  const int most = max(1, (longest + kStageKeys - 1) / kStageKeys);
  struct Tile {
    Rows w;
    int cls;
  };
  auto tile_at = [&](int i) __attribute__((always_inline)) {
    int lo = 0, hi = a.S - 1;  // the last sequence with at most i tiles before it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sums[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const Rows w = {first[lo], length[lo], i - sums[lo], 0};
    const int keys = min(w.len, quotient(w.tile * kTileRows + kTileRows - 1, a.G, a.G_magic) + 1);
    const int shorter = most - (keys + kStageKeys - 1) / kStageKeys;  // 0 .. most - 1
    return Tile{w, most <= kClasses ? shorter : (int)((int64_t)shorter * (kClasses - 1) / most)};
  };
  Tile mine = {};
  for (int i = tid; i < total; i += kPlanThreads) {
    const Tile t = tile_at(i);
    if (i == tid) mine = t;
    atomicAdd(count + t.cls, 1);
  }
  __syncthreads();
  int all;
  const int at = plan_scan(count[tid], waves, &all);
  count[tid] = at;
  __syncthreads();
  for (int i = tid; i < total; i += kPlanThreads) {
    const Tile t = i == tid ? mine : tile_at(i);
    ((Rows *)a.tiles)[atomicAdd(count + t.cls, 1)] = t.w;
  }
}

// The rows of a wave from row0 on, a row per pair of lanes l, l + 32 (each with half
// of the dims) and a key per step, in plain fp32: for waves that meet a V that only
// some of their rows see and that is not finite.  A key that a row does not see
// touches nothing of it.
template <int D, bool F16>
__device__ __forceinline__ void take_rows(const GqaPackedArgs &a, const Rows &w, int kvh, int row0, int tok_hi) {
  constexpr int kPart = D / 16;  // 16-byte chunks of a lane
  const int G = a.G, rows = w.len * G, lane = threadIdx.x & 63;
  const int row = min(row0 + lane % kWaveRows, rows - 1), tok = quotient(row, G, a.G_magic);
  const int head = kvh * G + row - tok * G;
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
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(q[c][i]));  // packed; as floats outside the loop they spill
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

// Workgroups per CU, by their LDS.  D = 64: with four instead of three 16 heads of 16384
// tokens take 622 us, not 640, and 50 prompts of 1000 125, not 134.
template <int D> constexpr int kResident = D == 128 ? 2 : 4;

template <int D, bool F16>
__global__ __launch_bounds__(64 * kWaves, kResident<D>) void gqa_packed_kernel(GqaPackedArgs a) {
  constexpr int kSteps = D / 16;                    // QK MFMAs per stage
  constexpr int kDims = D / 32;                     // 32-dim tiles of O
  constexpr int kTile = kStageKeys * D * 2;         // bytes of a stage's K (or V)
  constexpr int kLoads = kTile / 1024 / kWaves;     // of K (or V) per wave and stage
  constexpr int kChunks = D / 8;                    // 16-byte chunks of a row
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = sgpr(threadIdx.x >> 6);
  const int G = a.G;
  // Beside the waves of another workgroup on the CU, the dependent steps outside of
  // the loop go first.
  __builtin_amdgcn_s_setprio(3);

  // Workgroups go round the eight XCDs; the tiles of one KV head stay on the
  // XCDs of its class, which share K and V through their L2.
  // The second workgroups of an XCD's CUs come in the opposite order of the first, so
  // that the longest tile of the first round shares its CU with the shortest of
  // the second (four prompts of 512 tokens 23.3 -> 20.0 us, one of 2048 49.7 -> 48.0,
  // one of 3000 85.9 -> 87.0).
  const int xcd = blockIdx.x % kXcds, nth_xcd = blockIdx.x / kXcds;
  const int slot8 = nth_xcd >= a.xcd_cus && nth_xcd < 2 * a.xcd_cus ? 3 * a.xcd_cus - 1 - nth_xcd : nth_xcd;
  const int in_class = (slot8 << a.class_xcds) + (xcd >> (3 - a.class_xcds)), nth = in_class / a.per_class;
  const int kvh = (xcd & (7 >> a.class_xcds)) + ((in_class - nth * a.per_class) << (3 - a.class_xcds));
  Rows w;
  if (!a.listed) {  // S <= 64
    Rows q = {wave_max_scan(lane < a.S ? bound(a, lane) : 0), 0, 0, 0};
    if (lane < a.S) {
      q.len = max(0, bound(a, lane + 1) - q.start);
      check_bounds(a, lane, q);
    }
    const int T = (q.len * G + kTileRows - 1) / kTileRows;
    int at, x;  // the tile's sequence and its number there
    if (!a.searched) {  // in the order of the sequences, each one's longest first
      const int incl = wave_scan(T);
      const uint64_t behind = __builtin_amdgcn_ballot_w64(incl > nth);
      if (!behind) return;
      at = sgpr(__builtin_ctzll(behind));
      x = __builtin_amdgcn_readlane(incl, at) - 1 - nth;
    } else {
      // Tiles of the highest number, which see the most keys, first.  Tiles numbered
      // T and up: `above`; the least such T with at most nth of them, `top`, has the
      // wanted number just below, where every sequence of at least `top` tiles, `some`
      // in all, has one of each number.
      int above = 0;
#pragma unroll 4
      for (int j = 0; j < a.S; ++j) above += max(0, __builtin_amdgcn_readlane(T, j) - T);
      constexpr int kMore = 1 << 28;  // than tiles
      const int top = kMore - __builtin_amdgcn_readlane(wave_max_scan(above <= nth ? kMore - T : 0), kWave - 1);
      const uint64_t those = __builtin_amdgcn_ballot_w64(T >= top);
      const int some = (int)__popcll(those);
      const int rest = nth - __builtin_amdgcn_readlane(above, sgpr(__builtin_ctzll(__builtin_amdgcn_ballot_w64(T == top))));
      x = top - 1 - rest / some;
      if (x < 0) return;
      at = sgpr(__builtin_ctzll(__builtin_amdgcn_ballot_w64(T >= top && (int)__popcll(those & lanemask_lt()) == rest % some)));
    }
    w = Rows{__builtin_amdgcn_readlane(q.start, at), __builtin_amdgcn_readlane(q.len, at), x, 0};
  } else {
    // Scalar loads: the list does not change while the kernel runs.
    typedef const __attribute__((address_space(4))) int *Uniform;
    const Uniform list = (Uniform)(const __attribute__((address_space(4))) void *)a.tiles + 4 * (int64_t)min(nth, a.listed - 1);
    const int num = *(Uniform)(const __attribute__((address_space(4))) void *)a.num_tiles;
    w = Rows{list[0], list[1], list[2], 0};
    if (nth >= num) return;
  }

  const int rows = w.len * G;                                           // of the sequence
  const int row0 = w.tile * kTileRows + kWaveRows * wave;                      // of the wave
  const int keys = min(w.len, quotient(w.tile * kTileRows + kTileRows - 1, G, a.G_magic) + 1);  // that the workgroup sees
  const int stages = (keys + kStageKeys - 1) / kStageKeys;
  // The wave's stages: all up to its last token's key, the first `full` of them seen
  // by all of its tokens.
  const int tok_lo = quotient(row0, G, a.G_magic);
  const int tok_hi = min(w.len - 1, quotient(row0 + kWaveRows - 1, G, a.G_magic));
  const int own = row0 < rows ? tok_hi / kStageKeys + 1 : 0, full = (tok_lo + 1) / kStageKeys;

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
  // The next stage to load: its first rows of K and V, its slot and the keys from it on.
  uint64_t k_next = (uint64_t)k0, v_next = (uint64_t)v0;
  uint32_t load_slot = lds0 + wave * kLoads * 1024;
  int load_keys = w.len;
  auto issue = [&]() __attribute__((always_inline)) {
    const uint32_t n1 = (uint32_t)min(kStageKeys, load_keys) - 1u;
    const uint32_t dst = sgpr((int)load_slot);
    load_lds(buffer_words((const void *)k_next, n1 * ksb + 2 * D), dst, k_off);
    load_lds(buffer_words((const void *)v_next, n1 * vsb + 2 * D), dst + kTile, v_off);
    k_next += (uint64_t)kStageKeys * ksb;
    v_next += (uint64_t)kStageKeys * vsb;
    load_keys -= kStageKeys;
    load_slot = load_slot + 2 * kTile >= lds0 + kRing * 2 * kTile ? load_slot - (kRing - 1) * 2 * kTile
                                                                 : load_slot + 2 * kTile;
  };
  // In step st of the loop: stage st + 2 is there for every wave, and every wave is
  // done with stage st - 1, whose slot takes the next one.
  auto sync = [&](int st) __attribute__((always_inline)) {
    if (st + kRing - 2 < stages) wait_vmcnt<2 * kLoads * (kRing - 4)>();
    else wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (st + kRing - 1 < stages) issue();
  };
  // Three stages ahead of Q, since loads return in order; the others behind it.
  for (int st = 0; st < min(3, stages); ++st) issue();

  // ---- operands ----
  const int row = min(row0 + r, rows - 1), tok = quotient(row, G, a.G_magic);  // the lane's; tok: the last key that it sees
  const int64_t at_q = (int64_t)(w.start + tok), head = kvh * G + row - tok * G;
  u32x4 qf[kSteps];
#pragma unroll
  for (int ks = 0; ks < kSteps; ++ks) qf[ks] = *(const u32x4 *)(a.q + at_q * a.q_stride + head * D + 8 * h + 16 * ks);
  // K fragment ks: row r, chunk 2 ks + h.  V: the lane addresses dims 16 (gi % 2)
  // + 4 x .. of 32, key 4 h + c.
  const uint32_t k_at = (uint32_t)(r * 2 * D + 16 * (h ^ swizzle_k<D>(r)));
  const int v_key = 4 * h + ((lane >> 2) & 3), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = (uint32_t)(kTile + v_key * 2 * D + 16 * (v_chunk ^ swizzle_v<D>(v_key)) + 8 * (lane & 1));

  u32x4 kf[kSteps], vf[2][kDims];
  // Operand reads, spread over the MFMAs before their use: all at once they would
  // not fit the registers, and the waves' bursts would wait for each other.
  uint32_t slot[3] = {lds0, lds0 + 2 * kTile, lds0 + 4 * kTile};  // of this stage and the next two
  auto read_k = [&](uint32_t at, int ks) __attribute__((always_inline)) { kf[ks] = lds_b128((at + k_at) ^ (32 * ks)); };
  auto read_v = [&](int j, int db) __attribute__((always_inline)) {
    const uint32_t at = ((slot[0] + v_at) ^ (64 * db)) + j * 32 * D;
    const u32x2 lo = lds_tr16(at), hi = lds_tr16(at + 16 * D);
    vf[j][db] = u32x4{lo[0], lo[1], hi[0], hi[1]};
  };

  const float sl2 = a.scale * kLog2e;
  float m_run = -INFINITY, l_run = 0.f;  // base-2 domain; l of this lane's keys
  float m_top = -INFINITY;               // fp16: limit(m_run), kept (two instructions of a stage)
  f32x16 o[kDims], s0, s1;
#pragma unroll
  for (int db = 0; db < kDims; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  float mx = -INFINITY;  // of the raw scores of the stage at hand

  // One stage: its scores in s; the next one's come into sn.
  auto step = [&](int st, f32x16 &s, f32x16 &sn) __attribute__((always_inline)) {
    // The first of the next stage's scores; they need nothing of what follows.
    // (Behind the wave's last stage these are of rows in the ring that nothing
    // asks for.)
#pragma unroll
    for (int ks = kSteps / 2; ks < kSteps; ++ks) read_k(slot[1], ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) sn[i] = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m) sn = mfma32x32<F16>(kf[m], qf[m], sn);
    __builtin_amdgcn_sched_barrier(0);
    if (st >= full) {
      const int last = tok - kStageKeys * st - 4 * h;
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = 8 * (i >> 2) + (i & 3) <= last ? s[i] : -INFINITY;
        mx = fmaxf(mx, s[i]);
      }
    }
    if (__builtin_amdgcn_ballot_w64(mx * sl2 > (F16 ? m_top : limit<F16>(m_run)))) {
      mfma_settle();
      const f32x2_t both = halves(mx * sl2);
      const float m_new = fmaxf(m_run, reference<F16>(fmaxf(both[0], both[1])));
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
      m_run = m_new;
      m_top = limit<F16>(m_new);
#pragma unroll
      for (int db = 0; db < kDims; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = pin(o[db][i]) * alpha;
    }
    const float neg_m = m_run == -INFINITY ? 0.f : -m_run;

    // A: the rest of the next stage's scores beside this one's exponentials.
    u32x4 pb[2];
    float sum0 = 0.f, sum1 = 0.f, p0 = 0.f, p1 = 0.f;
    // Pair x of probabilities (in the type of V: half a step each, see reference(),
    // against fp32 sums of both) and of the sums; a pair later than its exponentials.
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
      if (m >= 2) sn = mfma32x32<F16>(kf[m], qf[m], sn);
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
      if (m < kSteps / 2) read_v(0, m % kDims);
      else read_v(1, m % kDims);
      __builtin_amdgcn_sched_barrier(0);
    }
    l_run += sum0 + sum1;
    if (st + 2 < stages) sync(st);

    // B: O of this stage beside the next one's maxima (from the third MFMA on: the
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
      if (m >= kDims) read_k(slot[2], m - kDims);
      __builtin_amdgcn_sched_barrier(0);
    }
    slot[0] = slot[1];
    slot[1] = slot[2];
    slot[2] = slot[2] + 2 * kTile >= lds0 + kRing * 2 * kTile ? lds0 : slot[2] + 2 * kTile;
  };

  wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  for (int st = 3; st < min(kRing - 1, stages); ++st) issue();
  __builtin_amdgcn_s_setprio(0);
  if (own > 0) {
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) read_k(slot[0], ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) s0[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < kSteps; ++ks) s0 = mfma32x32<F16>(kf[ks], qf[ks], s0);
#pragma unroll
    for (int ks = 0; ks < kSteps / 2; ++ks) read_k(slot[1], ks);
    mfma_settle();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s0[i] = pin(s0[i]);
      mx = fmaxf(mx, s0[i]);
    }
    for (int st = 0; st < own; st += 2) {
      step(st, s0, s1);
      if (st + 1 == own) break;
      step(st + 1, s1, s0);
    }
  }
  __builtin_amdgcn_s_setprio(3);
  // The stages that other waves still read.
  for (int st = own; st + 2 < stages; ++st) sync(st);
  mfma_settle();

  // In the masked stages a probability of 0 stood before values that the row does
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
    for (int key = kStageKeys * full + lane / kChunks; key < min(kStageKeys * own, w.len); key += 64 / kChunks) {
      const u32x4 v = *(const u32x4 *)(v0 + (int64_t)key * a.v_stride + 8 * (lane % kChunks));
#pragma unroll
      for (int c = 0; c < 4; ++c) bad |= not_finite2<F16>(v[c]);
    }
    if (own > 0 && __builtin_amdgcn_ballot_w64(bad)) {
      take_rows<D, F16>(a, w, kvh, row0, tok_hi);
      return;
    }
  }
  const f32x2_t both = halves(l_run);
  const float L = both[0] + both[1], inv = L == 0.f ? 0.f : 1.0f / L;
  // Lane (r, h) holds dims 32 db + 8 q + 4 h + i of its row.  Through LDS, in slots that
  // no stage is read from any more (at most the last three are), to whole rows:
  // stores of 8 bytes in each of 32 rows took longer than all of the rest here.
  const uint32_t tile = lds0 + (uint32_t)((stages + wave / 2) % kRing * (2 * kTile) + (wave & 1) * kTile);
#pragma unroll
  for (int db = 0; db < kDims; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u32x2 v;
      v[0] = pack2<F16>(o[db][4 * q] * inv, o[db][4 * q + 1] * inv);
      v[1] = pack2<F16>(o[db][4 * q + 2] * inv, o[db][4 * q + 3] * inv);
      lds_write_b64(tile + (uint32_t)(r * 2 * D + 16 * ((4 * db + q) ^ swizzle_k<D>(r)) + 8 * h), v);
    }
#pragma unroll
  for (int i = 0; i < kWaveRows * kChunks / 64; ++i) {
    const int x = (64 * i + lane) / kChunks, c = lane % kChunks, at = row0 + x, t = quotient(at, G, a.G_magic);
    const u32x4 v = lds_b128(tile + (uint32_t)(x * 2 * D + 16 * (c ^ swizzle_k<D>(x))));
    if (at < rows) *(u32x4 *)(a.out + ((int64_t)(w.start + t) * a.Hq + kvh * G + at - t * G) * D + 8 * c) = v;
  }
}

// Every sequence ends in at most one tile that is not full.  The list has so many entries.
int64_t max_tiles(int N, int G, int S) { return (int64_t)N * G / kTileRows + (S < N ? S : N); }

template <int D, bool F16>
hipError_t launch(GqaPackedArgs a, int cus, hipStream_t s) {
  auto k = gqa_packed_kernel<D, F16>;
  constexpr int lds = kRing * 2 * kStageKeys * D * 2;
  static std::atomic<uint64_t> allowed{0};
  if (const hipError_t e = allow_lds((const void *)k, lds, &allowed)) return e;
  const int64_t tiles = max_tiles(a.N, a.G, a.S);
  int64_t per_xcd = (tiles * a.per_class + (1 << a.class_xcds) - 1) >> a.class_xcds;
  a.xcd_cus = cus / kXcds;  // a second round that is turned round has to be whole
  if (per_xcd > a.xcd_cus && per_xcd < 2 * a.xcd_cus) per_xcd = 2 * a.xcd_cus;
  // Which tile a workgroup takes.  Up to 64 sequences a wave finds that out by itself: in
  // the order of the sequences; with the tiles that see the most keys first, 0.5 to 1 us
  // a workgroup, if CUs have more than one of some length (4 prompts of 900 tokens 47.2, 40.7 us;
  // 32 of 64 10.8, 11.9).  In more rounds than two, and for more sequences, the list,
  // 5 us and a launch (4 prompts of up to 48 tokens 6.5, 9.7 with it; 50 of 300, D = 64,
  // 24.3, 27.8; 64 of 20 to 800 248, 236).
  const bool rounds = per_xcd * kXcds > 2 * kResident<D> * (int64_t)cus;
  a.listed = a.S > kWave || (a.S > 1 && rounds) ? (int)tiles : 0;
  a.searched = !a.listed && a.S > 1 && per_xcd > a.xcd_cus && a.N >= 128 * (int64_t)a.S;
  if (a.listed)
    hipLaunchKernelGGL(a.S <= kPlanLds ? gqa_packed_plan<true> : gqa_packed_plan<false>, dim3(1), dim3(kPlanThreads), 0, s,
                       a);
  hipLaunchKernelGGL(k, dim3((uint32_t)(per_xcd * kXcds)), dim3(64 * kWaves), lds, s, a);
  return hipGetLastError();
}

}  // namespace

void gqa_packed_constants(GqaPackedArgs *a) {
  a->G = a->Hq / a->Hkv;
  a->G_magic = (uint32_t)(((1ull << 32) + a->G - 1) / a->G);
  // KV heads go round 8, 4, 2 or 1 classes of XCDs.
  a->class_xcds = a->Hkv % 8 == 0 ? 0 : a->Hkv % 4 == 0 ? 1 : a->Hkv % 2 == 0 ? 2 : 3;
  a->per_class = a->Hkv >> (3 - a->class_xcds);
}

namespace {
size_t align256(size_t v) { return (v + 255) / 256 * 256; }
}  // namespace

// {status and number of tiles; the tiles; three numbers per sequence}
size_t gqa_packed_workspace(int N, int Hq, int Hkv, int S) {
  return 256 + align256((size_t)max_tiles(N, Hq / Hkv, S) * sizeof(Rows)) + (S <= kPlanLds ? 0 : (size_t)S * 12);
}

void gqa_packed_bind(GqaPackedArgs *a, void *workspace) {
  uint8_t *const w = (uint8_t *)workspace;
  a->status = (uint32_t *)w;
  a->num_tiles = (int32_t *)(w + 128);
  a->tiles = (int32_t *)(w + 256);
  a->tile_sums = (int32_t *)(w + 256 + align256((size_t)max_tiles(a->N, a->Hq / a->Hkv, a->S) * sizeof(Rows)));
}

hipError_t launch_gqa_packed(const GqaPackedArgs &a, int cus, hipStream_t s) {
  const bool f16 = a.dtype == GQA_FP16;
  if (a.D == 128) return f16 ? launch<128, true>(a, cus, s) : launch<128, false>(a, cus, s);
  return f16 ? launch<64, true>(a, cus, s) : launch<64, false>(a, cus, s);
}

}  // namespace moe
