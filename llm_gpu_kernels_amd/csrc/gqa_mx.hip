// Attention of one new token per sequence over a paged cache of microscaled elements, on
// gfx950 (mx_dev.h says what those stand for, gqa_paged.hip has the formula).
//
// The cache's bytes bound it, a half or a quarter of the 16-bit cache's, and next to
// them the conversions: a step of 8 KiB has some 200 vector instructions.  So K and V go
// straight to registers, a whole step ahead of its use, and nothing through LDS:
//   * scores come transposed, S^T = K Q^T; which dims of a row are multiplied together
//     is free as long as K and Q agree, so a lane takes a quarter of a key's row, D/4
//     dims, and their scales;
//   * which dims make a tile of O is free too: a lane takes D/16 neighbouring dims of its
//     eight values' rows;
//   * elements are converted to q's type (exactly where it holds them) by single instructions
//     that apply the scale, and the 16-bit halves of two values are put side by side.
// The work is one flat list of steps, (sequence, KV head, step), cut into equal ranges, one
// per workgroup; in a range its four waves take the steps of a (sequence, head) in turn
// and join their states in LDS where it ends.  A (sequence, head) that a range's end
// cuts leaves its pieces' states in the workspace, and gqa_paged.hip's second launch
// joins them.  Where even a full table is a few steps per wave, a workgroup has a whole
// (sequence, head), and the second launch falls away.
//
// Measured, 32 query and 8 KV heads of 128, a copy of 2 GiB running at 5.1 TB/s, the join
// among it: 64 sequences of 1 to 7027 keys in eight bits (88 MB) 25.5 us, the main kernel
// 20.6 and the join 5.1; one of 131072 in four bits (143 MB) 37.6, 33.0 and 5.3; one of
// 700 in eight bits, a team, 8.7: launch, table, three dependent steps a wave, join in LDS.
// (The join by the last workgroup to arrive, in the same launch: 24.8 and 43.0, and counters
// that have to outlive a run.)
#include <type_traits>

#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"
#include "launch.h"
#include "mx_dev.h"

namespace moe {

using namespace gqa;

namespace {

constexpr int kBlock = 16;   // keys that lie in one page
constexpr int kRows = 16;    // query rows of an MFMA
constexpr int kWindow = 4;   // sequences per lane whose lengths a wave holds
// Workgroups of four waves per CU: 256 registers a lane.  (With three, 168, some spill: one
// sequence of 131072 keys, four bits, 44.3 us, with two 37.4.)
constexpr int kGroups = 2;

// 16-key blocks of a step: a step is 64 bytes of K and of V per lane.
template <int D, int FMT> constexpr int kBlocks = 2 * 128 / mx::row_bytes<FMT>(D);
template <int D, int FMT> constexpr int kStep = kBlock * kBlocks<D, FMT>;

// What a lane holds of a step, for each block: of key r the dims D/4 g.. of K and their
// scale; of the keys 4 g + i the dims D/16 r.. of V, and the four keys' scales there, a
// byte each.
template <int D, int FMT>
struct Raw {
  static constexpr int kKeyWords = mx::row_bytes<FMT>(D) / 16;
  static constexpr int kValueBytes = mx::row_bytes<FMT>(D) / 16, kValueWords = kValueBytes > 4 ? 2 : 1;
  static constexpr int N = kBlocks<D, FMT>;
  uint32_t k[N][kKeyWords], k_scale[N];
  uint32_t v[N][4][kValueWords], v_scales[N];
};
typedef const __attribute__((address_space(1))) uint8_t *Global;
template <int BYTES>
__device__ __forceinline__ void load(Global p, uint32_t off, uint32_t *w) {
  const Global q = p + off;
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int c = 0; c < BYTES / 16; ++c) {
      const u32x4 x = *(const __attribute__((address_space(1))) u32x4 *)(q + 16 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * c + i] = x[i];
    }
  } else if constexpr (BYTES == 8) {
    const u32x2 x = *(const __attribute__((address_space(1))) u32x2 *)q;
    w[0] = x[0];
    w[1] = x[1];
  } else if constexpr (BYTES == 4) {
    w[0] = *(const __attribute__((address_space(1))) uint32_t *)q;
  } else if constexpr (BYTES == 2) {
    w[0] = *(const __attribute__((address_space(1))) uint16_t *)q;
  } else {
    w[0] = *q;
  }
}

// A (sequence, head block)'s steps s to e of a workgroup's range; KV head and block of
// up to 16 of its query heads; where the pair's places in the list begin.
struct Segment {
  int b, kvh, part, len, steps, base, s, e;
};
// Places of a pair in the list besides its steps: what its start and end cost, in steps
// of a wave.
// (64 sequences of 1 to 7027 keys, eight bits: with 2 34.6 us, 6 25.7, 12 26.6; without, 78.)
constexpr int kOverhead = 6;

// Steps that a wave of a workgroup with a whole (sequence, head) may have, by those that the
// list would give it.  A team has one launch and nothing to join, but all of its sequence.
// By teams and by the list, 8 KV heads of 128, eight bits: one sequence of 128 keys 4.4,
// 10.0 us; of 700 8.7, 10.5; of 1500 13.2, 11.2; of 2048 16.0, 11.4; 16 of 512 7.8, 13.3; of 2048
// 17.3, 20.5; of 4096 35.5, 35.4; 64 of 700 19.6, 22.0; of 2048 52.4, 55.1; 256 of 1 to 1024 27.9,
// 33.8.  Four bits (steps of 64 keys): one of 1500 9.9, 11.1; of 2048 11.8, 11.6; 16 of 2048
// 13.6, 18.1; of 4096 22.5, 23.4.
__host__ __device__ inline int most_teamed(int64_t listed) { return listed >= 8 ? 17 : 2 * (int)listed + 2; }

// What the host divides for the kernel: query heads per KV head, blocks of up to 16 of them, and
// the logarithm of a page's blocks of keys (-1: not a power of two).
struct Shape {
  int group, blocks, page_shift;
};

// LISTED: ranges of the list; otherwise a (sequence, head block) per workgroup, of a grid
// (block of query heads, KV head, sequence).  TEAM waves.
//
// A call with a few steps is as long as its first pass over the code, whose instructions come
// from the L2: what a team does not need is not compiled into it, and its arguments are read
// at once, not line by line where they are used (700 keys 9.2 to 8.7 us, 128 5.4 to 4.4).
template <int D, bool F16, int FMT, int TEAM, bool LISTED>
__global__ __launch_bounds__(64 * TEAM, (TEAM == 8 ? 2 : kGroups)) void gqa_mx_kernel(GqaPagedArgs a, Shape shape) {
  constexpr int kSlices = D / 32, kTiles = D / 16;
  constexpr int kN = kBlocks<D, FMT>, kKeys = kStep<D, FMT>;
  constexpr uint32_t kRowBytes = (uint32_t)mx::row_bytes<FMT>(D);
  using R = Raw<D, FMT>;
  extern __shared__ __attribute__((aligned(16))) float states[];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = sgpr(threadIdx.x >> 6);
  if constexpr (!LISTED)
    asm volatile("" ::"s"(a.q), "s"(a.k), "s"(a.v), "s"(a.out), "s"(a.tables), "s"(a.lengths), "s"(a.k_page), "s"(a.k_head),
                 "s"(a.v_page), "s"(a.v_head), "s"(a.M), "s"(a.scale), "s"(a.k_scales), "s"(a.ks_page), "s"(a.vs_page),
                 "s"(shape.group));
  const int group = shape.group, blocks = shape.blocks, heads = a.Hkv * blocks;
  const int cap = a.M * a.page;
  auto steps_of = [](int keys) __attribute__((always_inline)) { return (int)(((uint32_t)keys + kKeys - 1) / kKeys); };

  // ---- the workgroup's range, and its first segment ----
  int window = 0, lens[kWindow];
  auto load_lengths = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kWindow; ++i) {
      const int at = window + kWave * i + lane;
      lens[i] = at < a.B ? a.lengths[at] : 0;
    }
#pragma unroll
    for (int i = 0; i < kWindow; ++i) {
      const int ok = max(0, min(lens[i], cap));
      if (lens[i] != ok) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
      lens[i] = ok;
    }
  };
  Segment seg;
  int per = 1, end = 0;  // places of a range; the end of this one
  bool paired = !LISTED;
  // Places of a sequence's heads in the list.
  auto places_of = [&](int keys) __attribute__((always_inline)) { return keys > 0 ? (steps_of(keys) + kOverhead) * heads : 0; };
  // The steps of the pair x that lie in places `from` to `end`.
  auto cut = [&](Segment &x, int from) __attribute__((always_inline)) {
    x.s = min(max(0, from - x.base - kOverhead), x.steps);
    x.e = max(x.s, min(x.steps, end - x.base - kOverhead));
  };
  if constexpr (LISTED) {
    int sum = 0, most = 0;
    for (;; window += kWave * kWindow) {
      load_lengths();
#pragma unroll
      for (int i = 0; i < kWindow; ++i) {
        sum += places_of(lens[i]);
        most = max(most, steps_of(lens[i]));
      }
      if (window + kWave * kWindow >= a.B) break;
    }
    const int all = wave_total(sum);  // < 2^31, checked on the host
    per = (all + gridDim.x - 1) / gridDim.x;
    paired = a.B * heads <= (int)gridDim.x &&
             !__builtin_amdgcn_ballot_w64(most > TEAM * most_teamed((per + TEAM - 1) / TEAM));
    if (!paired) {
      if ((int64_t)blockIdx.x * per >= all) return;
      const int first = blockIdx.x * per;
      end = min(all, first + per);
      if (window > 0) {
        window = 0;
        load_lengths();
      }
      int before = 0, b = -1, len = 0;
      while (b < 0) {
#pragma unroll
        for (int i = 0; i < kWindow; ++i) {
          const int incl = before + wave_scan(places_of(lens[i]));
          const uint64_t past = __builtin_amdgcn_ballot_w64(incl > first);
          if (b < 0) {
            if (past) {
              const int at = sgpr(__builtin_ctzll(past));
              b = window + kWave * i + at;
              len = __builtin_amdgcn_readlane(lens[i], at);
              before = __builtin_amdgcn_readlane(incl, at) - places_of(len);
            } else {
              before = __builtin_amdgcn_readlane(incl, 63);
            }
          }
        }
        if (b < 0) {
          window += kWave * kWindow;
          if (window >= a.B) return;  // only if lengths change meanwhile
          load_lengths();
        }
      }
      const int steps = steps_of(len), head = (first - before) / (steps + kOverhead);
      seg = Segment{b, head / blocks, head % blocks, len, steps, before + head * (steps + kOverhead), 0, 0};
      cut(seg, first);
    }
  }
  if (paired) {
    if (LISTED && (int)blockIdx.x >= a.B * heads) return;
    const int b = LISTED ? blockIdx.x / heads : blockIdx.z, head = blockIdx.x - b * heads;
    const int kvh = LISTED ? head / blocks : blockIdx.y, part = LISTED ? head - kvh * blocks : blockIdx.x;
    const int raw = a.lengths[b], len = sgpr(max(0, min(raw, cap)));
    if (raw != len && threadIdx.x == 0) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
    seg = Segment{b, kvh, part, len, steps_of(len), 0, 0, steps_of(len)};
    // For the launch that joins the list's pieces: nothing to do here.
    if (LISTED && threadIdx.x == 0) a.pieces[2 * blockIdx.x + 1] = 0;
  }
  // The segment behind one; none: e = s.
  auto next_segment = [&](const Segment &x) __attribute__((always_inline)) {
    Segment y = x;
    y.s = y.e = 0;
    y.base = x.base + x.steps + kOverhead;
    if (paired || y.base + kOverhead >= end) return y;
    if (++y.part == blocks) {
      y.part = 0;
      if (++y.kvh == a.Hkv) {
        y.kvh = 0;
        int found = -1;
        for (;;) {
#pragma unroll
          for (int i = 0; i < kWindow; ++i) {
            const int lo = max(0, x.b + 1 - window - kWave * i);
            const uint64_t some = __builtin_amdgcn_ballot_w64(lens[i] > 0);
            const uint64_t later = lo < kWave ? some >> lo << lo : 0ull;
            if (found < 0 && later) {
              const int at = sgpr(__builtin_ctzll(later));
              found = window + kWave * i + at;
              y.len = __builtin_amdgcn_readlane(lens[i], at);
            }
          }
          if (found >= 0) break;
          window += kWave * kWindow;
          if (window >= a.B) return y;  // only if lengths change meanwhile
          load_lengths();
        }
        y.b = found;
        y.steps = steps_of(y.len);
      }
    }
    cut(y, y.base);
    return y;
  };
  if (!paired && seg.e == seg.s) {  // the range begins behind a pair's last step
    seg = next_segment(seg);
    if (seg.e == seg.s) return;
  }

  // ---- loads ----
  const uint32_t k_off = (uint32_t)r * kRowBytes + (uint32_t)g * (kRowBytes / 4);
  const uint32_t v_off = (uint32_t)(4 * g) * kRowBytes + (uint32_t)r * R::kValueBytes;
  const uint32_t ks_off = (uint32_t)(g * (D / 4) / mx::kBlock * a.page + r);
  const uint32_t vs_off = (uint32_t)(r * (D / 16) / mx::kBlock * a.page + 4 * g);
  bool bad_page = false;
  // Pages and rows of the blocks of the wave's next kSteps steps of a segment, from step
  // t on: lane l has block l % kN of its step l / kN.  A page that is not there: row -1.
  constexpr int kSteps = kWave / kN;
  struct Window {
    int page, row;
  };
  auto look_up = [&](const Segment &x, int t) __attribute__((always_inline)) {
    const int blk = kN * (t + TEAM * (lane / kN)) + lane % kN;
    const int at = __builtin_expect(shape.page_shift >= 0, 1) ? blk >> shape.page_shift : blk / (a.page / kBlock);
    const bool in = (uint32_t)(kBlock * blk) < (uint32_t)x.len;  // (a window may go past 2^31 keys)
    const int page = in ? a.tables[(int64_t)x.b * a.table_stride + at] : 0;
    const bool ok = (uint32_t)page < (uint32_t)a.P;
    bad_page |= !ok;
    return Window{ok ? page : 0, in && ok ? blk * kBlock - at * a.page : -1};
  };
  // The nth step of a window, step t of the segment: the keys of its blocks that are there
  // (a byte each) into n, what they hold into raw.  Blocks that are not there are read from
  // page 0.
  auto issue = [&](const Segment &x, int t, const Window &win, int nth, R &raw, uint64_t &n) __attribute__((always_inline)) {
    const Global k = (Global)a.k + x.kvh * a.k_head, v = (Global)a.v + x.kvh * a.v_head;
    const Global ks = (Global)a.k_scales + x.kvh * a.ks_head, vs = (Global)a.v_scales + x.kvh * a.vs_head;
    n = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const uint32_t page = __builtin_amdgcn_readlane(win.page, kN * nth + i);
      const int there = __builtin_amdgcn_readlane(win.row, kN * nth + i);
      const uint32_t row = (uint32_t)max(there, 0);
      n |= (uint64_t)(there < 0 ? 0 : min(kBlock, x.len - kBlock * (kN * t + i))) << 8 * i;
      const Global kp = k + ((uint64_t)page * (uint32_t)a.k_page + row * kRowBytes);
      const Global vp = v + ((uint64_t)page * (uint32_t)a.v_page + row * kRowBytes);
      load<R::kKeyWords * 4>(kp, k_off, raw.k[i]);
      load<1>(ks + ((uint64_t)page * (uint32_t)a.ks_page + row), ks_off, &raw.k_scale[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) load<R::kValueBytes>(vp, v_off + j * kRowBytes, raw.v[i][j]);
      load<4>(vs + ((uint64_t)page * (uint32_t)a.vs_page + row), vs_off, &raw.v_scales[i]);
    }
  };
  u32x4 qf[kSlices];
  auto issue_q = [&](const Segment &x) __attribute__((always_inline)) {
    const int rows = min(kRows, group - kRows * x.part);
    const uint16_t *const base = a.q + x.b * a.q_stride + (int64_t)(x.kvh * group + kRows * x.part) * D;
    const auto rs = buffer(base, (uint32_t)rows * 2 * D);  // rows that are not there are 0
#pragma unroll
    for (int ks = 0; ks < kSlices; ++ks)
      qf[ks] = __builtin_amdgcn_raw_buffer_load_b128(rs, (uint32_t)(r * 2 * D + g * (D / 2) + 16 * ks), 0, 0);
  };

  // Softmax state of query row r (this lane's keys only in l), base-2 domain; O: rows
  // 4 g + i, dims kTiles r + dt.
  float m_run, l_run, m_top;
  f32x4 o[kTiles];
  const float sl2 = a.scale * kLog2e;

  auto compute = [&](R &raw, uint64_t n) __attribute__((always_inline)) {
    f32x4 sc[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float scale = mx::scale_of(raw.k_scale[i]);
      sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < kSlices; ++ks) {
        u32x4 kf;
        if constexpr (FMT == mx::kFp8) kf = mx::decode8<FMT, F16>(raw.k[i][2 * ks], raw.k[i][2 * ks + 1], scale);
        else kf = mx::decode8<FMT, F16>(raw.k[i][ks], 0u, scale);
        sc[i] = mfma16x16<F16>(kf, qf[ks], sc[i]);
      }
    }
    mfma_settle();  // read on both sides of a branch
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[i][j] = pin(sc[i][j]);
    if (n != (0x1010101010101010ull & (kN == 8 ? ~0ull : (1ull << 8 * (kN % 8)) - 1))) {
      // Keys that are not there: no score, and values of 0 under a scale of 0, whatever the
      // page holds.  Lane: keys 4 g + j of a block.
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int keys = min(max((int)(n >> 8 * i & 0xff) - 4 * g, 0), 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sc[i][j] = j < keys ? sc[i][j] : -INFINITY;
#pragma unroll
          for (int w = 0; w < R::kValueWords; ++w) raw.v[i][j][w] = j < keys ? raw.v[i][j][w] : 0u;
        }
        raw.v_scales[i] &= keys == 4 ? ~0u : (1u << 8 * keys) - 1u;
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kN; ++i) top = fmaxf(top, fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])));
    top *= sl2;
    if (__builtin_amdgcn_ballot_w64(top > (F16 ? m_top : limit<F16>(m_run)))) {
      mfma_settle();
      const float m_new = fmaxf(m_run, reference<F16>(quad_max(top)));
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
      l_run *= alpha;
      m_run = m_new;
      m_top = limit<F16>(m_new);
      float al[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) al[i] = __shfl(alpha, 4 * g + i, kWave);
#pragma unroll
      for (int dt = 0; dt < kTiles; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[dt][i] = pin(o[dt][i]) * al[i];
    }
    const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
    for (int hh = 0; hh < kN / 2; ++hh) {
      float p[2][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * hh + kt][i], sl2, neg_m));
      l_run += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
      // Probabilities in q's type, which the matrix instructions multiply: half a step each, see
      // reference(), against fp32 sums of both.  Against 64 bits a bf16 output is then off by
      // 0.0023 of its rms, by its own last rounding alone 0.0017.  As two 16-bit numbers each (cut
      // off and the rest, both multiplied) it was off by 0.0017: 700 keys 8.9 to 9.2 us, 64 ragged
      // sequences 25.8 to 26.8, 131072 keys in four bits 36.5 to 37.9, 16 of 4096 23.3 to 25.8, and
      // fp16 with heads of 64 27.9 to 30.8.  Not kept: the 16-bit cache's attention, which this
      // stands beside, rounds them too, and the elements have four bits or two.
      const u32x4 pa = {pack2<F16>(p[0][0], p[0][1]), pack2<F16>(p[0][2], p[0][3]), pack2<F16>(p[1][0], p[1][1]),
                        pack2<F16>(p[1][2], p[1][3])};
      float scale[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) scale[i][j] = mx::scale_of(raw.v_scales[2 * hh + i] >> 8 * j & 0xffu);
      // Two tiles at a time: dims 2 P and 2 P + 1 of the lane's eight keys, two keys of a
      // dim side by side.
      auto tiles = [&](auto pair) __attribute__((always_inline)) {
        constexpr int P = decltype(pair)::value;
        u32x4 even, odd;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t x[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t(&v)[R::kValueWords] = raw.v[2 * hh + i][2 * j + e];
              if constexpr (FMT == mx::kFp8) x[e] = mx::decode2<FMT, F16, P & 1>(v[P / 2], scale[i][2 * j + e]);
              else x[e] = mx::decode2<FMT, F16, P>(v[0], scale[i][2 * j + e]);
            }
            even[2 * i + j] = __builtin_amdgcn_perm(x[1], x[0], 0x05040100u);
            odd[2 * i + j] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
          }
        o[2 * P] = mfma16x16<F16>(pa, even, o[2 * P]);
        o[2 * P + 1] = mfma16x16<F16>(pa, odd, o[2 * P + 1]);
      };
      tiles(std::integral_constant<int, 0>());
      tiles(std::integral_constant<int, 1>());
      if constexpr (D == 128) {
        tiles(std::integral_constant<int, 2>());
        tiles(std::integral_constant<int, 3>());
      }
    }
  };

  // ---- the segments ----
  R cur, nxt;
  uint64_t n_cur = 0, n_nxt = 0;
  bool ahead = false;  // cur holds the wave's first step of the segment
  Window win = look_up(seg, seg.s + wave), win_next = {};
  issue_q(seg);
  const int rows_most = min(group, kRows), stride = rows_most * D + 2 * kRows;  // floats of a wave's state
  for (int nth = 0;; ++nth) {
    Segment next = seg;
    next.s = next.e = 0;
    if constexpr (LISTED) {
      next = next_segment(seg);
      win_next = look_up(next, next.s + wave);
    }
    m_run = m_top = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int dt = 0; dt < kTiles; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    int t = seg.s + wave, in_window = 0;
    if (!ahead && t < seg.e) issue(seg, t, win, 0, cur, n_cur);
    ahead = false;
    for (; t < seg.e; t += TEAM) {
      const bool more = t + TEAM < seg.e;
      ahead = !more && next.s + wave < next.e;
      if (more || ahead) {
        Segment x = seg;
        x.kvh = more ? seg.kvh : next.kvh;
        x.len = more ? seg.len : next.len;
        if (more && ++in_window == kSteps) {
          in_window = 0;
          win = look_up(seg, t + TEAM);
        }
        const Window w = {more ? win.page : win_next.page, more ? win.row : win_next.row};
        issue(x, more ? t + TEAM : next.s + wave, w, more ? in_window : 0, nxt, n_nxt);
      }
      __builtin_amdgcn_sched_barrier(0);  // the loads go out before what follows
      compute(cur, n_cur);
      cur = nxt;
      n_cur = n_nxt;
    }
    win = win_next;
    const bool last = next.e == next.s;
    if (!last) issue_q(next);

    // The waves' states, each in its own part of the LDS: O, then m and l per row.
    const int kvh = seg.kvh, part = seg.part, rows = min(kRows, group - kRows * part);
    const float l = quad_sum(l_run);
    float *const mine = states + wave * stride;
    mfma_settle();
    if (g == 0) {
      mine[rows_most * D + r] = m_run;
      mine[rows_most * D + kRows + r] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * g + i < rows) {
#pragma unroll
        for (int dt = 0; dt < kTiles; dt += 4)
          *(f32x4 *)(mine + (4 * g + i) * D + kTiles * r + dt) =
              f32x4{pin(o[dt][i]), pin(o[dt + 1][i]), pin(o[dt + 2][i]), pin(o[dt + 3][i])};
      }
    __syncthreads();
    const bool whole = seg.s == 0 && seg.e == seg.steps;
    const int slot = 2 * (int)blockIdx.x + (nth ? 1 : 0);
    if (!paired && seg.s == 0 && threadIdx.x == 0) {
      // Pieces: this one, then the first pieces of the following workgroups.
      const int at = 2 * (seg.b * heads + kvh * blocks + part);
      a.pieces[at] = slot;
      a.pieces[at + 1] = whole ? 0 : (seg.base + kOverhead + seg.steps - 1) / per - (int)blockIdx.x + 1;
    }
    const int64_t row0 = (int64_t)seg.b * a.Hq + kvh * group + kRows * part;
    for (int e = 2 * threadIdx.x; e < rows * D; e += 2 * 64 * TEAM) {
      const int row = e / D;
      float m[TEAM], high = -INFINITY, den = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) {
        m[w] = states[w * stride + rows_most * D + row];
        high = fmaxf(high, m[w]);
      }
      const float ref = high == -INFINITY ? 0.f : high;
#pragma unroll
      for (int w = 0; w < TEAM; ++w) {
        const float *const x = states + w * stride;
        const float f = __builtin_amdgcn_exp2f(m[w] - ref);
        const f32x2_t v = *(const f32x2_t *)(x + e);
        den = __builtin_fmaf(f, x[rows_most * D + kRows + row], den);
        o0 = __builtin_fmaf(f, v[0], o0);
        o1 = __builtin_fmaf(f, v[1], o1);
      }
      if (whole) {
        const float inv = den == 0.f ? 0.f : 1.0f / den;
        ((uint32_t *)(a.out + row0 * D))[e / 2] = pack2<F16>(o0 * inv, o1 * inv);
      } else {
        float *const to = a.partial + ((int64_t)slot * rows_most + row) * (D + 2);
        if (e % D == 0) *(f32x2_t *)to = f32x2_t{high, den};
        *(f32x2_t *)(to + 2 + e % D) = f32x2_t{o0, o1};
      }
    }
    if (last) break;
    __syncthreads();  // the states have been read
    seg = next;
  }
  if (__builtin_amdgcn_ballot_w64(bad_page) && lane == 0) atomicOr(a.status, GQA_STATUS_BAD_PAGE);
}

// Waves of a workgroup per (sequence, head block), or 0 for the list and its merge, by the
// steps of a full table.
int team_of(int64_t pairs, int64_t steps, int cus) {
  const int64_t waves = (int64_t)cus * kGroups * 4;
  const int team = 8 * pairs <= waves ? 8 : 4;
  const int64_t listed = (pairs * steps + waves - 1) / waves, teamed = (steps + team - 1) / team;
  return teamed <= most_teamed(listed) ? team : 0;
}

int step_keys(int D, int storage) {
  if (storage == GQA_STORAGE_MXFP8) return D == 128 ? kStep<128, mx::kFp8> : kStep<64, mx::kFp8>;
  return D == 128 ? kStep<128, mx::kFp4> : kStep<64, mx::kFp4>;
}

template <int D, bool F16, int FMT>
hipError_t launch(const GqaPagedArgs &a, int cus, hipStream_t s) {
  const int group = a.Hq / a.Hkv, rows = group < kRows ? group : kRows, pairs = a.B * a.Hkv * ((group + kRows - 1) / kRows);
  const int team = team_of(pairs, ((int64_t)a.M * a.page + kStep<D, FMT> - 1) / kStep<D, FMT>, cus);
  const int blocks = (group + kRows - 1) / kRows, per_page = a.page / kBlock;
  const Shape shape = {group, blocks, per_page & (per_page - 1) ? -1 : __builtin_ctz(per_page)};
  const int lds = (team == 8 ? 8 : 4) * (rows * D + 2 * kRows) * (int)sizeof(float);  // at most 66 KiB
  if (team == 8) {
    auto wide = gqa_mx_kernel<D, F16, FMT, 8, false>;
    static std::atomic<uint64_t> allowed{0};
    if (const hipError_t e = allow_lds((const void *)wide, 8 * (kRows * D + 2 * kRows) * (int)sizeof(float), &allowed)) return e;
    hipLaunchKernelGGL(wide, dim3(blocks, a.Hkv, a.B), dim3(512), lds, s, a, shape);
    return hipGetLastError();
  }
  if (team == 4) {
    hipLaunchKernelGGL((gqa_mx_kernel<D, F16, FMT, 4, false>), dim3(blocks, a.Hkv, a.B), dim3(256), lds, s, a, shape);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((gqa_mx_kernel<D, F16, FMT, 4, true>), dim3(cus * kGroups), dim3(256), lds, s, a, shape);
  if (const hipError_t e = hipGetLastError()) return e;
  return launch_gqa_paged_merge(a, cus, s);
}

template <int D, bool F16>
hipError_t launch(const GqaPagedArgs &a, int cus, hipStream_t s) {
  return a.storage == GQA_STORAGE_MXFP8 ? launch<D, F16, mx::kFp8>(a, cus, s) : launch<D, F16, mx::kFp4>(a, cus, s);
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

// As gqa_paged_workspace(): {status words; two words per (sequence, head block); two
// pieces' states per workgroup of the list}.
size_t gqa_mx_workspace(int B, int Hq, int Hkv, int D, int storage, int64_t keys, int cus) {
  const int group = Hq / Hkv, rows = group < kRows ? group : kRows, step = step_keys(D, storage);
  const size_t pairs = (size_t)B * Hkv * ((group + kRows - 1) / kRows);
  if (team_of(pairs, (keys + step - 1) / step, cus)) return 256;
  return 256 + align256(8 * pairs) + (size_t)2 * cus * kGroups * rows * (D + 2) * sizeof(float);
}

hipError_t launch_gqa_mx(const GqaPagedArgs &a, int cus, hipStream_t s) {
  if (a.D == 128) return a.dtype == GQA_FP16 ? launch<128, true>(a, cus, s) : launch<128, false>(a, cus, s);
  return a.dtype == GQA_FP16 ? launch<64, true>(a, cus, s) : launch<64, false>(a, cus, s);
}

}  // namespace moe
