// Attention of one new token per sequence over a paged cache on gfx950.
//
//   out[b][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b][h] . k_j - max),
//   over the lengths[b] keys of row b; head h reads KV head h / (Hq / Hkv).
//
// Every K and V byte is used by one KV head's queries only (at most 16 rows of
// an MFMA), so the cache's bytes bound it, and what counts is that every wave
// has loads in flight all the time and that all of them end together:
//   * the work is one flat list of 32-key steps, (sequence, KV head, step), cut
//     into equal ranges, one per wave of a grid that fills the chip once.  Waves
//     work for themselves (no barrier): a wave's next step is loaded while the
//     present one computes, across the ends of sequences too;
//   * a wave's range may end inside a (sequence, head).  Such pieces leave their
//     (max, sum, O) in the workspace and a second launch joins them in the order
//     of the keys; whole ones are written at once;
//   * where even a full table is a few steps per wave, a workgroup takes a
//     (sequence, head) instead, its waves' states are joined in LDS, and the second
//     launch falls away (team_of() has the rule).  Where the table is wider than
//     that but the lengths are not, the kernel finds out from the lengths and does
//     the same, and the second launch has nothing to do;
//   * K and V rows go from HBM to LDS in whole rows (buffer loads with an LDS
//     destination, a descriptor per 16-key block: a block lies in one page),
//     permuted within a row so that the operand reads have no bank conflicts.
// Scores are computed transposed, S^T = K Q^T, so they land in the A layout of
// the P.V product; V comes back transposed with ds_read_b64_tr_b16.
//
// Measured, a copy of 2 GiB running at 5.0 TB/s: one sequence of 131072 tokens, 8 KV heads
// of 128 (537 MB), 96 us, 5.6 TB/s, and 6.4 us for the join; 64 sequences of 1 to 7787 (288
// MB), 68 us with the join; by teams, 200 sequences of 16 to 1997, 2 KV heads of 64 (39
// MB), 14.6 us, and one of 700, 8 heads of 128, 8.1 us: launch, table, keys, join.
#include <type_traits>

#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"
#include "launch.h"

namespace moe {

using namespace gqa;

namespace {

constexpr int kStep = 32;       // keys of a step
constexpr int kBlock = 16;      // keys that lie in one page
constexpr int kRows = 16;       // query rows of an MFMA
constexpr int kWaves = 4;       // per workgroup; only the LDS is shared out by it
constexpr int kWindow = 4;      // sequences per lane whose lengths a wave holds

// LDS of a wave: 32 rows of K, 32 of V, 16 of Q.  Row i's 16-byte chunk c lies
// at place c ^ swizzle(i) of its row: the sixteen lanes that read one chunk of
// sixteen K rows, and the sixteen that read two chunks of four V rows, meet
// sixteen (eight) different bank groups.
template <int D> constexpr int kStage = kStep * D * 2;
template <int D> constexpr int kWaveLds = 5 * kStage<D> / 2;
template <int D> constexpr int kWorkgroups = 160 * 1024 / (kWaves * kWaveLds<D>);  // per CU
template <int D>
__device__ __forceinline__ int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swizzle_v(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

// K fragments (key block kt, 32-dim slice ks) -> k[2 ks + kt], and Q's.
template <int D>
__device__ __forceinline__ void read_kq(uint32_t base, const uint32_t (&at)[D / 32], u32x4 (&k)[D / 16], u32x4 (&q)[D / 32]) {
  if constexpr (D == 128) {
    asm volatile(
        "ds_read_b128 %0, %12\n\t"
        "ds_read_b128 %8, %12 offset:16384\n\t"
        "ds_read_b128 %1, %12 offset:4096\n\t"
        "ds_read_b128 %2, %13\n\t"
        "ds_read_b128 %9, %13 offset:16384\n\t"
        "ds_read_b128 %3, %13 offset:4096\n\t"
        "ds_read_b128 %4, %14\n\t"
        "ds_read_b128 %10, %14 offset:16384\n\t"
        "ds_read_b128 %5, %14 offset:4096\n\t"
        "ds_read_b128 %6, %15\n\t"
        "ds_read_b128 %11, %15 offset:16384\n\t"
        "ds_read_b128 %7, %15 offset:4096\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(k[4]), "=&v"(k[5]), "=&v"(k[6]), "=&v"(k[7]),
          "=&v"(q[0]), "=&v"(q[1]), "=&v"(q[2]), "=&v"(q[3])
        : "v"(base + at[0]), "v"(base + at[1]), "v"(base + at[2]), "v"(base + at[3])
        : "memory");
  } else {
    asm volatile(
        "ds_read_b128 %0, %6\n\t"
        "ds_read_b128 %4, %6 offset:8192\n\t"
        "ds_read_b128 %1, %6 offset:2048\n\t"
        "ds_read_b128 %2, %7\n\t"
        "ds_read_b128 %5, %7 offset:8192\n\t"
        "ds_read_b128 %3, %7 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3]), "=&v"(q[0]), "=&v"(q[1])
        : "v"(base + at[0]), "v"(base + at[1])
        : "memory");
  }
}
// V of 16 dims dt and the lane group's keys 4 g + 0..3 -> v[2 dt], keys 16
// further -> v[2 dt + 1].  ds_read_b64_tr_b16: within 16 lanes, lane 4 a + b
// receives element b of the 8-byte rows addressed by lanes a, a + 4, a + 8, a + 12.
template <int D>
__device__ __forceinline__ void read_v(uint32_t base, u32x2 (&v)[D / 8]) {
  const uint32_t a0 = base, a1 = base ^ 32, a2 = base ^ 64, a3 = base ^ 96;
  if constexpr (D == 128) {
    const uint32_t a4 = base ^ 128, a5 = base ^ 160, a6 = base ^ 192, a7 = base ^ 224;
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16\n\t"
        "ds_read_b64_tr_b16 %1, %16 offset:4096\n\t"
        "ds_read_b64_tr_b16 %2, %17\n\t"
        "ds_read_b64_tr_b16 %3, %17 offset:4096\n\t"
        "ds_read_b64_tr_b16 %4, %18\n\t"
        "ds_read_b64_tr_b16 %5, %18 offset:4096\n\t"
        "ds_read_b64_tr_b16 %6, %19\n\t"
        "ds_read_b64_tr_b16 %7, %19 offset:4096\n\t"
        "ds_read_b64_tr_b16 %8, %20\n\t"
        "ds_read_b64_tr_b16 %9, %20 offset:4096\n\t"
        "ds_read_b64_tr_b16 %10, %21\n\t"
        "ds_read_b64_tr_b16 %11, %21 offset:4096\n\t"
        "ds_read_b64_tr_b16 %12, %22\n\t"
        "ds_read_b64_tr_b16 %13, %22 offset:4096\n\t"
        "ds_read_b64_tr_b16 %14, %23\n\t"
        "ds_read_b64_tr_b16 %15, %23 offset:4096\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]),
          "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]), "=&v"(v[14]), "=&v"(v[15])
        : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "v"(a4), "v"(a5), "v"(a6), "v"(a7)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %9\n\t"
        "ds_read_b64_tr_b16 %3, %9 offset:2048\n\t"
        "ds_read_b64_tr_b16 %4, %10\n\t"
        "ds_read_b64_tr_b16 %5, %10 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %11\n\t"
        "ds_read_b64_tr_b16 %7, %11 offset:2048\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
        : "v"(a0), "v"(a1), "v"(a2), "v"(a3)
        : "memory");
  }
}

// Read by scalar loads: the tables do not change while the kernel runs.
__device__ __forceinline__ int uniform_load(const int32_t *p) {
  return *(const __attribute__((address_space(4))) int32_t *)(const __attribute__((address_space(4))) void *)p;
}

// A step: up to 32 keys of one (sequence, head block).  All fields are the same
// in every lane.
struct Step {
  int b, head;       // sequence, block of up to 16 query heads
  int s, steps;      // number among the steps of its (sequence, head block)
  int page[2], row[2], n[2];  // its 16-key blocks: page, first row, keys (0: none)
};

// The most steps of a wave with which teams are faster than the list, by those that
// the list gives it (team_of() has figures).
__host__ __device__ inline int most_teamed(int64_t listed) { return listed >= 20 ? 16 : (int)listed / 2 + 6; }

// TEAM > 0: a workgroup of TEAM waves per (sequence, head block), each taking every
// TEAM-th step, whose states are joined in LDS at the end.  TEAM 0: a range of the
// flat list per wave, or teams of the workgroups' waves if the lengths make those
// faster and one grid has a workgroup for every pair, of rows of length 0 too
// (tables of 8192 keys, 8 heads of 128: 64 sequences of 128 keys 14.5 us by the list,
// 9.3 so, 16 of 500 13.7, 10.1, 64 of 1000 48.4, 41.6; what the list loses by
// looking is 0.3 us).
template <int D, bool F16, int TEAM>
__global__ __launch_bounds__(64 * (TEAM ? TEAM : kWaves), TEAM == 8 ? 1 : kWorkgroups<D>)
void gqa_paged_kernel(GqaPagedArgs a) {
  constexpr int kSlices = D / 32;               // 32-dim slices of a row
  constexpr int kTiles = D / 16;                // 16-dim tiles of O
  constexpr int kLoads = kBlock * D * 2 / 1024; // loads of a block
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = sgpr(threadIdx.x >> 6);
  const int worker = sgpr(wave * gridDim.x + blockIdx.x), workers = gridDim.x * kWaves;  // few steps: on many CUs
  constexpr int kTeam = TEAM ? TEAM : kWaves;
  const int group = a.Hq / a.Hkv, blocks = (group + kRows - 1) / kRows, heads = a.Hkv * blocks;
  const int cap = a.M * a.page;
  uint8_t *const kst = smem + wave * kWaveLds<D>, *const vst = kst + kStage<D>, *const qst = vst + kStage<D>;

  // ---- the wave's range of the flat list, or its first step ----
  // (Unsigned: lengths go up to 2^31 - 16.)
  auto steps_of = [](int keys) __attribute__((always_inline)) { return (int)(((uint32_t)keys + kStep - 1) / kStep); };
  // Lengths of 64 kWindow sequences from `window` on: i-th of a lane at 64 i + lane.
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
  int b = -1, len = 0, head, s;           // of the next step, with its sequence's length
  int steps, left;                        // of its (sequence, head block), of the wave
  int all = 0, per = 1, first = 0;        // steps, those of a wave, the wave's first in the list
  bool team = TEAM > 0;
  if constexpr (TEAM == 0) {
    int sum = 0, most = 0;
    for (;; window += kWave * kWindow) {
      load_lengths();
#pragma unroll
      for (int i = 0; i < kWindow; ++i) {
        sum += steps_of(lens[i]);
        most = max(most, steps_of(lens[i]));
      }
      if (window + kWave * kWindow >= a.B) break;
    }
    all = wave_total(sum) * heads;                          // < 2^31, checked on the host
    per = (all + workers - 1) / workers;
    team = a.B * heads <= (int)gridDim.x && !__builtin_amdgcn_ballot_w64(most > kTeam * most_teamed(per));
  }
  if (!team) {
    if ((int64_t)worker * per >= all) return;
    first = worker * per;
    left = min(per, all - first);
    if (window > 0) {
      window = 0;
      load_lengths();
    }
    // The sequence where the range begins, and the steps before it.
    int before = 0;
    while (b < 0) {
#pragma unroll
      for (int i = 0; i < kWindow; ++i) {
        const int incl = before + wave_scan(steps_of(lens[i]) * heads);
        const uint64_t past = __builtin_amdgcn_ballot_w64(incl > first);
        if (b < 0) {
          if (past) {
            const int at = sgpr(__builtin_ctzll(past));
            b = window + kWave * i + at;
            len = __builtin_amdgcn_readlane(lens[i], at);
            before = __builtin_amdgcn_readlane(incl, at) - steps_of(len) * heads;
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
    steps = steps_of(len);
    const int rest = first - before;
    head = rest / steps;
    s = rest % steps;
  } else {
    if ((int)blockIdx.x >= a.B * heads) return;
    b = blockIdx.x / heads;
    head = blockIdx.x % heads;
    const int raw = a.lengths[b];
    len = sgpr(max(0, min(raw, cap)));
    if (raw != len && threadIdx.x == 0) atomicOr(a.status, GQA_STATUS_BAD_BOUNDS);
    steps = steps_of(len);
    s = wave;
    left = s < steps ? (steps - s + kTeam - 1) / kTeam : 0;
    // For the launch that joins the list's pieces: nothing to do here.
    if (TEAM == 0 && threadIdx.x == 0) a.pieces[2 * blockIdx.x + 1] = 0;
  }
  // The next sequence that has keys, from `from` on; -1 only if lengths change
  // meanwhile.
  auto next_sequence = [&](int from) __attribute__((always_inline)) {
    for (;;) {
      int found = -1;
#pragma unroll
      for (int i = 0; i < kWindow; ++i) {
        const int lo = max(0, from - window - kWave * i);
        const uint64_t some = __builtin_amdgcn_ballot_w64(lens[i] > 0);
        const uint64_t later = lo < kWave ? some >> lo << lo : 0ull;
        if (found < 0 && later) {
          const int at = sgpr(__builtin_ctzll(later));
          found = window + kWave * i + at;
          len = __builtin_amdgcn_readlane(lens[i], at);
        }
      }
      if (found >= 0) return found;
      window += kWave * kWindow;
      if (window >= a.B) return -1;
      load_lengths();
    }
  };
  const int per_page = a.page / kBlock;
  int page_at = 2 * s / per_page, block_at = 2 * s % per_page;  // of the next step's first block

  // Its steps; by teams or by the list (each with code of its own: tests of `team` in the
  // steps cost the list 1 to 3 %).
  auto work = [&](auto mode) __attribute__((always_inline)) {
    constexpr bool kTeams = decltype(mode)::value;
    // The next step of the range; none left: no keys.
    auto next_step = [&]() __attribute__((always_inline)) {
      Step t;
      t.b = b;
      t.head = head;
      t.s = s;
      t.steps = steps;
      const int n = left > 0 ? min(kStep, len - kStep * s) : 0;
      t.n[0] = min(kBlock, n);
      t.n[1] = max(0, n - kBlock);
      t.row[0] = block_at * kBlock;
      const int32_t *const table = a.tables + (int64_t)b * a.table_stride;
      t.page[0] = n > 0 ? uniform_load(table + page_at) : 0;
      if (++block_at == per_page) {
        block_at = 0;
        ++page_at;
      }
      t.row[1] = block_at * kBlock;
      t.page[1] = n > kBlock ? uniform_load(table + page_at) : 0;
      if (++block_at == per_page) {
        block_at = 0;
        ++page_at;
      }
      if constexpr (kTeams) {
        --left;
        s += kTeam;
        block_at += 2 * (kTeam - 1);
        page_at += block_at / per_page;
        block_at %= per_page;
      } else if (--left > 0 && ++s == steps) {
        s = page_at = block_at = 0;
        if (++head == heads) {
          head = 0;
          const int next = next_sequence(b + 1);
          if (next < 0) {
            left = 0;
          } else {
            b = next;
            steps = steps_of(len);
          }
        }
      }
      return t;
    };

    // ---- loads ----
    // Load j of a block, lane l: 16 bytes of row (64 j + l) / (D / 8), which land
    // at place (64 j + l) % (D / 8) of that row.
    uint32_t k_off[kLoads], v_off[kLoads], q_off[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int row = (64 * j + lane) / (D / 8), place = lane % (D / 8);
      k_off[j] = (uint32_t)row * (uint32_t)(2 * a.k_row) + 16 * (place ^ swizzle_k<D>(row));
      v_off[j] = (uint32_t)row * (uint32_t)(2 * a.v_row) + 16 * (place ^ swizzle_v<D>(row));
      q_off[j] = (uint32_t)row * (2 * D) + 16 * (place ^ swizzle_k<D>(row));
    }
    // Keys of a block that are there: none of a page outside the cache.
    auto usable = [&](const Step &t, int i) __attribute__((always_inline)) {
      return (uint32_t)t.page[i] < (uint32_t)a.P ? t.n[i] : 0;
    };
    auto issue = [&](const Step &t, const uint16_t *pages, int64_t page_st, int64_t head_st, int64_t row_st,
                     const uint32_t (&off)[kLoads], uint8_t *stage) __attribute__((always_inline)) {
      const int64_t head_at = (t.head / blocks) * head_st;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = usable(t, i);
        const uint16_t *const base = pages + (n ? t.page[i] * page_st + head_at + t.row[i] * row_st : 0);
        const auto rs = buffer(base, n ? (uint32_t)(n - 1) * (uint32_t)(2 * row_st) + 2 * D : 0u);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) load_lds16(rs, stage + (i * kLoads + j) * 1024, off[j]);
      }
    };
    auto issue_k = [&](const Step &t) __attribute__((always_inline)) {
      issue(t, a.k, a.k_page, a.k_head, a.k_row, k_off, kst);
      asm volatile("" ::: "memory");  // the counted waits rely on the order
    };
    auto issue_v = [&](const Step &t) __attribute__((always_inline)) {
      issue(t, a.v, a.v_page, a.v_head, a.v_row, v_off, vst);
      asm volatile("" ::: "memory");
    };
    auto issue_q = [&](const Step &t) __attribute__((always_inline)) {
      const int kvh = t.head / blocks, part = t.head % blocks, rows = min(kRows, group - kRows * part);
      const uint16_t *const base = a.q + t.b * a.q_stride + (int64_t)(kvh * group + kRows * part) * D;
      const auto rs = buffer(base, (uint32_t)rows * 2 * D);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) load_lds16(rs, qst + j * 1024, q_off[j]);
      asm volatile("" ::: "memory");
    };

    // ---- operand addresses ----
    uint32_t k_at[kSlices];  // chunk 4 ks + g of row r
#pragma unroll
    for (int ks = 0; ks < kSlices; ++ks) k_at[ks] = (uint32_t)(r * 2 * D + 16 * ((4 * ks + g) ^ swizzle_k<D>(r)));
    const uint32_t k_base = lds_addr(kst);
    const int v_row = 4 * g + (r >> 2);  // the lane addresses dims 4 (r % 4) .. of this key
    const uint32_t v_base = lds_addr(vst) + (uint32_t)(v_row * 2 * D + 16 * (((r & 3) >> 1) ^ swizzle_v<D>(v_row)) + 8 * (r & 1));

    // Softmax state of query row r (this lane's keys only in l), base-2 domain; O:
    // rows 4 g + i, dims 16 dt + r.
    float m_run = -INFINITY, l_run = 0.f;
    float m_top = -INFINITY;  // fp16: limit(m_run), kept
    f32x4 o[kTiles];
#pragma unroll
    for (int dt = 0; dt < kTiles; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float sl2 = a.scale * kLog2e;
    int piece_from = s, piece_unit = first;  // where the present piece began
    int unit = first;
    bool bad_page = false;

    Step cur = next_step(), nx = next_step();
    issue_q(cur);
    issue_k(cur);
    issue_v(cur);
    while (cur.n[0] > 0) {
      // K (and Q) have landed once at most V's loads remain.
      wait_vmcnt<2 * kLoads>();
      u32x4 kf[2 * kSlices], qf[kSlices];
      read_kq<D>(k_base, k_at, kf, qf);
      f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < kSlices; ++ks)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) sc[kt] = mfma16x16<F16>(kf[2 * ks + kt], qf[ks], sc[kt]);
      if (nx.b != cur.b || nx.head != cur.head) issue_q(nx);
      issue_k(nx);
      // Lane: keys 16 kt + 4 g + i of query row r.
      const int n0 = usable(cur, 0), n1 = usable(cur, 1);
      if (n0 + n1 < kStep) {
        bad_page |= n0 != cur.n[0] || n1 != cur.n[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[0][i] = 4 * g + i < n0 ? sc[0][i] : -INFINITY;
          sc[1][i] = 4 * g + i < n1 ? sc[1][i] : -INFINITY;
        }
      }
      const float lmax = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                               fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3]))) * sl2;
      if (__builtin_amdgcn_ballot_w64(lmax > (F16 ? m_top : limit<F16>(m_run)))) {
        const float m_new = fmaxf(m_run, reference<F16>(quad_max(lmax)));
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
          for (int i = 0; i < 4; ++i) o[dt][i] *= al[i];
      }
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      float p[2][4];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kt][i], sl2, neg_m));
      l_run += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
      // Probabilities in the type of V: half a step each, see reference(), against fp32
      // sums of both.
      const u32x4 pa = {pack2<F16>(p[0][0], p[0][1]), pack2<F16>(p[0][2], p[0][3]), pack2<F16>(p[1][0], p[1][1]),
                        pack2<F16>(p[1][2], p[1][3])};
      // V has landed once at most the next K's loads remain.
      wait_vmcnt<2 * kLoads>();
      u32x2 vr[2 * kTiles];
      read_v<D>(v_base, vr);
      issue_v(nx);
#pragma unroll
      for (int dt = 0; dt < kTiles; ++dt)
        o[dt] = mfma16x16<F16>(pa, u32x4{vr[2 * dt][0], vr[2 * dt][1], vr[2 * dt + 1][0], vr[2 * dt + 1][1]}, o[dt]);

      // ---- the end of a piece ----
      const bool pair_ends = cur.s + 1 == cur.steps;
      if (!kTeams && (pair_ends || nx.n[0] == 0)) {
        const int kvh = cur.head / blocks, part = cur.head % blocks, rows = min(kRows, group - kRows * part);
        const int64_t head0 = (int64_t)cur.b * a.Hq + kvh * group + kRows * part;
        const float l = quad_sum(l_run);
        const bool whole = pair_ends && piece_from == 0;
        const int slot = 2 * worker + (piece_unit == first ? 0 : 1);
        if (piece_from == 0 && lane == 0) {
          // Pieces of the (sequence, head block): this one, then the first pieces
          // of the following waves.
          const int last = (piece_unit + cur.steps - 1) / per;
          a.pieces[2 * (cur.b * heads + cur.head)] = slot;
          a.pieces[2 * (cur.b * heads + cur.head) + 1] = whole ? 0 : last - worker + 1;
        }
        float L[4], M[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          L[i] = __shfl(l, 4 * g + i, kWave);
          M[i] = __shfl(m_run, 4 * g + i, kWave);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 4 * g + i;
          if (row >= rows) continue;
          if (whole) {
            const float inv = L[i] == 0.f ? 0.f : 1.0f / L[i];
            uint16_t *const op = a.out + (head0 + row) * D + r;
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt) op[16 * dt] = (uint16_t)pack2<F16>(o[dt][i] * inv, 0.f);
          } else {
            float *const pp = a.partial + ((int64_t)slot * min(group, kRows) + row) * (D + 2);
            if (r == 0) {
              pp[0] = M[i];
              pp[1] = L[i];
            }
#pragma unroll
            for (int dt = 0; dt < kTiles; ++dt) pp[2 + 16 * dt + r] = o[dt][i];
          }
        }
        m_run = m_top = -INFINITY;
        l_run = 0.f;
#pragma unroll
        for (int dt = 0; dt < kTiles; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        piece_from = 0;
        piece_unit = unit + 1;
      }
      ++unit;
      cur = nx;
      nx = next_step();
    }
    wait_vmcnt<0>();  // the last (empty) step's loads write LDS
    if (bad_page && lane == 0) atomicOr(a.status, GQA_STATUS_BAD_PAGE);

    if constexpr (kTeams) {
      // The waves' states, each in its own part of the LDS: O, then m and l per row.
      const int kvh = head / blocks, part = head % blocks, rows = min(kRows, group - kRows * part);
      const float l = quad_sum(l_run);
      float *const mine = (float *)kst;
      mfma_settle();
      if (g == 0) {
        mine[kRows * D + r] = m_run;
        mine[kRows * D + kRows + r] = l;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (4 * g + i < rows) {
#pragma unroll
          for (int dt = 0; dt < kTiles; ++dt) mine[(4 * g + i) * D + 16 * dt + r] = pin(o[dt][i]);
        }
      __syncthreads();
      uint32_t *const out = (uint32_t *)(a.out + ((int64_t)b * a.Hq + kvh * group + kRows * part) * D);
      for (int e = 2 * threadIdx.x; e < rows * D; e += 2 * 64 * kTeam) {
        const int row = e / D;
        float m[kTeam], top = -INFINITY, den = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int w = 0; w < kTeam; ++w) {
          m[w] = ((const float *)(smem + w * kWaveLds<D>))[kRows * D + row];
          top = fmaxf(top, m[w]);
        }
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kTeam; ++w) {
          const float *const x = (const float *)(smem + w * kWaveLds<D>);
          const float f = __builtin_amdgcn_exp2f(m[w] - ref);
          const f32x2_t v = *(const f32x2_t *)(x + e);
          den = __builtin_fmaf(f, x[kRows * D + kRows + row], den);
          o0 = __builtin_fmaf(f, v[0], o0);
          o1 = __builtin_fmaf(f, v[1], o1);
        }
        const float inv = den == 0.f ? 0.f : 1.0f / den;
        out[e / 2] = pack2<F16>(o0 * inv, o1 * inv);
      }
    }
  };
  if constexpr (TEAM > 0) work(std::true_type());
  else if (team) work(std::true_type());
  else work(std::false_type());
}

// Joins the pieces of a (sequence, head block), in the order of the keys.  A thread
// takes two elements of O of all pieces, or, where there are too few elements to
// fill the chip, of every groups-th piece, and the groups are joined in order;
// kBatch pieces' loads are in flight together.  A piece without a usable key (m =
// -inf) has weight 0, a row without any is 0; NaN passes through.  Sequences of
// length 0 get their zeros here.
constexpr int kMergeThreads = 256;
constexpr int kBatch = 16;
struct State {
  float m, l;
  f32x2_t o;
};
template <bool F16>
__global__ __launch_bounds__(kMergeThreads) void gqa_paged_merge(GqaPagedArgs a, int chunk) {
  __shared__ State states[kMergeThreads];
  const int group = a.Hq / a.Hkv, blocks = (group + kRows - 1) / kRows, heads = a.Hkv * blocks;
  const int b = blockIdx.x / heads, head = blockIdx.x % heads;
  const bool empty = a.lengths[b] <= 0;
  const int slot = a.pieces[2 * blockIdx.x], n = empty ? 0 : a.pieces[2 * blockIdx.x + 1];
  if (!empty && n == 0) return;  // written by the wave that had all of it
  const int kvh = head / blocks, part = head % blocks, rows = min(kRows, group - kRows * part);
  const int per_slot = min(group, kRows), groups = kMergeThreads / chunk;
  const int e = 2 * (blockIdx.y * chunk + threadIdx.x % chunk), mine = threadIdx.x / chunk;  // element, group
  const int half = a.D == 128 ? 7 : 6;                                                       // log2 D
  const bool live = e < rows * a.D;
  const int row = live ? e >> half : 0, d = e & (a.D - 1);
  uint32_t *const op = (uint32_t *)(a.out + (((int64_t)b * a.Hq + kvh * group + kRows * part + row) * a.D + d));
  if (empty) {
    if (live && mine == 0) *op = 0;
    return;
  }
  // Piece 0 lies in `slot`, the i-th in the first slot of the i-th following wave
  // (32-bit offsets: the states take 35 MB at most).
  const uint32_t row_bytes = (uint32_t)(a.D + 2) * 4, slot_bytes = (uint32_t)per_slot * row_bytes;
  const uint8_t *const base = (const uint8_t *)a.partial;
  const uint32_t own = (uint32_t)row * row_bytes, first = (uint32_t)(slot / 2 * 2) * slot_bytes + own;
  State st = {-INFINITY, 0.f, f32x2_t{0.f, 0.f}};
  for (int i = mine; i < n; i += groups * kBatch) {
    f32x2_t ml[kBatch], x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int at = min(i + j * groups, n - 1);
      const uint32_t off = at ? first + (uint32_t)at * 2 * slot_bytes : (uint32_t)slot * slot_bytes + own;
      ml[j] = *(const f32x2_t *)(base + off);
      x[j] = *(const f32x2_t *)(base + off + 8 + 4 * d);
    }
    float top = st.m;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) top = i + j * groups < n ? fmaxf(top, ml[j][0]) : top;
    const float ref = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(st.m - ref);
    st.m = top;
    st.l *= old;
    st.o[0] *= old;
    st.o[1] *= old;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (i + j * groups >= n) break;
      const float w = __builtin_amdgcn_exp2f(ml[j][0] - ref);
      st.l = __builtin_fmaf(w, ml[j][1], st.l);
      st.o[0] = __builtin_fmaf(w, x[j][0], st.o[0]);
      st.o[1] = __builtin_fmaf(w, x[j][1], st.o[1]);
    }
  }
  if (groups > 1) {
    states[threadIdx.x] = st;
    __syncthreads();
    if (mine > 0) return;
    for (int g = 1; g < groups; ++g) {
      const State y = states[g * chunk + threadIdx.x];
      const float top = fmaxf(st.m, y.m), ref = top == -INFINITY ? 0.f : top;
      const float wa = __builtin_amdgcn_exp2f(st.m - ref), wb = __builtin_amdgcn_exp2f(y.m - ref);
      st.m = top;
      st.l = st.l * wa + y.l * wb;
      st.o[0] = st.o[0] * wa + y.o[0] * wb;
      st.o[1] = st.o[1] * wa + y.o[1] * wb;
    }
  }
  const float inv = st.l == 0.f ? 0.f : 1.0f / st.l;
  if (live) *op = pack2<F16>(st.o[0] * inv, st.o[1] * inv);
}

__global__ void clear_bits(uint32_t *w, uint32_t bits) { atomicAnd(w, ~bits); }

int waves_of(int D, int cus) { return cus * kWaves * (D == 128 ? kWorkgroups<128> : kWorkgroups<64>); }

// Waves of a workgroup per (sequence, head block), or 0 for the list and its merge,
// by the steps of a full table.  A team needs no second launch (4 to 7 us), but has all
// of its sequence, however long it is.  So: eight waves if all teams then run at
// once, else four (short prologues overlap; 2048 teams, lengths 1..512: 42 us, by
// eight 53); and a team only if one with a full table has at most 16 steps a wave, and
// not many more than half of what the list would give a wave.  By the list and by teams, 8
// heads of 128, so 8 pairs a sequence: 8 pairs of 128 keys 9.2, 4.7 us; 128 of 512 keys 14.0,
// 7.8; 128 of 2048 keys 28, 22; 2048 of 1..1024 keys 98, 80; 128, 8 of 2048 keys and the
// others of 40, 13.0, 13.7.  Left to the list: 8 of 2048 keys 10.1, 13.6; 8 of 4096
// keys 11.8, 22.5.
int team_of(int64_t pairs, int64_t steps, int64_t waves) {
  const int team = 8 * pairs <= waves ? 8 : 4;
  const int64_t listed = (pairs * steps + waves - 1) / waves, teamed = (steps + team - 1) / team;
  return teamed <= most_teamed(listed) ? team : 0;
}

template <int D, bool F16, int TEAM>
hipError_t launch_kernel(const GqaPagedArgs &a, int grid, hipStream_t s) {
  auto k = gqa_paged_kernel<D, F16, TEAM>;
  constexpr int waves = TEAM ? TEAM : kWaves, lds = waves * kWaveLds<D>;
  static std::atomic<uint64_t> allowed{0};
  if (const hipError_t e = allow_lds((const void *)k, lds, &allowed)) return e;
  hipLaunchKernelGGL(k, dim3(grid), dim3(64 * waves), lds, s, a);
  return hipGetLastError();
}

template <int D, bool F16>
hipError_t launch(const GqaPagedArgs &a, int cus, hipStream_t s) {
  const int group = a.Hq / a.Hkv, heads = a.Hkv * ((group + kRows - 1) / kRows), pairs = a.B * heads;
  const int team = team_of(pairs, ((int64_t)a.M * a.page + kStep - 1) / kStep, waves_of(D, cus));
  if (team == 8) return launch_kernel<D, F16, 8>(a, pairs, s);
  if (team == 4) return launch_kernel<D, F16, 4>(a, pairs, s);
  const hipError_t e = launch_kernel<D, F16, 0>(a, cus * kWorkgroups<D>, s);
  if (e != hipSuccess) return e;
  // Threads per piece in a merge workgroup: all of a (sequence, head block), two
  // elements each; fewer, and pieces shared out over groups, while that leaves CUs
  // without a workgroup.
  const int need = min(group, kRows) * D / 2;
  int chunk = kMergeThreads;
  while (chunk > 16 && (chunk >= 2 * need || (int64_t)pairs * ((need + chunk - 1) / chunk) < cus)) chunk /= 2;
  hipLaunchKernelGGL(gqa_paged_merge<F16>, dim3(pairs, (need + chunk - 1) / chunk), dim3(kMergeThreads), 0, s, a, chunk);
  return hipGetLastError();
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

// {status words; two words per (sequence, head block); the pieces' states}; teams
// have no pieces.
size_t gqa_paged_workspace(int B, int Hq, int Hkv, int D, int64_t keys, int cus) {
  const int group = Hq / Hkv, rows = group < kRows ? group : kRows;
  const size_t pairs = (size_t)B * Hkv * ((group + kRows - 1) / kRows);
  if (team_of(pairs, (keys + kStep - 1) / kStep, waves_of(D, cus))) return 256;
  return 256 + align256(8 * pairs) + (size_t)2 * waves_of(D, cus) * rows * (D + 2) * sizeof(float);
}

void gqa_paged_bind(GqaPagedArgs *a, void *workspace) {
  uint8_t *const w = (uint8_t *)workspace;
  const int group = a->Hq / a->Hkv;
  const size_t pairs = (size_t)a->B * a->Hkv * ((group + kRows - 1) / kRows);
  a->status = (uint32_t *)w;
  a->pieces = (int32_t *)(w + 256);
  a->partial = (float *)(w + 256 + align256(8 * pairs));
}

hipError_t launch_gqa_paged(const GqaPagedArgs &a, int cus, hipStream_t s) {
  if (a.D == 128) return a.dtype == GQA_FP16 ? launch<128, true>(a, cus, s) : launch<128, false>(a, cus, s);
  return a.dtype == GQA_FP16 ? launch<64, true>(a, cus, s) : launch<64, false>(a, cus, s);
}

// Clears the bits that it returns, no others, and is done with that on return: a bit
// that work on another stream latches meanwhile is in this reading or in the next.
hipError_t read_and_clear_status(uint32_t *status, uint32_t *flags, hipStream_t s) {
  hipError_t e = hipStreamSynchronize(s);
  if (e == hipSuccess) e = hipMemcpy(flags, status, sizeof(uint32_t), hipMemcpyDeviceToHost);
  if (e == hipSuccess && *flags) {
    hipLaunchKernelGGL(clear_bits, dim3(1), dim3(1), 0, s, status, *flags);
    e = hipGetLastError();
    if (e == hipSuccess) e = hipStreamSynchronize(s);
  }
  return e;
}

}  // namespace moe
