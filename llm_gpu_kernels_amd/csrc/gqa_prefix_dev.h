// The part of attention with shared prefixes that goes over the prefixes (a workgroup of
// four waves; gqa_shared.hip has the whole, gqa_paged.hip calls it).
#pragma once

#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"

namespace moe {
namespace gqa {
namespace shared {

constexpr int kWaves = 4, kWaveRows = 32;
constexpr int kStep = 32, kBlock = 16;
static_assert(kWaves * kWaveRows == kSharedRows, "a wave's rows");

__device__ __forceinline__ void lds_write_b128(uint32_t at, f32x4 v) {
#if defined(__HIP_DEVICE_COMPILE__)
  *(GQA_AS_LDS f32x4 *)at = v;
#endif
}
__device__ __forceinline__ f32x2_t lds_read_b64(uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
  return *(const GQA_AS_LDS f32x2_t *)at;
#else
  return f32x2_t{0.f, 0.f};
#endif
}

// Row i of a stage's K (V) tile holds its 16-byte chunk c at place c ^ swizzle(i), as in
// the packed kernel: reads meet different bank groups.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swizzle_v(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

constexpr int kRing = 5;                                 // stages of 32 keys in LDS
template <int D> constexpr int kTile = kStep * D * 2;   // bytes of a stage's K (or V)

// Keys that every row of a group sees, in pages; the loop is the packed kernel's, where its
// overlaps and operand layouts are explained.  A workgroup has up to 128 query rows of a
// group and KV head (row = member * G + head), 32 per wave.
template <int D, bool F16>
__device__ __forceinline__ void prefix(const GqaPagedArgs &p, uint8_t *smem) {
  constexpr int kSteps = D / 16;                        // QK MFMAs per stage
  constexpr int kDims = D / 32;                         // 32-dim tiles of O
  constexpr int kChunks = D / 8;                        // 16-byte chunks of a row
  constexpr int kLoads = kTile<D> / 1024 / kWaves;      // of K (or V) per wave and stage, 1 KiB each
  const GqaSharedState &a = p.shared;
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = sgpr(threadIdx.x >> 6);
  const int group = p.Hq / p.Hkv, per_page = p.page / kBlock;
  // Neighbouring units, whose rows see the same keys, on one XCD, which has them in its L2.
  const int units = uniform_load(a.header), workgroups = uniform_load(a.header + 1);
  const int xcd = blockIdx.x % kXcds, first_unit = xcd * (workgroups / kXcds) + min(xcd, workgroups % kXcds) + (int)blockIdx.x / kXcds;
  const uint32_t lds0 = lds_addr(smem);
  const float sl2 = p.scale * kLog2e;
  bool bad_page = false;

  // The wave's part of a stage: a quarter of K's rows and of V's, all in one 16-key block.
  const int block = wave >> 1;
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int row = (64 * (wave * kLoads + j) + lane) / kChunks, place = lane % kChunks;
    k_off[j] = (uint32_t)(row % kBlock) * (uint32_t)(2 * p.k_row) + 16 * (place ^ swizzle_k<D>(row));
    v_off[j] = (uint32_t)(row % kBlock) * (uint32_t)(2 * p.v_row) + 16 * (place ^ swizzle_v<D>(row));
  }
  const uint32_t k_bytes = 15u * (uint32_t)(2 * p.k_row) + 2 * D, v_bytes = 15u * (uint32_t)(2 * p.v_row) + 2 * D;
  // K fragment ks: row r, chunk 2 ks + h.  V: the lane addresses dims 16 (gi % 2)
  // + 4 x .. of 32, key 4 h + c.
  const uint32_t k_at = (uint32_t)(r * 2 * D + 16 * (h ^ swizzle_k<D>(r)));
  const int v_key = 4 * h + ((lane >> 2) & 3), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = (uint32_t)(kTile<D> + v_key * 2 * D + 16 * (v_chunk ^ swizzle_v<D>(v_key)) + 8 * (lane & 1));

  for (int u = first_unit; u < units; u += workgroups) {
    // The last group with at most u units before it has some: a chunk of 64 groups, then a
    // lane for each.
    int lo = 0, hi = (a.G - 1) / kWave;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (uniform_load(a.groups + 16 * kWave * mid) <= u) lo = mid;
      else hi = mid - 1;
    }
    const int at_lane = kWave * lo + lane < a.G ? a.groups[16 * (kWave * lo + lane)] : 0x7fffffff;
    const int g = kWave * lo + (int)__popcll(__builtin_amdgcn_ballot_w64(at_lane <= u)) - 1;
    const int32_t *const rec = a.groups + 16 * g;
    const int before = uniform_load(rec), chunk_steps = uniform_load(rec + 1), first = uniform_load(rec + 2);
    const int rows = uniform_load(rec + 3), source = uniform_load(rec + 4), keys = uniform_load(rec + 5);
    const int tiles = uniform_load(rec + 6), tile_rows = uniform_load(rec + 7), chunks = uniform_load(rec + 8);
    const int rest = (u - before) / tiles, tile = u - before - rest * tiles, kvh = rest / chunks, chunk = rest - kvh * chunks;
    const int s0 = chunk * chunk_steps, stages = min(chunk_steps, (keys + kStep - 1) / kStep - s0);
    const int row0 = tile * tile_rows + kWaveRows * wave;
    const bool own = kWaveRows * wave < tile_rows && row0 < rows;
    const int more_at = uniform_load(rec + 9) + (kvh * (chunks - 1) + chunk - 1) * tiles + tile;  // chunk > 0

    // ---- loads ----
    const int32_t *const table = p.tables + (int64_t)source * p.table_stride;
    const uint16_t *const k_head = p.k + kvh * p.k_head, *const v_head = p.v + kvh * p.v_head;
    // The next stage's blocks: place in the table, block there, page, which is loaded a stage
    // ahead, and whether it is within the keys.
    int at[2], in[2], page[2], loaded = 0;
    auto find = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        page[i] = (2 * (s0 + loaded) + i) * kBlock < keys ? uniform_load(table + at[i]) : 0x7fffffff;
    };
    at[0] = 2 * s0 / per_page;
    in[0] = 2 * s0 - at[0] * per_page;
    at[1] = in[0] + 1 == per_page ? at[0] + 1 : at[0];
    in[1] = in[0] + 1 == per_page ? 0 : in[0] + 1;
    find();
    // Blocks of the stages in flight that are there, two bits each, the last loaded lowest.
    uint32_t there = 0, load_slot = lds0 + wave * kLoads * 1024;
    auto issue = [&]() __attribute__((always_inline)) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        bits |= (uint32_t)page[i] < (uint32_t)p.P ? 1u << i : 0u;
        bad_page |= (uint32_t)page[i] >= (uint32_t)p.P && (2 * (s0 + loaded) + i) * kBlock < keys;
      }
      there = there << 2 | bits;
      const bool mine = bits >> block & 1u;
      const int64_t my_page = mine ? (block ? page[1] : page[0]) : 0, my_row = (block ? in[1] : in[0]) * kBlock;
      const uint32_t slot = sgpr((int)load_slot);
      load_lds(buffer_words(k_head + my_page * p.k_page + my_row * p.k_row, mine ? k_bytes : 0u), slot, k_off);
      load_lds(buffer_words(v_head + my_page * p.v_page + my_row * p.v_row, mine ? v_bytes : 0u), slot + kTile<D>, v_off);
      load_slot = load_slot + 2 * kTile<D> >= lds0 + kRing * 2 * kTile<D> ? load_slot - (kRing - 1) * 2 * kTile<D>
                                                                          : load_slot + 2 * kTile<D>;
      ++loaded;
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // a stage on: two blocks, a page has one at least
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (++in[i] == per_page) {
            in[i] = 0;
            ++at[i];
          }
      }
      find();
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
    for (int st = 0; st < min(3, stages); ++st) issue();

    // ---- operands ----
    // Rows of Q, one per lane pair; those behind the last are the last again.
    const int row = min(row0 + r, rows - 1), member = row / group, head = kvh * group + row - member * group;
    u32x4 qf[kSteps];
    {
      const uint16_t *const qp = p.q + (int64_t)(first + member) * p.q_stride + (int64_t)head * D + 8 * h;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) qf[ks] = *(const u32x4 *)(qp + 16 * ks);
    }
    u32x4 kf[kSteps], vf[2][kDims];
    uint32_t slot[3] = {lds0, lds0 + 2 * kTile<D>, lds0 + 4 * kTile<D>};  // of this stage and the next two
    auto read_k = [&](uint32_t from, int ks) __attribute__((always_inline)) { kf[ks] = lds_b128((from + k_at) ^ (32 * ks)); };
    auto read_v = [&](int j, int db) __attribute__((always_inline)) {
      const uint32_t from = ((slot[0] + v_at) ^ (64 * db)) + j * 32 * D;
      const u32x2 lo = lds_tr16(from), hi = lds_tr16(from + 16 * D);
      vf[j][db] = u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    float m_run = -INFINITY, l_run = 0.f, m_top = -INFINITY;  // base-2 domain; l of this lane's keys
    f32x16 o[kDims], sa, sb;
#pragma unroll
    for (int db = 0; db < kDims; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float top = -INFINITY;  // of the raw scores of the stage at hand

    // One stage: its scores in s; the next one's come into sn.
    auto step = [&](int st, f32x16 &s, f32x16 &sn) __attribute__((always_inline)) {
      // (Behind the last stage these are of rows in the ring that nothing asks for.)
#pragma unroll
      for (int ks = kSteps / 2; ks < kSteps; ++ks) read_k(slot[1], ks);
#pragma unroll
      for (int i = 0; i < 16; ++i) sn[i] = 0.f;
#pragma unroll
      for (int m = 0; m < 2; ++m) sn = mfma32x32<F16>(kf[m], qf[m], sn);
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t bits = there >> 2 * (loaded - 1 - st) & 3u;
      if (bits != 3u) {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = bits >> (i >> 3) & 1u ? s[i] : -INFINITY;
          top = fmaxf(top, s[i]);
        }
      }
      if (__builtin_amdgcn_ballot_w64(top * sl2 > (F16 ? m_top : limit<F16>(m_run)))) {
        mfma_settle();
        const f32x2_t both = halves(top * sl2);
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
      // The rest of the next stage's scores beside this one's exponentials.
      u32x4 pb[2];
      float sum0 = 0.f, sum1 = 0.f, p0 = 0.f, p1 = 0.f;
      // Pair x of probabilities (in the type of V: half a step each, see reference(),
      // against fp32 sums of both) and of the sums; a pair later than its exponentials.
      auto take = [&](int y) __attribute__((always_inline)) {
        uint32_t w = pack2<F16>(p0, p1);
        sum0 += p0;
        sum1 += p1;
        asm volatile("" : "+v"(w), "+v"(sum0), "+v"(sum1));  // here, not where they are used
        pb[y / 4][y % 4] = w;
      };
      constexpr int kEach = 8 / kSteps;  // pairs of scores per MFMA
#pragma unroll
      for (int m = 0; m < kSteps; ++m) {
        if (m >= 2) sn = mfma32x32<F16>(kf[m], qf[m], sn);
#pragma unroll
        for (int y = kEach * m; y < kEach * (m + 1); ++y) {
          const float e0 = pin(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * y], sl2, neg_m)));
          const float e1 = pin(__builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * y + 1], sl2, neg_m)));
          if (y > 0) take(y - 1);
          p0 = e0;
          p1 = e1;
        }
        if (m == kSteps - 1) take(7);
        if (m < kSteps / 2) read_v(0, m % kDims);
        else read_v(1, m % kDims);
        __builtin_amdgcn_sched_barrier(0);
      }
      l_run += sum0 + sum1;
      if (st + 2 < stages) sync(st);
      // O of this stage beside the next one's maxima.
      constexpr int kPv = 2 * kDims;
      top = -INFINITY;
#pragma unroll
      for (int m = 0; m < kPv; ++m) {
        o[m % kDims] = mfma32x32<F16>(vf[m / kDims][m % kDims], pb[m / kDims], o[m % kDims]);
#pragma unroll
        for (int y = m < 2 ? 0 : 8 * (m - 2) / (kPv - 2); y < (m < 2 ? 0 : 8 * (m - 1) / (kPv - 2)); ++y) {
          sn[2 * y] = pin(sn[2 * y]);
          sn[2 * y + 1] = pin(sn[2 * y + 1]);
          top = pin(fmaxf(fmaxf(sn[2 * y], sn[2 * y + 1]), top));
        }
        if (m >= kDims) read_k(slot[2], m - kDims);
        __builtin_amdgcn_sched_barrier(0);
      }
      slot[0] = slot[1];
      slot[1] = slot[2];
      slot[2] = slot[2] + 2 * kTile<D> >= lds0 + kRing * 2 * kTile<D> ? lds0 : slot[2] + 2 * kTile<D>;
    };

    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    for (int st = 3; st < min(kRing - 1, stages); ++st) issue();
    if (own) {
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) read_k(slot[0], ks);
#pragma unroll
      for (int i = 0; i < 16; ++i) sa[i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) sa = mfma32x32<F16>(kf[ks], qf[ks], sa);
#pragma unroll
      for (int ks = 0; ks < kSteps / 2; ++ks) read_k(slot[1], ks);
      mfma_settle();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sa[i] = pin(sa[i]);
        top = fmaxf(top, sa[i]);
      }
      for (int st = 0; st < stages; st += 2) {
        step(st, sa, sb);
        if (st + 1 == stages) break;
        step(st + 1, sb, sa);
      }
    } else {
      for (int st = 0; st + 2 < stages; ++st) sync(st);
    }
    mfma_settle();
    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();  // no stage is read any more
    asm volatile("" ::: "memory");
    if (own) {
      // Lane (r, h) holds dims 32 db + 8 q + 4 h + i of its row.  Through LDS to whole rows:
      // stores of 8 bytes in each of 64 places took 10 us.
      const f32x2_t both = halves(l_run);
      const uint32_t mine = lds0 + (uint32_t)wave * (kWaveRows * D * 4);
      constexpr int kQuads = D / 4;
#pragma unroll
      for (int db = 0; db < kDims; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          lds_write_b128(mine + (uint32_t)(r * D * 4 + 16 * ((8 * db + 2 * q + h) ^ (r & (kQuads - 1)))),
                         f32x4{pin(o[db][4 * q]), pin(o[db][4 * q + 1]), pin(o[db][4 * q + 2]), pin(o[db][4 * q + 3])});
      const int there_rows = min(kWaveRows, rows - row0);
      // The first chunk's states by row, another's by unit.
      auto record = [&](int y) __attribute__((always_inline)) {
        const int nth = row0 + y, m = nth / group;
        return chunk > 0 ? a.more + ((int64_t)more_at * kSharedRows + kWaveRows * wave + y) * (D + 2)
                         : a.heads + ((int64_t)(first + m) * p.Hq + kvh * group + nth - m * group) * (D + 2);
      };
      if (h == 0 && r < there_rows) *(f32x2_t *)record(r) = f32x2_t{m_run, both[0] + both[1]};
      constexpr int kAtOnce = 128 / D;  // rows of a store
#pragma unroll 4
      for (int y0 = 0; y0 < there_rows; y0 += kAtOnce) {
        const int y = y0 + lane / (D / 2), d = 2 * (lane % (D / 2));
        if (y < there_rows)
          *(f32x2_t *)(record(y) + 2 + d) =
              lds_read_b64(mine + (uint32_t)(y * D * 4 + 16 * ((d / 4) ^ (y & (kQuads - 1))) + 4 * (d % 4)));
      }
    }
    // The next unit's loads are counted from here, into slots that nobody reads.
    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  if (bad_page && threadIdx.x == 0) atomicOr(p.status, GQA_STATUS_BAD_PAGE);
}

}  // namespace shared
}  // namespace gqa
}  // namespace moe
