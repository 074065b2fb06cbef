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

// A group's work; a lane of a wave has one.  A unit: a KV head's tile of rows over a chunk of
// the steps, in the order (KV head, chunk, tile).
struct Group {
  int before, chunk_steps, first, rows;     // units before, steps of a chunk, first member, query rows
  int source, keys, tiles, tile_rows;       // member whose table is read, keys that are shared
  int chunks, more;                         // units before but each (KV head, tile)'s first
};
// The plan of a run: units, the workgroups for them, the groups of the wave's lanes and the
// keys that a group attends for the rows 64 i + lane.
struct Plan {
  int units, workgroups;
  Group group;
  int skips[4];
};
constexpr int kLocalRows = 64 * kWaves, kLocalGroups = kWave;

// Length of a row as the paged kernels take it.
__device__ __forceinline__ int length_of(const GqaPagedArgs &p, int b) { return max(0, min(p.lengths[b], p.M * p.page)); }
__device__ __forceinline__ int steps_of(int keys) { return (int)(((uint32_t)keys + kStep - 1) / kStep); }

// What a group of `rows` query rows of a KV head and `live` members with keys shares: the
// multiple of 16 keys up to its prefix and its shortest member, if there are two of those.
__device__ __forceinline__ void share(Group *g, int wanted, int least, int live) {
  g->keys = live < 2 ? 0 : max(0, min(wanted, least)) / kBlock * kBlock;
  g->tiles = g->keys ? (g->rows + kSharedRows - 1) / kSharedRows : 0;
  const int blocks = (g->rows + 31) / 32;
  g->tile_rows = g->tiles ? (blocks + g->tiles - 1) / g->tiles * 32 : 32;
}
// Workgroups for the prefixes, of all, by steps: those are as many bytes in either part, and
// the four waves of the list's have a step each in flight, as the others have four stages.
__device__ __forceinline__ int share_of(int64_t shared, int64_t listed, int workgroups) {
  if (shared == 0) return 0;
  const int n = (int)((float)workgroups * ((float)shared / (float)(shared + listed)) + 0.5f);
  return max(1, min(n, listed ? workgroups - 1 : workgroups));
}
// Steps of a chunk: the fewest with which the units are not more than the workgroups, of
// kSizes from the average up to three times that.  If none is (there are more groups than
// that), the average, and a workgroup has several units.
constexpr int kLeastSteps = 2;  // one costs more in states than it gains
constexpr int kSizes = 16;
__device__ __forceinline__ int chunk_size(int64_t shared, int n, int i) {  // shared < 2^30, checked on the host
  const int even = n ? max(kLeastSteps, (int)(((uint32_t)shared + (uint32_t)n - 1u) / (uint32_t)n)) : 1;
  return even + (int)((int64_t)even * i >> 3);
}
__device__ __forceinline__ void cut(Group *g, int size) {
  const uint32_t steps = (uint32_t)steps_of(g->keys), chunks = (steps + (uint32_t)size - 1u) / (uint32_t)size;
  g->chunks = (int)chunks;
  g->chunk_steps = chunks ? (int)((steps + chunks - 1u) / chunks) : 1;
}

// The plan by one workgroup of four waves for itself: up to 64 groups and 256 rows.  Bounds
// that do not ascend within [0, B]: nothing is shared.  Workgroup 0 reports those, negative
// prefixes and lengths out of range (the list reports lengths too, but has no workgroup where
// no key lies behind a prefix) and leaves what the join needs of each row.
__device__ __forceinline__ Plan plan_here(const GqaPagedArgs &p, uint8_t *smem) {
  struct Lds {
    int starts[kLocalGroups + 1], least[kLocalGroups], live[kLocalGroups], source[kLocalGroups], keys[kLocalGroups];
    int skips[kLocalRows], fits[kSizes], rest, wrong;
  };
  Lds *const lds = (Lds *)smem;
  const GqaSharedState &st = p.shared;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per_head = st.group, G = st.G;
  const int raw = tid < p.B ? p.lengths[tid] : 0, len = max(0, min(raw, p.M * p.page));
  const int wanted = lane < G ? st.prefixes[lane] : 0;
  if (tid <= G) lds->starts[tid] = st.starts[tid];
  if (tid < G) {
    lds->least[tid] = lds->source[tid] = 0x7fffffff;
    lds->live[tid] = 0;
  }
  if (tid == 0) lds->rest = lds->wrong = 0;
  __syncthreads();
  // (__syncthreads_or() has LDS of its own, and with it one workgroup per CU less.)
  if (tid <= G && (lds->starts[tid] < 0 || lds->starts[tid] > p.B || (tid > 0 && lds->starts[tid] < lds->starts[tid - 1]))) lds->wrong = 1;
  int g = -1;  // the row's group, if no bound is wrong
  if (G > 0 && tid < p.B && tid >= lds->starts[0] && tid < lds->starts[G]) {
    int hi = G - 1;
    g = 0;
    while (g < hi) {
      const int mid = (g + hi + 1) >> 1;
      if (lds->starts[mid] <= tid) g = mid;
      else hi = mid - 1;
    }
  }
  if (g >= 0 && len > 0) {
    atomicMin(lds->least + g, len);
    atomicMin(lds->source + g, tid);
    atomicAdd(lds->live + g, 1);
  }
  __syncthreads();
  const bool bad = lds->wrong != 0;
  if (bad) g = -1;
  if (blockIdx.x == 0 && ((bad && tid == 0) || wanted < 0 || raw != len)) atomicOr(p.status, GQA_STATUS_BAD_BOUNDS);
  Plan plan = {};
  Group &mine = plan.group;  // every wave has all groups
  mine.before = 0x7fffffff;
  if (lane < G) {
    mine.first = bad ? 0 : lds->starts[lane];
    mine.rows = bad ? 0 : (lds->starts[lane + 1] - mine.first) * per_head;
    share(&mine, wanted, lds->least[lane], bad ? 0 : lds->live[lane]);
    mine.source = mine.keys ? lds->source[lane] : 0;
    if (wave == 0) lds->keys[lane] = mine.keys;
  }
  __syncthreads();
  const int skip = g >= 0 && len > 0 ? lds->keys[g] : 0;
  lds->skips[tid] = skip;
  const int rest = wave_total(steps_of(len - skip));
  if (lane == 0) atomicAdd(&lds->rest, rest);
  const int heads_units = mine.tiles * p.Hkv;  // of a chunk
  const int64_t shared = wave_total(steps_of(mine.keys) * heads_units);
  __syncthreads();
  plan.workgroups = share_of(shared, (int64_t)lds->rest * p.Hkv * ((per_head + 15) / 16), gridDim.x);
  constexpr int kOwn = kSizes / kWaves;  // sizes of a wave
  int units_of[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int size = chunk_size(shared, plan.workgroups, kOwn * wave + i);
    units_of[i] = heads_units * (int)(((uint32_t)steps_of(mine.keys) + (uint32_t)size - 1u) / (uint32_t)size);
  }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    units_of[i] = wave_total(units_of[i]);
    if (lane == 0) lds->fits[kOwn * wave + i] = units_of[i] <= plan.workgroups;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) plan.skips[i] = lds->skips[kWave * i + lane];
  __syncthreads();
  const uint64_t fit = __builtin_amdgcn_ballot_w64(lane < kSizes && lds->fits[lane & (kSizes - 1)]);
  cut(&mine, chunk_size(shared, plan.workgroups, fit ? sgpr(__builtin_ctzll(fit)) : 0));
  const int units = mine.chunks * heads_units, extra = max(0, units - heads_units);
  const int incl = wave_scan(units);
  if (lane < G) mine.before = incl - units;
  mine.more = wave_scan(extra) - extra;
  plan.units = __builtin_amdgcn_readlane(incl, 63);
  if (blockIdx.x == 0) {
    const int from = max(g, 0);  // all lanes take part in the exchange
    const int chunks = __shfl(mine.chunks, from, kWave), tiles = __shfl(mine.tiles, from, kWave);
    const int tile_rows = __shfl(mine.tile_rows, from, kWave), first = __shfl(mine.first, from, kWave);
    const int more = __shfl(mine.more, from, kWave);
    if (tid < p.B) {
      int32_t *const rec = st.rows + 8 * tid;
      *(int4 *)rec = make_int4(skip, chunks, tiles, tile_rows);
      *(int2 *)(rec + 4) = make_int2((tid - first) * per_head, more);
    }
  }
  __syncthreads();  // the LDS is the work's from here
  return plan;
}
// Reports bounds and prefixes, for a launch that does without a plan: by one workgroup.
__device__ __forceinline__ void check_groups(const GqaPagedArgs &p) {
  const GqaSharedState &st = p.shared;
  for (int g = threadIdx.x; g <= st.G; g += blockDim.x) {
    const int at = st.starts[g];
    if (at < 0 || at > p.B || (g > 0 && at < st.starts[g - 1]) || (g < st.G && st.prefixes[g] < 0))
      atomicOr(p.status, GQA_STATUS_BAD_BOUNDS);
  }
}
// The plan as gqa_shared_plan() left it.
__device__ __forceinline__ Plan plan_there(const GqaPagedArgs &p) {
  Plan plan = {};
  plan.units = uniform_load(p.shared.header);
  plan.workgroups = uniform_load(p.shared.header + 1);
  return plan;
}

// Keys that every row of a group sees, in pages; the loop is the packed kernel's, where its
// overlaps and operand layouts are explained.  A workgroup has up to 128 query rows of a
// group and KV head (row = member * G + head), 32 per wave.
template <int D, bool F16>
__device__ __forceinline__ void prefix(const GqaPagedArgs &p, const Plan &plan, uint8_t *smem) {
  constexpr int kSteps = D / 16;                        // QK MFMAs per stage
  constexpr int kDims = D / 32;                         // 32-dim tiles of O
  constexpr int kChunks = D / 8;                        // 16-byte chunks of a row
  constexpr int kLoads = kTile<D> / 1024 / kWaves;      // of K (or V) per wave and stage, 1 KiB each
  const GqaSharedState &a = p.shared;
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = sgpr(threadIdx.x >> 6);
  const int group = a.group;
  // Neighbouring units, whose rows see the same keys, on one XCD, which has them in its L2.
  const int units = plan.units, workgroups = plan.workgroups;
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
    // The last group with at most u units before it has some: a lane for each of 64.
    Group of = plan.group;
    if (!a.local) {
      int lo = 0, hi = (a.G - 1) / kWave;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (uniform_load(a.groups + 16 * kWave * mid) <= u) lo = mid;
        else hi = mid - 1;
      }
      of.before = 0x7fffffff;
      if (kWave * lo + lane < a.G) {
        const int32_t *const rec = a.groups + 16 * (kWave * lo + lane);
        const int4 x = *(const int4 *)rec, y = *(const int4 *)(rec + 4);
        const int2 z = *(const int2 *)(rec + 8);
        of = Group{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y};
      }
    }
    const int g = sgpr((int)__popcll(__builtin_amdgcn_ballot_w64(of.before <= u)) - 1);
    const int before = __builtin_amdgcn_readlane(of.before, g), chunk_steps = __builtin_amdgcn_readlane(of.chunk_steps, g);
    const int first = __builtin_amdgcn_readlane(of.first, g), rows = __builtin_amdgcn_readlane(of.rows, g);
    const int source = __builtin_amdgcn_readlane(of.source, g), keys = __builtin_amdgcn_readlane(of.keys, g);
    const int tiles = __builtin_amdgcn_readlane(of.tiles, g), tile_rows = __builtin_amdgcn_readlane(of.tile_rows, g);
    const int chunks = __builtin_amdgcn_readlane(of.chunks, g), more = __builtin_amdgcn_readlane(of.more, g);
    const int rest = (u - before) / tiles, tile = u - before - rest * tiles, kvh = rest / chunks, chunk = rest - kvh * chunks;
    const int s0 = chunk * chunk_steps, stages = min(chunk_steps, steps_of(keys) - s0);
    const int row0 = tile * tile_rows + kWaveRows * wave;
    const bool own = kWaveRows * wave < tile_rows && row0 < rows;
    const int more_at = more + (kvh * (chunks - 1) + chunk - 1) * tiles + tile;  // chunk > 0

    // ---- loads ----
    const int32_t *const table = p.tables + (int64_t)source * p.table_stride;
    const uint16_t *const k_head = p.k + kvh * p.k_head, *const v_head = p.v + kvh * p.v_head;
    // Pages and rows of the unit's next 128 blocks of 16 keys, from `base` on: lane l has blocks
    // l and 64 + l; a block that is not there: row -1.  (Scalar loads stage by stage made every
    // wait for operands from LDS wait for them too.)
    int base = 2 * s0, pages[2], rows_at[2], loaded = 0;
    auto look_up = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int blk = base + kWave * i + lane;
        const int at = blk / (p.page / kBlock);
        const bool in = blk * kBlock < keys && blk < 2 * (s0 + stages);
        const int page = in ? table[at] : 0;
        const bool ok = (uint32_t)page < (uint32_t)p.P;
        bad_page |= in && !ok;
        pages[i] = ok ? page : 0;
        rows_at[i] = in && ok ? blk * kBlock - at * p.page : -1;
      }
    };
    look_up();
    // Blocks of the stages in flight that are there, two bits each, the last loaded lowest.
    uint32_t there = 0, load_slot = lds0 + wave * kLoads * 1024;
    auto issue = [&]() __attribute__((always_inline)) {
      int at = 2 * (s0 + loaded) - base;
      if (at == 2 * kWave) {
        base += at;
        at = 0;
        look_up();
      }
      int row[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        row[i] = at < kWave ? __builtin_amdgcn_readlane(rows_at[0], at + i) : __builtin_amdgcn_readlane(rows_at[1], at + i - kWave);
      const int my_page = at < kWave ? __builtin_amdgcn_readlane(pages[0], at + block)
                                     : __builtin_amdgcn_readlane(pages[1], at + block - kWave);
      const int my_row = block ? row[1] : row[0];
      there = there << 2 | (row[0] >= 0 ? 1u : 0u) | (row[1] >= 0 ? 2u : 0u);
      const bool mine = my_row >= 0;
      const int64_t from_row = mine ? my_row : 0;
      const uint32_t slot = sgpr((int)load_slot);
      load_lds(buffer_words(k_head + my_page * p.k_page + from_row * p.k_row, mine ? k_bytes : 0u), slot, k_off);
      load_lds(buffer_words(v_head + my_page * p.v_page + from_row * p.v_row, mine ? v_bytes : 0u), slot + kTile<D>, v_off);
      load_slot = load_slot + 2 * kTile<D> >= lds0 + kRing * 2 * kTile<D> ? load_slot - (kRing - 1) * 2 * kTile<D>
                                                                          : load_slot + 2 * kTile<D>;
      ++loaded;
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
      // They are what gqa_paged.hip's are, whose results these stand for: a bf16 output is off by
      // 0.0023 of its rms, by its last rounding alone 0.0017.  As two 16-bit numbers each it was
      // off by 0.0017, and the calls took 74 us instead of 66 (four groups of 22 to 40 sequences), 55
      // instead of 48 (64 with 16000 keys) and, row by row, 12.6 instead of 11.9: not kept.
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
  if (__builtin_amdgcn_ballot_w64(bad_page) && threadIdx.x == 0) atomicOr(p.status, GQA_STATUS_BAD_PAGE);
}

}  // namespace shared
}  // namespace gqa
}  // namespace moe
