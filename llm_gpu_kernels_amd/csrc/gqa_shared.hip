// Attention of one new token per sequence over a paged cache, where groups of sequences
// start with the same keys (samples of one prompt, users of one instruction), on gfx950.
//
// softmax(q K^T) V over a prefix and the rest of a row's keys is joined from the two
// parts' (max, sum, O), so a prefix is read once for all rows of its group: up to 256
// query rows (the members' heads of one KV head) are one workgroup's, 32 per wave, and K
// and V go through LDS for all of them.  With few rows its bytes bound it, with some
// hundreds the matrix cores.  The keys behind the prefix are worked on as
// gqa_paged.hip works on whole rows.
//
//   plan    one workgroup: the keys that each group shares, and its steps of 32 keys
//           before which others' lie;
//   prefix  the steps of all (group, KV head, 256 rows) cut into equal ranges, one per
//           workgroup; a piece of one that begins there leaves its states by row, one
//           that goes on from the workgroup before by workgroup;
//   rest    gqa_paged.hip's list of steps over the keys behind;
//   join    all pieces' states of a row in the order of the keys.
#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"
#include "launch.h"

namespace moe {

using namespace gqa;

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanLds = 8192;  // sequences whose lengths lie in LDS
constexpr int kWaves = 8, kWaveRows = 32;
constexpr int kStep = 32, kBlock = 16;
constexpr int kMergeThreads = 256, kBatch = 8;
static_assert(kWaves * kWaveRows == kSharedRows, "a wave's rows");

__device__ __forceinline__ int wave_least(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, kWave));
  return x;
}

// Row length as the paged kernels take it.
__device__ __forceinline__ int length_of(const GqaPagedArgs &p, int b) { return max(0, min(p.lengths[b], p.M * p.page)); }

// What each group shares: the multiple of 16 keys up to its prefix, and up to the shortest
// of its members that have keys, if there are two of those.  Bounds that do not ascend
// within [0, B]: nothing is shared, and every row is attended by itself.
__global__ __launch_bounds__(kPlanThreads) void gqa_shared_plan(GqaSharedArgs a) {
  __shared__ int lens[kPlanLds], sums[kPlanThreads / kWave];
  __shared__ int running;
  const GqaPagedArgs &p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  bool bad = false;
  for (int g = tid; g <= a.G; g += kPlanThreads) {
    const int at = a.starts[g];
    bad |= at < 0 || at > p.B || (g > 0 && at < a.starts[g - 1]);
  }
  for (int b = tid; b < p.B; b += kPlanThreads) {
    if (b < kPlanLds) lens[b] = length_of(p, b);
    a.group_of[b] = -1;
    a.skips[b] = 0;
  }
  if (tid == 0) running = 0;
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) atomicOr(p.status, GQA_STATUS_BAD_BOUNDS);
  const int rows_per = p.Hq / p.Hkv;
  for (int g = wave; g < a.G; g += kPlanThreads / kWave) {
    const int first = bad ? 0 : a.starts[g], last = bad ? 0 : a.starts[g + 1], wanted = a.prefixes[g];
    int least = 0x7fffffff, live = 0, source = 0x7fffffff;
    for (int b = first + lane; b < last; b += kWave) {
      const int len = b < kPlanLds ? lens[b] : length_of(p, b);
      if (len > 0) {
        least = min(least, len);
        source = min(source, b);
        ++live;
      }
    }
    least = wave_least(least);
    source = wave_least(source);
    live = wave_sum_i(live);
    const int keys = live < 2 ? 0 : max(0, min(wanted, least)) / kBlock * kBlock;
    for (int b = first + lane; b < last; b += kWave) {
      const int len = b < kPlanLds ? lens[b] : length_of(p, b);
      a.group_of[b] = g;
      a.skips[b] = len > 0 ? keys : 0;
    }
    if (lane == 0) {
      if (wanted < 0) atomicOr(p.status, GQA_STATUS_BAD_BOUNDS);
      a.first[g] = first;
      a.first[g + 1] = last;  // the next group writes the same
      a.source[g] = live ? source : 0;
      a.steps[g] = (keys + kStep - 1) / kStep;
    }
  }
  __syncthreads();
  // Steps before each group's.
  for (int base = 0; base < a.G; base += kPlanThreads) {
    const int g = base + tid;
    int mine = 0;
    if (g < a.G) {
      const int first = bad ? 0 : a.starts[g], last = bad ? 0 : a.starts[g + 1];
      mine = a.steps[g] * p.Hkv * ((int)(((int64_t)(last - first) * rows_per + kSharedRows - 1) / kSharedRows));
    }
    const int incl = wave_scan(mine);
    if (lane == kWave - 1) sums[wave] = incl;
    __syncthreads();
    int before = running, all = 0;
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      before += w < wave ? sums[w] : 0;
      all += sums[w];
    }
    if (g < a.G) a.at[g] = before + incl - mine;
    __syncthreads();
    if (tid == 0) running += all;
    __syncthreads();
  }
  if (tid == 0) {
    a.at[a.G] = running;
    *a.total = running;
  }
}

// A group's unit of work at a step of the list: KV head and rows, the step there.
struct Unit {
  int g, kvh, tile, s, steps;
};
__device__ __forceinline__ Unit unit_at(const GqaSharedArgs &a, int x) {
  int lo = 0, hi = a.G - 1;  // the last group with at most x steps before it has steps
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.at[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  const int rows = (a.first[lo + 1] - a.first[lo]) * (a.p.Hq / a.p.Hkv), tiles = (rows + kSharedRows - 1) / kSharedRows;
  const int steps = a.steps[lo], rest = x - a.at[lo], unit = rest / steps;
  return Unit{lo, unit / tiles, unit % tiles, rest % steps, steps};
}

// Row i of a stage's K (V) tile holds its 16-byte chunk c at place c ^ swizzle(i), as in
// the packed kernel: reads meet different bank groups.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swizzle_v(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

template <int D> constexpr int kRing = D == 128 ? 6 : 8;       // stages of 32 keys in LDS
template <int D> constexpr int kTile = kStep * D * 2;          // bytes of a stage's K (or V)
template <int D> constexpr int kPrefixLds = kRing<D> * 2 * kTile<D>;

template <int D, bool F16>
__global__ __launch_bounds__(64 * kWaves, 2) void gqa_shared_prefix(GqaSharedArgs a) {
  constexpr int kSteps = D / 16;                  // QK MFMAs per stage
  constexpr int kDims = D / 32;                   // 32-dim tiles of O
  constexpr int kChunks = D / 8;                  // 16-byte chunks of a row
  constexpr int kLoads = 2 * kTile<D> / 1024 / kWaves;  // per wave and stage: K and V, or one of them
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const GqaPagedArgs &p = a.p;
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
  const int wave = sgpr(threadIdx.x >> 6);
  const int group = p.Hq / p.Hkv, per_page = p.page / kBlock;
  const int total = sgpr(*a.total), per = (total + gridDim.x - 1) / gridDim.x;
  const int64_t begin = (int64_t)blockIdx.x * per;
  if (begin >= total) return;
  const int end = (int)min((int64_t)total, begin + per);
  const uint32_t lds0 = lds_addr(smem);
  const float sl2 = p.scale * kLog2e;
  bool bad_page = false;

  // The wave's part of a stage: 1 KiB of K and of V, or of one of them, whole rows of one
  // 16-key block.
  constexpr int kRowsOfLoad = 1024 / (2 * D);
  const int part = kLoads == 2 ? wave : wave % (kWaves / 2), block = part * kRowsOfLoad / kBlock;
  const int row_in_tile = part * kRowsOfLoad + lane / kChunks, place = lane % kChunks;
  const uint32_t k_off[1] = {(uint32_t)(row_in_tile % kBlock) * (uint32_t)(2 * p.k_row) + 16 * (place ^ swizzle_k<D>(row_in_tile))};
  const uint32_t v_off[1] = {(uint32_t)(row_in_tile % kBlock) * (uint32_t)(2 * p.v_row) + 16 * (place ^ swizzle_v<D>(row_in_tile))};
  // K fragment ks: row r, chunk 2 ks + h.  V: the lane addresses dims 16 (gi % 2)
  // + 4 x .. of 32, key 4 h + c.
  const uint32_t k_at = (uint32_t)(r * 2 * D + 16 * (h ^ swizzle_k<D>(r)));
  const int v_key = 4 * h + ((lane >> 2) & 3), v_chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_at = (uint32_t)(kTile<D> + v_key * 2 * D + 16 * (v_chunk ^ swizzle_v<D>(v_key)) + 8 * (lane & 1));

  for (int x = (int)begin; x < end;) {
    const Unit u = unit_at(a, x);
    const int g = sgpr(u.g), kvh = sgpr(u.kvh), tile = sgpr(u.tile), s0 = sgpr(u.s);
    const int s1 = min(sgpr(u.steps), s0 + end - x);
    const int first = sgpr(a.first[g]), rows = (sgpr(a.first[g + 1]) - first) * group;
    const int source = sgpr(a.source[g]), keys = sgpr(p.B > 0 ? a.skips[source] : 0);
    const int32_t *const table = p.tables + (int64_t)source * p.table_stride;
    const int row0 = tile * kSharedRows + kWaveRows * wave;
    const bool own = row0 < rows;

    // Rows of Q, one per lane pair; those behind the last are the last again.
    const int row = min(row0 + r, rows - 1), member = row / group, head = kvh * group + row - member * group;
    u32x4 qf[kSteps];
    {
      const uint16_t *const qp = p.q + (int64_t)(first + member) * p.q_stride + (int64_t)head * D + 8 * h;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) qf[ks] = *(const u32x4 *)(qp + 16 * ks);
    }

    // Blocks of the stages in flight that are there, two bits each, the last loaded lowest.
    uint32_t there = 0;
    int loaded = s0;
    auto issue = [&]() __attribute__((always_inline)) {
      uint32_t bits = 0;
      const uint16_t *k_base = p.k, *v_base = p.v;
      bool mine = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int blk = 2 * loaded + i;
        if (blk * kBlock < keys) {
          const int page = uniform_load(table + blk / per_page);
          const bool ok = (uint32_t)page < (uint32_t)p.P;
          bits |= ok ? 1u << i : 0u;
          bad_page |= !ok;
          if (i == block && ok) {
            const int64_t at = blk % per_page * kBlock;
            mine = true;
            k_base = p.k + page * p.k_page + kvh * p.k_head + at * p.k_row;
            v_base = p.v + page * p.v_page + kvh * p.v_head + at * p.v_row;
          }
        }
      }
      there = there << 2 | bits;
      const uint32_t slot = lds0 + (uint32_t)((loaded - s0) % kRing<D>) * (2 * kTile<D>) + part * 1024;
      const uint32_t k_bytes = mine ? 15u * (uint32_t)(2 * p.k_row) + 2 * D : 0u, v_bytes = mine ? 15u * (uint32_t)(2 * p.v_row) + 2 * D : 0u;
      if (kLoads == 2 || wave < kWaves / 2) load_lds(buffer_words(k_base, k_bytes), sgpr((int)slot), k_off);
      if (kLoads == 2 || wave >= kWaves / 2) load_lds(buffer_words(v_base, v_bytes), sgpr((int)(slot + kTile<D>)), v_off);
      ++loaded;
    };

    float m_run = -INFINITY, l_run = 0.f, m_top = -INFINITY;
    f32x16 o[kDims];
#pragma unroll
    for (int db = 0; db < kDims; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.f;

    for (int i = 0; i < kRing<D> - 1 && loaded < s1; ++i) issue();
    for (int st = s0; st < s1; ++st) {
      // The wave's part of this stage has landed once at most those of the later ones
      // remain; then the others' too, and nobody reads the stage before any more.
      if (st + kRing<D> - 2 < s1) wait_vmcnt<(kRing<D> - 2) * kLoads>();
      else wait_vmcnt<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (loaded < s1) issue();
      if (!own) continue;
      const uint32_t slot = lds0 + (uint32_t)((st - s0) % kRing<D>) * (2 * kTile<D>);
      const uint32_t bits = there >> 2 * (loaded - 1 - st) & 3u;
      f32x16 s;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks) s = mfma32x32<F16>(lds_b128((slot + k_at) ^ (32 * ks)), qf[ks], s);
      mfma_settle();  // read on both sides of a branch
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = pin(s[i]);
      if (bits != 3u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = bits >> (i >> 3) & 1u ? s[i] : -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
      top *= sl2;
      if (__builtin_amdgcn_ballot_w64(top > (F16 ? m_top : limit<F16>(m_run)))) {
        mfma_settle();
        const f32x2_t both = halves(top);
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
      // Probabilities in the type of V: half a step each, see reference(), against fp32
      // sums of both.
      u32x4 pb[2];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], sl2, neg_m));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], sl2, neg_m));
        pb[i / 4][i % 4] = pack2<F16>(e0, e1);
        sum += e0 + e1;
      }
      l_run += sum;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int db = 0; db < kDims; ++db) {
          const uint32_t at = ((slot + v_at) ^ (64 * db)) + j * 32 * D;
          const u32x2 lo = lds_tr16(at), hi = lds_tr16(at + 16 * D);
          o[db] = mfma32x32<F16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pb[j], o[db]);
        }
    }
    mfma_settle();
    if (own) {
      const f32x2_t both = halves(l_run);
      if (row0 + r < rows) {
        float *const to = s0 > 0 ? a.more + ((int64_t)blockIdx.x * kSharedRows + kWaveRows * wave + r) * (D + 2)
                                 : a.heads + ((int64_t)(first + member) * p.Hq + head) * (D + 2);
        if (h == 0) *(f32x2_t *)to = f32x2_t{m_run, both[0] + both[1]};
        // Lane (r, h) holds dims 32 db + 8 q + 4 h + i of its row.
#pragma unroll
        for (int db = 0; db < kDims; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float *const op = to + 2 + 32 * db + 8 * q + 4 * h;
            *(f32x2_t *)op = f32x2_t{pin(o[db][4 * q]), pin(o[db][4 * q + 1])};
            *(f32x2_t *)(op + 2) = f32x2_t{pin(o[db][4 * q + 2]), pin(o[db][4 * q + 3])};
          }
      }
    }
    x += s1 - s0;
    // The next unit's loads are counted from here, into slots that nobody reads.
    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  if (bad_page && threadIdx.x == 0) atomicOr(p.status, GQA_STATUS_BAD_PAGE);
}

struct State {
  float m, l;
  f32x2_t o;
};

// A row's pieces: of the prefix, then of the keys behind, each in their order.  A thread
// takes two elements of O of all pieces, or, where there are too few elements to fill the
// chip, of every groups-th piece, and the groups are joined in order.
template <bool F16>
__global__ __launch_bounds__(kMergeThreads) void gqa_shared_join(GqaSharedArgs a, int chunk, int workgroups) {
  __shared__ State states[kMergeThreads];
  const GqaPagedArgs &p = a.p;
  constexpr int kRows = 16;  // query heads of a piece of the rest
  const int group = p.Hq / p.Hkv, blocks = (group + kRows - 1) / kRows, heads = p.Hkv * blocks;
  const int b = blockIdx.x / heads, head = blockIdx.x % heads, kvh = head / blocks, part = head % blocks;
  const int rows = min(group, kRows * (part + 1)) - kRows * part, per_slot = min(group, kRows), groups = kMergeThreads / chunk;
  const int e = 2 * (blockIdx.y * chunk + threadIdx.x % chunk), mine = threadIdx.x / chunk;  // element, group
  const int half = p.D == 128 ? 7 : 6;                                                       // log2 D
  const bool live = e < rows * p.D;
  const int row = live ? e >> half : 0, d = e & (p.D - 1), qh = kvh * group + kRows * part + row;
  const int64_t record = p.D + 2;

  const int skip = a.skips[b], len = length_of(p, b);
  int in_prefix = 0, from = 0, at = 0;  // pieces of the prefix, the workgroup of the first, the row in its tile
  if (skip > 0) {
    const int g = a.group_of[b], place = (b - a.first[g]) * group + kRows * part + row, tile = place / kSharedRows;
    const int tiles = ((a.first[g + 1] - a.first[g]) * group + kSharedRows - 1) / kSharedRows;
    const int per = (*a.total + workgroups - 1) / workgroups, begin = a.at[g] + (kvh * tiles + tile) * a.steps[g];
    from = begin / per;
    in_prefix = (begin + a.steps[g] - 1) / per - from + 1;
    at = place % kSharedRows;
  }
  const int slot = a.p.pieces[2 * blockIdx.x], behind = len > skip ? p.pieces[2 * blockIdx.x + 1] : 0;
  const int n = in_prefix + behind;
  auto piece = [&](int i) __attribute__((always_inline)) {
    if (i < in_prefix)
      return i ? a.more + ((int64_t)(from + i) * kSharedRows + at) * record : a.heads + ((int64_t)b * p.Hq + qh) * record;
    const int j = i - in_prefix, s = j ? (slot / 2 + j) * 2 : slot;
    return p.partial + ((int64_t)s * per_slot + row) * record;
  };
  State st = {-INFINITY, 0.f, f32x2_t{0.f, 0.f}};
  for (int i = mine; i < n; i += groups * kBatch) {
    f32x2_t ml[kBatch], x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float *const y = piece(min(i + j * groups, n - 1));
      ml[j] = *(const f32x2_t *)y;
      x[j] = *(const f32x2_t *)(y + 2 + d);
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
  if (live) *(uint32_t *)(p.out + ((int64_t)b * p.Hq + qh) * p.D + d) = pack2<F16>(st.o[0] * inv, st.o[1] * inv);
}

template <int D, bool F16>
hipError_t launch(const GqaSharedArgs &a, int cus, hipStream_t s) {
  auto prefix = gqa_shared_prefix<D, F16>;
  static std::atomic<uint64_t> allowed{0};
  if (const hipError_t e = allow_lds((const void *)prefix, kPrefixLds<D>, &allowed)) return e;
  hipLaunchKernelGGL(gqa_shared_plan, dim3(1), dim3(kPlanThreads), 0, s, a);
  if (a.G > 0) hipLaunchKernelGGL(prefix, dim3(cus), dim3(64 * kWaves), kPrefixLds<D>, s, a);
  if (const hipError_t e = launch_gqa_shared_rest(a.p, cus, s)) return e;
  const int group = a.p.Hq / a.p.Hkv, pairs = a.p.B * a.p.Hkv * ((group + 15) / 16), need = (group < 16 ? group : 16) * D / 2;
  int chunk = kMergeThreads;
  while (chunk > 16 && (chunk >= 2 * need || (int64_t)pairs * ((need + chunk - 1) / chunk) < cus)) chunk /= 2;
  hipLaunchKernelGGL(gqa_shared_join<F16>, dim3(pairs, (need + chunk - 1) / chunk), dim3(kMergeThreads), 0, s, a, chunk, cus);
  return hipGetLastError();
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Places in the workspace: {status words; the total; skips; groups; first members, sources,
// steps, steps before; two words per (sequence, 16 heads) and the states of the rest; the
// states of the prefixes by row; those by workgroup}.
struct Layout {
  size_t total, skips, group_of, groups[4], pieces, partial, heads, more, bytes;
};
Layout layout_of(int B, int Hq, int Hkv, int D, int G, int cus) {
  const int group = Hq / Hkv, rows = group < 16 ? group : 16;
  const size_t pairs = (size_t)B * Hkv * ((group + 15) / 16), record = (size_t)(D + 2) * sizeof(float);
  Layout l;
  size_t at = 256;
  auto take = [&](size_t *where, size_t bytes) {
    *where = at;
    at += align256(bytes);
  };
  take(&l.total, 4);
  take(&l.skips, (size_t)B * 4);
  take(&l.group_of, (size_t)B * 4);
  for (size_t &g : l.groups) take(&g, ((size_t)G + 1) * 4);
  take(&l.pieces, 8 * pairs);
  take(&l.partial, (2 * (size_t)gqa_shared_rest_waves(D, cus) + pairs) * rows * record);
  take(&l.heads, (size_t)B * Hq * record);
  take(&l.more, (size_t)cus * kSharedRows * record);
  l.bytes = at;
  return l;
}

}  // namespace

size_t gqa_shared_workspace(int B, int Hq, int Hkv, int D, int G, int cus) { return layout_of(B, Hq, Hkv, D, G, cus).bytes; }

void gqa_shared_bind(GqaSharedArgs *a, void *workspace, int cus) {
  uint8_t *const w = (uint8_t *)workspace;
  const Layout l = layout_of(a->p.B, a->p.Hq, a->p.Hkv, a->p.D, a->G, cus);
  a->p.status = (uint32_t *)w;
  a->total = (int32_t *)(w + l.total);
  a->skips = (int32_t *)(w + l.skips);
  a->group_of = (int32_t *)(w + l.group_of);
  int32_t **const groups[4] = {&a->first, &a->source, &a->steps, &a->at};
  for (int i = 0; i < 4; ++i) *groups[i] = (int32_t *)(w + l.groups[i]);
  a->p.skips = a->skips;
  a->p.pieces = (int32_t *)(w + l.pieces);
  a->p.partial = (float *)(w + l.partial);
  a->heads = (float *)(w + l.heads);
  a->more = (float *)(w + l.more);
}

hipError_t launch_gqa_shared(const GqaSharedArgs &a, int cus, hipStream_t s) {
  if (a.p.D == 128) return a.p.dtype == GQA_FP16 ? launch<128, true>(a, cus, s) : launch<128, false>(a, cus, s);
  return a.p.dtype == GQA_FP16 ? launch<64, true>(a, cus, s) : launch<64, false>(a, cus, s);
}

}  // namespace moe
