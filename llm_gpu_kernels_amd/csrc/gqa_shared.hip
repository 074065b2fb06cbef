// Attention of one new token per sequence over a paged cache, where groups of sequences
// start with the same keys (samples of one prompt, users of one instruction), on gfx950.
//
// Tables that are wide for the rows are worked on in two launches; of narrow ones
// every row goes by itself (gqa_shared_by_rows() has the rule).
//
// softmax(q K^T) V over a prefix and the rest of a row's keys is joined from the two
// parts' (max, sum, O), so a prefix is read once for all rows of its group: up to 128
// query rows (the members' heads of one KV head) are one workgroup's, 32 per wave, and K
// and V go through LDS for all of them.  With few rows its bytes bound it, with some
// hundreds the matrix cores.  The keys behind the prefix are worked on as
// gqa_paged.hip works on whole rows.
//
//   plan    the keys that each group shares, and how they are cut into chunks, so that the
//           units of work, (group, KV head, chunk, up to 128 rows), are as many as the
//           workgroups for them.  Up to 64 groups and 256 sequences every workgroup finds
//           that out by itself, else one does before;
//   work    one launch for both parts, which fill the chip together: a unit per workgroup
//           of the first ones; gqa_paged.hip's list of steps over the keys behind, a range
//           per wave of the others.  Every piece leaves its states;
//   join    all pieces' states of a row in the order of the keys.
//
// Measured, 32 query and 8 KV heads of 128, a copy of 2 GiB running at 5.1 TB/s: four groups
// of 22 to 40 sequences, prefixes of 4995 to 11383 keys, up to 600 keys of their own (186 MB)
// 63.2 us (by gqa_paged.hip 593), of which the plan 4 and the join 7; the prefixes alone 59,
// the rest alone 36.  The loads alone and the products alone take 9 in 10 of that each, the
// states 5: a stage of two tiles on a CU takes 1.07, the packed kernel's 1.0, and tiles of less
// than 128 rows leave SIMDs without work.  Eight sequences with one prefix of 1500 keys, row
// by row, 11.7.
#include "common.h"
#include "../../include/gqa_mi355x.h"
#include "gqa_dev.h"
#include "gqa_internal.h"
#include "gqa_prefix_dev.h"

namespace moe {

using namespace gqa;
using shared::length_of;
using shared::steps_of;

namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave;
constexpr int kRows = 16;       // query heads of a piece of the rest
constexpr int kMergeThreads = 256, kBatch = 16;

// A thread per group, and one per row of the batch.
static_assert(kMaxGroups <= kPlanThreads, "a thread per group");
__global__ __launch_bounds__(kPlanThreads) void gqa_shared_plan(GqaPagedArgs p, int workgroups) {
  __shared__ int starts[kMaxGroups + 1], least[kMaxGroups], live[kMaxGroups], source[kMaxGroups];
  __shared__ shared::Group groups[kMaxGroups];
  __shared__ int sums[2][kPlanWaves], fits[kPlanWaves];
  __shared__ unsigned long long shared_steps, rest_steps;
  static_assert(kPlanWaves == shared::kSizes, "a wave per size");
  const GqaSharedState &st = p.shared;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per_head = p.Hq / p.Hkv, G = st.G;
  for (int g = tid; g <= G; g += kPlanThreads) starts[g] = st.starts[g];
  const int wanted = tid < G ? st.prefixes[tid] : 0;
  if (tid < G) {
    least[tid] = source[tid] = 0x7fffffff;
    live[tid] = 0;
  }
  if (tid == 0) shared_steps = rest_steps = 0;
  __syncthreads();
  bool wrong = false;
  for (int g = tid; g <= G; g += kPlanThreads) wrong |= starts[g] < 0 || starts[g] > p.B || (g > 0 && starts[g] < starts[g - 1]);
  const bool bad = __syncthreads_or(wrong);
  if ((bad && tid == 0) || wanted < 0) atomicOr(p.status, GQA_STATUS_BAD_BOUNDS);
  // The group of a row; -1: none.
  auto group_of = [&](int b) {
    if (bad || G == 0 || b < starts[0] || b >= starts[G]) return -1;
    int lo = 0, hi = G - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (starts[mid] <= b) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  for (int b = tid; b < p.B; b += kPlanThreads) {
    const int g = group_of(b), len = length_of(p, b);
    // Here, since where no key lies behind a prefix the list has no workgroup that would.
    if (p.lengths[b] != len) atomicOr(p.status, GQA_STATUS_BAD_BOUNDS);
    if (g < 0 || len == 0) continue;
    atomicMin(least + g, len);
    atomicMin(source + g, b);
    atomicAdd(live + g, 1);
  }
  __syncthreads();
  shared::Group mine = {};
  if (tid < G) {
    mine.first = bad ? 0 : starts[tid];
    mine.rows = bad ? 0 : (starts[tid + 1] - mine.first) * per_head;
    shared::share(&mine, wanted, least[tid], live[tid]);
    mine.source = mine.keys ? source[tid] : 0;
    groups[tid] = mine;
    if (mine.keys) atomicAdd(&shared_steps, (unsigned long long)steps_of(mine.keys) * mine.tiles * p.Hkv);
  }
  __syncthreads();
  unsigned long long rest = 0;  // steps of the keys that no group has
  for (int b = tid; b < p.B; b += kPlanThreads) {
    const int g = group_of(b), len = length_of(p, b);
    rest += steps_of(len - (g >= 0 && len > 0 ? groups[g].keys : 0));
  }
  if (rest) atomicAdd(&rest_steps, rest);
  __syncthreads();
  const int64_t all_shared = (int64_t)shared_steps;
  const int n = shared::share_of(all_shared, (int64_t)rest_steps * p.Hkv * ((per_head + kRows - 1) / kRows), workgroups);
  const int size = shared::chunk_size(all_shared, n, wave);
  int units = 0;
  for (int g = lane; g < G; g += kWave) units += groups[g].tiles * p.Hkv * ((steps_of(groups[g].keys) + size - 1) / size);
  units = wave_total(units);
  if (lane == 0) fits[wave] = units <= n;
  __syncthreads();
  int chosen = 0;
  while (chosen < kPlanWaves && !fits[chosen]) ++chosen;
  shared::cut(&mine, shared::chunk_size(all_shared, n, chosen < kPlanWaves ? chosen : 0));
  const int per_chunk = mine.tiles * p.Hkv, own = mine.chunks * per_chunk, extra = max(0, own - per_chunk);
  const int incl = wave_scan(own), incl_extra = wave_scan(extra);
  if (lane == kWave - 1) {
    sums[0][wave] = incl;
    sums[1][wave] = incl_extra;
  }
  __syncthreads();
  mine.before = incl - own;
  mine.more = incl_extra - extra;
  int all = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    mine.before += w < wave ? sums[0][w] : 0;
    mine.more += w < wave ? sums[1][w] : 0;
    all += sums[0][w];
  }
  if (tid < G) {
    groups[tid] = mine;
    int32_t *const rec = st.groups + 16 * tid;
    *(int4 *)rec = make_int4(mine.before, mine.chunk_steps, mine.first, mine.rows);
    *(int4 *)(rec + 4) = make_int4(mine.source, mine.keys, mine.tiles, mine.tile_rows);
    *(int2 *)(rec + 8) = make_int2(mine.chunks, mine.more);
  }
  if (tid == 0) {
    st.header[0] = all;
    st.header[1] = n;
  }
  __syncthreads();
  for (int b = tid; b < p.B; b += kPlanThreads) {
    const int g = group_of(b);
    const shared::Group x = groups[max(g, 0)];
    int32_t *const rec = st.rows + 8 * b;
    *(int4 *)rec = make_int4(g >= 0 && length_of(p, b) > 0 ? x.keys : 0, x.chunks, x.tiles, x.tile_rows);
    *(int2 *)(rec + 4) = make_int2((b - x.first) * per_head, x.more);
  }
}

struct State {
  float m, l;
  f32x2_t o;
};

// A row's pieces: of the prefix, then of the keys behind, each in their order.  A thread
// takes two elements of O of all pieces, or, where there are too few elements to fill the
// chip, of every groups-th piece, and the groups are joined in order.
template <bool F16>
__global__ __launch_bounds__(kMergeThreads) void gqa_shared_join(GqaPagedArgs p, int chunk) {
  __shared__ State states[kMergeThreads];
  const GqaSharedState &a = p.shared;
  const int group = a.group, blocks = (group + kRows - 1) / kRows, heads = p.Hkv * blocks;
  const int b = blockIdx.x / heads, head = blockIdx.x % heads, kvh = head / blocks, part = head % blocks;
  const int rows = min(kRows, group - kRows * part), per_slot = min(group, kRows), groups = kMergeThreads / chunk;
  const int e = 2 * (blockIdx.y * chunk + threadIdx.x % chunk), mine = threadIdx.x / chunk;  // element, group
  const int half = p.D == 128 ? 7 : 6;                                                       // log2 D
  const bool live = e < rows * p.D;
  const int row = live ? e >> half : 0, d = e & (p.D - 1), qh = kvh * group + kRows * part + row;
  const int64_t record = p.D + 2;

  // (All at once: a launch of small loads is as long as its chain of them.)
  const int32_t *const rec = a.rows + 8 * b;
  const int skip = uniform_load(rec), of_chunks = uniform_load(rec + 1), tiles = uniform_load(rec + 2);
  const int tile_rows = uniform_load(rec + 3), first_row = uniform_load(rec + 4), more = uniform_load(rec + 5);
  const int len = length_of(p, b), slot = p.pieces[2 * blockIdx.x], left = p.pieces[2 * blockIdx.x + 1];
  int chunks = 0;
  int64_t at = 0, apart = 0;  // of the second chunk's record, between two chunks'
  if (skip > 0) {
    chunks = of_chunks;
    const int place = first_row + kRows * part + row, tile = place / tile_rows;
    at = ((int64_t)(more + kvh * (chunks - 1) * tiles + tile) * kSharedRows + place - tile * tile_rows) * record;
    apart = (int64_t)tiles * kSharedRows * record;
  }
  const int n = chunks + (len > skip ? left : 0);
  auto piece = [&](int i) __attribute__((always_inline)) {
    if (i < chunks) return i ? a.more + at + (i - 1) * apart : a.heads + ((int64_t)b * p.Hq + qh) * record;
    const int j = i - chunks, s = j ? (slot / 2 + j) * 2 : slot;
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

size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// Places in the workspace, in the order of the members; partial: two pieces of a wave, and
// one of every (sequence, 16 heads).
struct Layout {
  size_t header, groups, rows, pieces, partial, heads, more, bytes;
};
Layout layout_of(int B, int Hq, int Hkv, int D, int G, int cus) {
  const int group = Hq / Hkv, rows = group < kRows ? group : kRows;
  const size_t pairs = (size_t)B * Hkv * ((group + kRows - 1) / kRows), record = (size_t)(D + 2) * sizeof(float);
  const size_t workgroups = gqa_shared_workgroups(D, cus);
  Layout l;
  size_t at = 256;  // the status words
  auto take = [&](size_t *where, size_t bytes) {
    *where = at;
    at += align256(bytes);
  };
  take(&l.header, 8);
  take(&l.groups, (size_t)G * 64);
  take(&l.rows, (size_t)B * 32);
  take(&l.pieces, 8 * pairs);
  take(&l.partial, (2 * 4 * workgroups + pairs) * rows * record);
  take(&l.heads, (size_t)B * Hq * record);
  take(&l.more, workgroups * kSharedRows * record);
  l.bytes = at;
  return l;
}

}  // namespace

size_t gqa_shared_workspace(int B, int Hq, int Hkv, int D, int64_t keys, int G, int cus) {
  return gqa_shared_by_rows(B, Hq, Hkv, D, keys, cus) ? 256 : layout_of(B, Hq, Hkv, D, G, cus).bytes;
}

void gqa_shared_bind(GqaPagedArgs *a, int G, const int32_t *starts, const int32_t *prefixes, void *workspace, int cus) {
  uint8_t *const w = (uint8_t *)workspace;
  const int per_page = a->page / 16;
  a->status = (uint32_t *)w;
  a->shared = GqaSharedState{G, G <= shared::kLocalGroups && a->B <= shared::kLocalRows, starts, prefixes, nullptr, nullptr,
                             nullptr, nullptr, nullptr, a->Hq / a->Hkv, per_page & (per_page - 1) ? -1 : __builtin_ctz(per_page)};
  if (gqa_shared_by_rows(a->B, a->Hq, a->Hkv, a->D, (int64_t)a->M * a->page, cus)) return;
  const Layout l = layout_of(a->B, a->Hq, a->Hkv, a->D, G, cus);
  a->pieces = (int32_t *)(w + l.pieces);
  a->partial = (float *)(w + l.partial);
  a->shared.header = (int32_t *)(w + l.header);
  a->shared.groups = (int32_t *)(w + l.groups);
  a->shared.rows = (int32_t *)(w + l.rows);
  a->shared.heads = (float *)(w + l.heads);
  a->shared.more = (float *)(w + l.more);
}

hipError_t launch_gqa_shared(const GqaPagedArgs &p, int cus, hipStream_t s) {
  if (gqa_shared_by_rows(p.B, p.Hq, p.Hkv, p.D, (int64_t)p.M * p.page, cus)) return launch_gqa_shared_rows(p, s);
  if (!p.shared.local)
    hipLaunchKernelGGL(gqa_shared_plan, dim3(1), dim3(kPlanThreads), 0, s, p, gqa_shared_workgroups(p.D, cus));
  if (const hipError_t e = launch_gqa_shared_work(p, cus, s)) return e;
  const int group = p.Hq / p.Hkv, pairs = p.B * p.Hkv * ((group + kRows - 1) / kRows), need = (group < kRows ? group : kRows) * p.D / 2;
  int chunk = kMergeThreads;
  while (chunk > 16 && (chunk >= 2 * need || (int64_t)pairs * ((need + chunk - 1) / chunk) < cus)) chunk /= 2;
  hipLaunchKernelGGL(p.dtype == GQA_FP16 ? gqa_shared_join<true> : gqa_shared_join<false>,
                     dim3(pairs, (need + chunk - 1) / chunk), dim3(kMergeThreads), 0, s, p, chunk);
  return hipGetLastError();
}

}  // namespace moe
