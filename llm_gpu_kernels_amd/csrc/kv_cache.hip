// Paged key-value cache on gfx950: pages handed out, shared, given back and
// moved, and the keys and values of new tokens written to their slots.
//
// All decisions are integer work over a few thousand words and are taken by one
// workgroup (no grid-wide synchronisation, and the pages come out in the same
// order every time); what moves bytes (copies of pages, slots, table rows) is a
// second launch over the whole chip that reads the decisions.  The decisions are
// bound by latency (the launch and the chain of dependent loads), the moves by HBM;
// a copy of 2 GiB runs at 5.0 TB/s.
#include "common.h"
#include "../../include/kv_mi355x.h"
#include "kv_internal.h"

namespace moe {

namespace {

constexpr int kPlanThreads = 1024;  // one row of the cache each
constexpr int kWaves = kPlanThreads / kWave;
constexpr int kScanPages = 8;       // pages of a thread per scanned chunk
static_assert(KV_MAX_SEQUENCES <= kPlanThreads, "a thread per row");

// (Unsigned: a row's tokens go up to 2^31 - 1, a page's up to 1024.)
__device__ __forceinline__ int ceil_div(int a, int b) { return (int)(((uint32_t)a + b - 1u) / (uint32_t)b); }

// Exclusive sums over the workgroup's threads of two numbers and of a flag, and the
// totals.
struct Scan {
  int a, b, flag, all_a, all_b, all_flag;
};
struct ScanLds {
  int a[kWaves], b[kWaves], flag[kWaves];
};
__device__ __forceinline__ Scan block_scan(int a, int b, bool flag, ScanLds *lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ia = wave_scan(a), ib = wave_scan(b);
  const uint64_t set = __builtin_amdgcn_ballot_w64(flag);
  __syncthreads();  // the last scan's sums have been read
  if (lane == kWave - 1) {
    lds->a[wave] = ia;
    lds->b[wave] = ib;
    lds->flag[wave] = (int)__popcll(set);
  }
  __syncthreads();
  Scan r = {ia - a, ib - b, (int)__popcll(set & lanemask_lt()), 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int wa = lds->a[w], wb = lds->b[w], wf = lds->flag[w];
    r.a += w < wave ? wa : 0;
    r.b += w < wave ? wb : 0;
    r.flag += w < wave ? wf : 0;
    r.all_a += wa;
    r.all_b += wb;
    r.all_flag += wf;
  }
  return r;
}

// One bit per page of a thread's eight: in use.
__device__ __forceinline__ uint32_t used_bits(const KvState &s, int first) {
  uint32_t bits = 0;
  if (first + kScanPages <= s.pages) {
    const int4 a = *(const int4 *)(s.refs + first), b = *(const int4 *)(s.refs + first + 4);
    bits = (a.x > 0) | (a.y > 0) << 1 | (a.z > 0) << 2 | (a.w > 0) << 3 | (b.x > 0) << 4 | (b.y > 0) << 5 |
           (b.z > 0) << 6 | (b.w > 0) << 7;
  } else {
#pragma unroll
    for (int i = 0; i < kScanPages; ++i)
      if (first + i < s.pages && s.refs[first + i] > 0) bits |= 1u << i;
  }
  return bits;
}
__device__ __forceinline__ uint32_t valid_bits(const KvState &s, int first) {
  const int n = s.pages - first;
  return n >= kScanPages ? 0xffu : n > 0 ? (1u << n) - 1u : 0u;
}

// Pages, lengths and slots of a reserve.  Thread s is row s.  One workgroup, so
// what bounds it is the chain of dependent loads: the first pages' holders are
// loaded beside the rows, and short lists of pages stay in LDS.  128 rows that grow by
// a token on shared pages: 7.9 us.
constexpr int kListLds = 4096;
__global__ __launch_bounds__(kPlanThreads) void kv_reserve_plan(KvState s, const int32_t *counts, int stride) {
  __shared__ ScanLds sums;
  __shared__ __attribute__((aligned(16))) int last_page[kPlanThreads];
  __shared__ int need_at[kPlanThreads], row_len[kPlanThreads];
  __shared__ int copy_at[kPlanThreads];  // the row's copy's number, -1: none
  __shared__ int list_lds[kListLds];
  const int row = threadIdx.x;
  const bool live = row < s.sequences;
  const int cap = s.max_pages * s.page_size;  // < 2^31
  int len = live ? s.lengths[row] : 0, count = live ? counts[row] : 0;
  uint32_t used0 = row * kScanPages < s.pages ? used_bits(s, row * kScanPages) : 0u;
  uint32_t bad = 0;
  if (len < 0 || len > cap) {
    bad |= KV_STATUS_BAD_STATE;
    len = 0;
  }
  if (count < 0 || count > s.max_tokens || (stride > 0 && count > stride)) {
    bad |= KV_STATUS_BAD_COUNT;
    count = 0;
  }
  if (count > cap - len) {
    bad |= KV_STATUS_TOO_LONG;
    count = 0;
  }
  // A shared, partly filled last page.
  int last = -1, holders = 0;
  if (count > 0 && len % s.page_size) {
    const int p = s.tables[(int64_t)row * s.max_pages + len / s.page_size];
    if (p < 0 || p >= s.pages) {
      bad |= KV_STATUS_BAD_STATE;
    } else if ((holders = s.refs[p]) > 1) {
      last = p;
    }
  }
  last_page[row] = last;
  row_len[row] = len;
  bool copy = last >= 0;
  __syncthreads();
  if (__builtin_amdgcn_ballot_w64(copy)) {
    int growing = 0, later = -1;  // rows that grow on this page, the last of them
#pragma unroll 4
    for (int j = 0; j < s.sequences; j += 4) {
      const int4 p = *(const int4 *)(last_page + j);
      growing += (p.x == last) + (p.y == last) + (p.z == last) + (p.w == last);
      later = p.x == last ? j : later;
      later = p.y == last ? j + 1 : later;
      later = p.z == last ? j + 2 : later;
      later = p.w == last ? j + 3 : later;
    }
    copy = copy && (growing < holders || later > row);
  }
  const int used = ceil_div(len, s.page_size);
  const int need = ceil_div(len + count, s.page_size) - used + copy;  // <= 2^16 + 1
  const Scan sc = block_scan(need, count, copy, &sums);  // sums below 2^27 and 2^31
  const int total = sc.all_a, tokens = sc.all_b;
  if (tokens > s.max_tokens) bad |= KV_STATUS_BAD_COUNT;
  need_at[row] = sc.a;
  copy_at[row] = copy ? sc.flag : -1;

  bool refuse = __syncthreads_or(bad != 0);
  int32_t *const list = total <= kListLds ? list_lds : s.list;
  if (!refuse && total > 0) {
    int found = 0;
    for (int base = 0; base < s.pages && found < total; base += kPlanThreads * kScanPages) {
      const int first = base + row * kScanPages;
      if (base > 0) used0 = first < s.pages ? used_bits(s, first) : 0u;
      uint32_t free_bits = ~used0 & valid_bits(s, first);
      const Scan f = block_scan(__popc(free_bits), 0, false, &sums);
      int at = found + f.a;
      for (; free_bits && at < total; free_bits &= free_bits - 1, ++at) list[at] = first + __ffs(free_bits) - 1;
      found += f.all_a;
    }
    if (found < total) {
      bad |= KV_STATUS_OUT_OF_PAGES;
      refuse = true;
    }
  }
  if (bad) atomicOr(s.status, bad);
  if (refuse) {
    for (int i = row; i <= s.sequences; i += kPlanThreads) s.starts[i] = 0;
    if (row == 0) *s.num_moves = 0;
    return;
  }
  __syncthreads();  // list is complete
  for (int i = row; i < total; i += kPlanThreads) {
    // The row whose pages i lies among: the last one that starts at or before i.
    int lo = 0, hi = s.sequences - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (need_at[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const int page = list[i], nth = i - need_at[lo], c = copy_at[lo], l = row_len[lo];
    int column = ceil_div(l, s.page_size) + nth;
    if (c >= 0) {
      --column;  // the copy takes the last page's place
      if (nth == 0) {
        s.move_src[c] = last_page[lo];
        s.move_dst[c] = page;
        atomicSub(s.refs + last_page[lo], 1);
      }
    }
    s.tables[(int64_t)lo * s.max_pages + column] = page;
    s.refs[page] = 1;
  }
  if (live) {
    s.lengths[row] = len + count;
    s.starts[row] = sc.b;
  }
  if (row == 0) {
    s.starts[s.sequences] = tokens;
    *s.num_moves = sc.all_flag;
  }
}

// Copies the moves' pages in every layer, keys and values, in pieces of kPiece
// bytes that the workgroups take in turn.  A compaction that moves 269 MB: 107 us,
// 5.0 TB/s read and written.
constexpr int kPiece = 16384;
__device__ __forceinline__ void copy_moves(const KvState &s, int block, int blocks) {
  const int n = *s.num_moves;
  if (n == 0) return;
  const int64_t page_bytes = (int64_t)s.kv_heads * s.page_size * s.head_dim * 2;
  const int pieces = (int)((page_bytes + kPiece - 1) / kPiece);
  const int64_t total = (int64_t)n * 2 * s.layers * pieces;
  for (int64_t u = block; u < total; u += blocks) {
    const int piece = (int)(u % pieces);
    const int64_t rest = u / pieces;
    const int plane = (int)(rest % (2 * s.layers)), m = (int)(rest / (2 * s.layers));
    uint8_t *const base = (uint8_t *)(plane < s.layers ? s.k : s.v) +
                          (int64_t)(plane < s.layers ? plane : plane - s.layers) * s.pages * page_bytes +
                          (int64_t)piece * kPiece;
    const uint8_t *const from = base + s.move_src[m] * page_bytes;
    uint8_t *const to = base + s.move_dst[m] * page_bytes;
    const int bytes = (int)min((int64_t)kPiece, page_bytes - (int64_t)piece * kPiece);
    for (int o = threadIdx.x * 16; o < bytes; o += blockDim.x * 16) *(u32x4 *)(to + o) = *(const u32x4 *)(from + o);
  }
}

constexpr int kWideThreads = 256;
constexpr int kCopyBlocks = 1024;

// Slots of the reserved tokens and the copies of shared pages.  96 copies of 131 kB
// (two layers): 5.6 us.
__global__ __launch_bounds__(kWideThreads) void kv_reserve_finish(KvState s, int stride, int slot_blocks) {
  if ((int)blockIdx.x >= slot_blocks) {
    copy_moves(s, blockIdx.x - slot_blocks, gridDim.x - slot_blocks);
    return;
  }
  for (int i = blockIdx.x * kWideThreads + threadIdx.x; i < s.max_tokens; i += slot_blocks * kWideThreads) {
    int row = s.sequences, nth = 0;
    if (stride > 0) {
      row = i / stride;
      nth = i % stride;
    } else if (i < s.starts[s.sequences]) {
      int lo = 0, hi = s.sequences - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s.starts[mid] <= i) lo = mid;
        else hi = mid - 1;
      }
      row = lo;
      nth = i - s.starts[lo];
    }
    int64_t slot = -1;
    if (row < s.sequences) {
      const int count = s.starts[row + 1] - s.starts[row];
      if (nth < count) {
        const int at = s.lengths[row] - count + nth;
        slot = (int64_t)s.tables[(int64_t)row * s.max_pages + at / s.page_size] * s.page_size + at % s.page_size;
      }
    }
    s.slots[i] = slot;
  }
}

// 16 bytes of a token's keys and of its values per thread: whole rows of a head on
// both sides.  8191 tokens of 8 heads of 128 (67 MB read and written): 11.8 us, 5.7 TB/s;
// 64 tokens: 3.0 us, the launch and two dependent loads.
__global__ __launch_bounds__(kWideThreads) void kv_append(KvState s, int layer, const uint16_t *k, const uint16_t *v,
                                                         int64_t k_stride, int64_t v_stride, int n) {
  const int chunks = s.kv_heads * s.head_dim / 8;  // of a token
  const int64_t total = (int64_t)n * chunks;
  const int64_t cells = (int64_t)s.pages * s.page_size, plane = (int64_t)layer * cells * s.kv_heads * s.head_dim;
  for (int64_t u = (int64_t)blockIdx.x * kWideThreads + threadIdx.x; u < total; u += (int64_t)gridDim.x * kWideThreads) {
    const int token = (int)(u / chunks), c = (int)(u % chunks) * 8;
    const int64_t slot = s.slots[token];
    if (slot < 0 || slot >= cells) continue;
    const int head = c / s.head_dim, d = c % s.head_dim;
    const int64_t page = slot / s.page_size;
    const int row = (int)(slot % s.page_size);
    const int64_t to = plane + ((page * s.kv_heads + head) * s.page_size + row) * s.head_dim + d;
    *(u32x4 *)(s.k + to) = *(const u32x4 *)(k + token * k_stride + c);
    *(u32x4 *)(s.v + to) = *(const u32x4 *)(v + token * v_stride + c);
  }
}

// Pages of a row that hold tokens; -1 (and a status) for a length out of range.
__device__ __forceinline__ int row_pages(const KvState &s, int row) {
  const int len = s.lengths[row];
  if (len < 0 || len > s.max_pages * s.page_size) {
    if (threadIdx.x == 0) atomicOr(s.status, KV_STATUS_BAD_STATE);
    return -1;
  }
  return ceil_div(len, s.page_size);
}

// A pair of a fork: 0 if it may go ahead, else why not (KV_STATUS_*; ~0: left out
// by the caller).  Rows are as before the call: lengths are written at its end.
// `named` says that an earlier pair that goes by valid rows names dst.
__device__ __forceinline__ bool fork_rows_valid(const KvState &s, int a, int b) {
  return a >= 0 && b >= 0 && a < s.sequences && b < s.sequences;
}
__device__ __forceinline__ uint32_t fork_status(const KvState &s, int a, int b, bool named) {
  if (a < 0 || b < 0) return ~0u;
  if (!fork_rows_valid(s, a, b)) return KV_STATUS_BAD_ROW;
  return named || s.lengths[b] != 0 ? KV_STATUS_NOT_EMPTY : 0u;
}

// One workgroup per pair: the table row, and one more holder of its pages.  The
// last one to finish sets the lengths: no other reads them any more then.  96 pairs of
// up to 217 pages: 5.2 us (a second launch for the lengths cost 1.4 us more and the
// launch).
__device__ __forceinline__ void fork_lengths(const KvState &s, const int32_t *src, const int32_t *dst, int n);
__global__ __launch_bounds__(kWideThreads) void kv_fork(KvState s, const int32_t *src, const int32_t *dst) {
  const int i = blockIdx.x, a = src[i], b = dst[i];
  bool named = false;
  for (int j = threadIdx.x; j < i; j += kWideThreads) named |= dst[j] == b && fork_rows_valid(s, src[j], b);
  const uint32_t why = fork_status(s, a, b, __syncthreads_or(named));
  if (why) {
    if (threadIdx.x == 0 && why != ~0u) atomicOr(s.status, why);
  } else {
    const int n = row_pages(s, a);
    const int32_t *const from = s.tables + (int64_t)a * s.max_pages;
    int32_t *const to = s.tables + (int64_t)b * s.max_pages;
    for (int c = threadIdx.x; c < n; c += kWideThreads) {
      const int p = from[c];
      to[c] = p;
      if (p >= 0 && p < s.pages) atomicAdd(s.refs + p, 1);
      else atomicOr(s.status, KV_STATUS_BAD_STATE);
    }
  }
  __shared__ bool last;
  __syncthreads();  // every thread has read what it reads of lengths
  if (threadIdx.x == 0) last = atomicAdd(s.arrived, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  if (threadIdx.x == 0) atomicExch(s.arrived, 0);
  fork_lengths(s, src, dst, gridDim.x);
}
// The first pair that names a row by valid rows owns it.
__device__ __forceinline__ void fork_lengths(const KvState &s, const int32_t *src, const int32_t *dst, int n) {
  constexpr int kEach = KV_MAX_SEQUENCES / kWideThreads;  // pairs of a thread
  __shared__ int owner[KV_MAX_SEQUENCES];
  int to[kEach], len[kEach], old[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = k * kWideThreads + threadIdx.x, a = i < n ? src[i] : -1, b = i < n ? dst[i] : -1;
    const bool valid = fork_rows_valid(s, a, b);
    to[k] = valid ? b : -1;
    len[k] = valid ? s.lengths[a] : -1;
    old[k] = valid ? s.lengths[b] : -1;
    owner[i] = KV_MAX_SEQUENCES;
  }
  __syncthreads();  // every length has been read
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (to[k] >= 0) atomicMin(owner + to[k], k * kWideThreads + (int)threadIdx.x);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (to[k] >= 0 && owner[to[k]] == k * kWideThreads + (int)threadIdx.x && old[k] == 0 && len[k] >= 0 &&
        len[k] <= s.max_pages * s.page_size)
      s.lengths[to[k]] = len[k];
}

// One workgroup per row that gives its pages back.  96 rows: 3.3 us.
__global__ __launch_bounds__(kWideThreads) void kv_free(KvState s, const int32_t *rows) {
  const int row = rows[blockIdx.x];
  bool named = false;  // before
  for (int j = threadIdx.x; j < (int)blockIdx.x; j += kWideThreads) named |= rows[j] == row;
  if (__syncthreads_or(named) || row < 0) return;
  if (row >= s.sequences) {
    if (threadIdx.x == 0) atomicOr(s.status, KV_STATUS_BAD_ROW);
    return;
  }
  const int n = row_pages(s, row);
  int32_t *const table = s.tables + (int64_t)row * s.max_pages;
  for (int c = threadIdx.x; c < n; c += kWideThreads) {
    const int p = table[c];
    table[c] = -1;
    if (p >= 0 && p < s.pages) atomicSub(s.refs + p, 1);
    else atomicOr(s.status, KV_STATUS_BAD_STATE);
  }
  __syncthreads();
  if (threadIdx.x == 0) s.lengths[row] = 0;
}

// Moves of a compaction: with U pages in use, the free pages below U in order
// take the used pages from U on in order.  About 4000 pages: 5.4 us.
__global__ __launch_bounds__(kPlanThreads) void kv_compact_plan(KvState s) {
  __shared__ ScanLds sums;
  const int chunk = kPlanThreads * kScanPages, mine = threadIdx.x * kScanPages;
  int used = 0;
  uint32_t bits = 0;
  for (int base = 0; base < s.pages; base += chunk) {
    bits = base + mine < s.pages ? used_bits(s, base + mine) : 0u;
    used += __popc(bits);
  }
  const int U = block_scan(used, 0, false, &sums).all_a;
  // Free pages below U and used ones from U on, numbered.
  int holes = 0, movers = 0;
  for (int base = 0; base < s.pages; base += chunk) {
    const int first = base + mine;
    if (s.pages > chunk) bits = first < s.pages ? used_bits(s, first) : 0u;
    const int k = U - first;
    const uint32_t below = k >= kScanPages ? 0xffu : k > 0 ? (1u << k) - 1u : 0u;
    uint32_t hole = ~bits & below & valid_bits(s, first), mover = bits & ~below;
    const Scan sc = block_scan(__popc(hole), __popc(mover), false, &sums);
    int h = holes + sc.a, m = movers + sc.b;
    for (; hole; hole &= hole - 1) s.move_dst[h++] = first + __ffs(hole) - 1;
    for (; mover; mover &= mover - 1) s.move_src[m++] = first + __ffs(mover) - 1;
    holes += sc.all_a;
    movers += sc.all_b;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
    const int a = s.move_src[i], b = s.move_dst[i];
    s.move_of[a] = i;
    s.refs[b] = s.refs[a];
    s.refs[a] = 0;
  }
  if (threadIdx.x == 0) {
    *s.num_moves = movers;
    s.status[1] = (uint32_t)U;
  }
}

// Tables of the rows (a workgroup each in turn) and the pages' bytes.
__global__ __launch_bounds__(kWideThreads) void kv_compact_finish(KvState s, int row_blocks) {
  if ((int)blockIdx.x >= row_blocks) {
    copy_moves(s, blockIdx.x - row_blocks, gridDim.x - row_blocks);
    return;
  }
  const int U = (int)s.status[1], moves = *s.num_moves;
  for (int row = blockIdx.x; row < s.sequences; row += row_blocks) {
    const int n = row_pages(s, row);
    int32_t *const table = s.tables + (int64_t)row * s.max_pages;
    for (int c = threadIdx.x; c < n; c += kWideThreads) {
      const int p = table[c];
      if (p >= 0 && p < U) continue;
      // move_of holds what earlier calls left for pages that did not move in this one.
      const uint32_t i = p >= U && p < s.pages ? (uint32_t)s.move_of[p] : ~0u;
      if (i < (uint32_t)moves && s.move_src[i] == p) table[c] = s.move_dst[i];
      else atomicOr(s.status, KV_STATUS_BAD_STATE);
    }
  }
}

}  // namespace

namespace {
size_t align256(size_t v) { return (v + 255) / 256 * 256; }
}  // namespace

size_t kv_workspace_bytes(int pages) { return 256 + 4 * align256((size_t)pages * 4); }

void kv_bind_workspace(KvState *s, void *workspace) {
  uint8_t *const w = (uint8_t *)workspace;
  const size_t each = align256((size_t)s->pages * 4);
  s->num_moves = (int32_t *)w;
  s->arrived = (int32_t *)(w + 128);
  s->move_src = (int32_t *)(w + 256);
  s->move_dst = (int32_t *)(w + 256 + each);
  s->list = (int32_t *)(w + 256 + 2 * each);
  s->move_of = (int32_t *)(w + 256 + 3 * each);
}

hipError_t launch_kv_reserve(const KvState &s, const int32_t *counts, int stride, hipStream_t st) {
  hipLaunchKernelGGL(kv_reserve_plan, dim3(1), dim3(kPlanThreads), 0, st, s, counts, stride);
  const int slot_blocks = min((s.max_tokens + kWideThreads - 1) / kWideThreads, 256);
  hipLaunchKernelGGL(kv_reserve_finish, dim3(slot_blocks + kCopyBlocks), dim3(kWideThreads), 0, st, s, stride,
                     slot_blocks);
  return hipGetLastError();
}

hipError_t launch_kv_append(const KvState &s, int layer, const uint16_t *k, const uint16_t *v, int64_t k_stride,
                            int64_t v_stride, int n, hipStream_t st) {
  const int64_t total = (int64_t)n * (s.kv_heads * s.head_dim / 8);
  const int64_t want = (total + kWideThreads - 1) / kWideThreads;
  hipLaunchKernelGGL(kv_append, dim3((uint32_t)(want < 65536 ? want : 65536)), dim3(kWideThreads), 0, st, s, layer, k, v,
                     k_stride, v_stride, n);
  return hipGetLastError();
}

hipError_t launch_kv_fork(const KvState &s, const int32_t *src, const int32_t *dst, int n, hipStream_t st) {
  hipLaunchKernelGGL(kv_fork, dim3(n), dim3(kWideThreads), 0, st, s, src, dst);
  return hipGetLastError();
}

hipError_t launch_kv_free(const KvState &s, const int32_t *rows, int n, hipStream_t st) {
  hipLaunchKernelGGL(kv_free, dim3(n), dim3(kWideThreads), 0, st, s, rows);
  return hipGetLastError();
}

hipError_t launch_kv_compact(const KvState &s, hipStream_t st) {
  hipLaunchKernelGGL(kv_compact_plan, dim3(1), dim3(kPlanThreads), 0, st, s);
  const int row_blocks = min(s.sequences, 256);
  hipLaunchKernelGGL(kv_compact_finish, dim3(row_blocks + kCopyBlocks), dim3(kWideThreads), 0, st, s, row_blocks);
  return hipGetLastError();
}

}  // namespace moe
