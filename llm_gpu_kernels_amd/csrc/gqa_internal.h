// Internal launch interface of the segmented-KV GQA attention kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moe {

constexpr int kGqaMaxSegments = 4;

struct GqaArgs {
  const uint16_t *q;                     // [T, Hq, 128] bf16
  uint16_t *out;                         // [T, Hq, 128] bf16
  const uint16_t *k[kGqaMaxSegments];    // [len, Hkv, 128] bf16, token stride k_stride
  const uint16_t *v[kGqaMaxSegments];
  int64_t k_stride[kGqaMaxSegments];     // elements between consecutive tokens
  int64_t v_stride[kGqaMaxSegments];
  int len[kGqaMaxSegments];
  int num_segments;                      // the last one is the current (causal) chunk
  int T, Hq, Hkv, history;
  float scale;
  float *partial;                        // split-K partial states (nsplit > 1)
};

// Launch shape: key splits across workgroups (merged by a second kernel when
// > 1), waves per workgroup (4 or 8) and 16-row blocks per wave (1 or 2); or
// the long-chunk kernel (gqa_prefill.hip), whose workgroups share their keys.
struct GqaShape {
  int nsplit;
  int waves;
  int rb;
  bool prefill;
};
GqaShape gqa_shape(const int *len, int nseg, int Hq, int Hkv, int num_cus);  // segment lengths, T last
// The shape without the long-chunk kernel, for callers whose workspace does not
// hold that kernel's split states.
GqaShape gqa_short_shape(int T, int Hq, int Hkv, int num_cus);
// Workgroups of the long-chunk kernel before splitting (256 query rows each).
int gqa_prefill_workgroups(int T, int Hq, int Hkv);
hipError_t launch_gqa_prefill(const GqaArgs &a, int nsplit, hipStream_t s);
size_t gqa_partial_bytes(int T, int Hq, int nsplit);
hipError_t launch_gqa(const GqaArgs &a, GqaShape shape, hipStream_t s);

// Packed prompts (gqa_packed.hip).  dtype: GQA_BF16 or GQA_FP16.
struct GqaPackedArgs {
  const uint16_t *q, *k, *v;             // [N, H, D], token strides in elements
  uint16_t *out;                         // [N, Hq, D] contiguous
  const int32_t *starts;                 // [S + 1]
  int64_t q_stride, k_stride, v_stride;
  int N, S, Hq, Hkv, D, dtype;
  float scale;
  uint32_t *status;
  int32_t *num_tiles, *tiles, *tile_sums;  // workspace
  // Set by gqa_packed_constants: the group Hq / Hkv; log2 of the XCDs that share a
  // class of KV heads, and a class's heads; ceil(2^32 / G).
  int G, class_xcds, per_class;
  uint32_t G_magic;
  // Set by the launch: entries of the list, 0 without one; whether tiles are searched
  // for in the order of their keys; CUs of an XCD.
  int listed, searched, xcd_cus;
};
size_t gqa_packed_workspace(int N, int Hq, int Hkv, int S);
void gqa_packed_bind(GqaPackedArgs *a, void *workspace);
void gqa_packed_constants(GqaPackedArgs *a);
hipError_t launch_gqa_packed(const GqaPackedArgs &a, int cus, hipStream_t s);

constexpr int kSharedRows = 128;         // query rows of a workgroup over a prefix
constexpr int kMaxGroups = 1024;
// What gqa_shared.hip plans for a run, and the states of its prefixes.
struct GqaSharedState {
  int G;
  int local;                             // every workgroup of the work plans by itself
  const int32_t *starts, *prefixes;      // [G + 1], [G]
  int32_t *header;                       // {units, workgroups for them}
  // [G][16]: {units before, steps of a chunk, first member, query rows of a KV head, member
  // whose table is read, keys, tiles, rows of a tile, chunks, units before but each (KV
  // head, tile)'s first}.  A unit: a KV head's tile of rows over a chunk of the steps, in the
  // order (KV head, chunk, tile).
  int32_t *groups;
  // [B][8]: {keys that its group attends for it, chunks, tiles, rows of a tile, its first row
  // in the group, units before but each (KV head, tile)'s first}.
  int32_t *rows;
  float *heads;                          // [B][Hq]{m, l, O[D]}: of a prefix's first chunk
  float *more;                           // [unit but each first][kSharedRows]: of the others
  int group;                             // query heads per KV head
  int page_shift;                        // log2 of a page's blocks of 16 keys; -1: no power of two
};

// One new token per sequence over a paged cache (gqa_paged.hip).
struct GqaPagedArgs {
  const uint16_t *q, *k, *v;             // q [B, Hq, D]; k, v: pages
  uint16_t *out;                         // [B, Hq, D] contiguous
  const int32_t *tables, *lengths;
  int64_t q_stride, table_stride;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;  // strides in elements
  int B, Hq, Hkv, D, P, page, M, dtype;
  float scale;
  uint32_t *status;
  int32_t *pieces;                       // {first slot, pieces (0: none, written at once)} per
                                         // (sequence, block of query heads)
  float *partial;                        // [2 per wave][rows]{m, l, O[D]}
  // Microscaled pages (GQA_STORAGE_*, 0: 16-bit ones): then the strides of k and v above
  // are in bytes, as these of their scales.
  int storage;
  const uint8_t *k_scales, *v_scales;
  int64_t ks_page, ks_head, vs_page, vs_head;
  GqaSharedState shared;
};
size_t gqa_paged_workspace(int B, int Hq, int Hkv, int D, int64_t keys, int cus);
void gqa_paged_bind(GqaPagedArgs *a, void *workspace);
hipError_t launch_gqa_paged(const GqaPagedArgs &a, int cus, hipStream_t s);
// Joins the pieces of each (sequence, block of query heads): the first in slot
// pieces[2 i], the j-th in slot 2 (pieces[2 i] / 2 + j).
hipError_t launch_gqa_paged_merge(const GqaPagedArgs &a, int cus, hipStream_t s);
// Over microscaled pages (gqa_mx.hip); the workspace is bound as above.
size_t gqa_mx_workspace(int B, int Hq, int Hkv, int D, int storage, int64_t keys, int cus);
hipError_t launch_gqa_mx(const GqaPagedArgs &a, int cus, hipStream_t s);

// The same where groups of sequences start with the same keys (gqa_shared.hip), of 16-bit
// pages: with a.shared.  keys: of a full table; a call that goes row by row needs the status
// words alone.
size_t gqa_shared_workspace(int B, int Hq, int Hkv, int D, int64_t keys, int G, int cus);
void gqa_shared_bind(GqaPagedArgs *a, int G, const int32_t *starts, const int32_t *prefixes, void *workspace, int cus);
hipError_t launch_gqa_shared(const GqaPagedArgs &a, int cus, hipStream_t s);
// Of gqa_paged.hip: workgroups of four waves, and the launch over the planned work.
int gqa_shared_workgroups(int D, int cus);
hipError_t launch_gqa_shared_work(const GqaPagedArgs &a, int cus, hipStream_t s);
// Whether every row is worked on by itself, and that.
bool gqa_shared_by_rows(int B, int Hq, int Hkv, int D, int64_t keys, int cus);
hipError_t launch_gqa_shared_rows(const GqaPagedArgs &a, hipStream_t s);

// Synchronises `s`, reads a status word and clears the bits that it had.
hipError_t read_and_clear_status(uint32_t *status, uint32_t *flags, hipStream_t s);

}  // namespace moe
