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
};
size_t gqa_paged_workspace(int B, int Hq, int Hkv, int D, int64_t keys, int cus);
void gqa_paged_bind(GqaPagedArgs *a, void *workspace);
hipError_t launch_gqa_paged(const GqaPagedArgs &a, int cus, hipStream_t s);

// Synchronises `s`, reads a status word and clears the bits that it had.
hipError_t read_and_clear_status(uint32_t *status, uint32_t *flags, hipStream_t s);

}  // namespace moe
