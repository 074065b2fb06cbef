/*
 * gqa_mi355x.h -- C ABI of the MI355X (gfx950) segmented-KV GQA prefill
 * attention (secondary path of the MoE build).
 *
 * Replaces CompactCudaGqaPlan(q, ks, vs, out, stages) + run()
 * (src/llm_gpu_kernels/cuda_gqa_attention_compact.cu:211-280) behind
 * prepare_cuda_gqa_compact (attention_cuda_compact.py:135-186).  Same
 * conventions as moe_mi355x.h: device pointers owned by the caller, 0 or a
 * negative MOE_E* code, message in moe_last_error().
 *
 * q [T, Hq, 128] bf16 contiguous; 1..4 KV segments, each k/v [L, Hkv, 128]
 * bf16 with inner strides (128, 1) and a token stride (elements) >= Hkv*128
 * and <= 2^25,
 * multiple of 8; the last segment is the current chunk (L == T, causal), the
 * others are fully visible history.  out [T, Hq, 128] bf16 contiguous.
 * Hq % Hkv == 0 and Hq / Hkv in {1, 2, 4, 8}; head_dim must be 128.
 */
#ifndef GQA_MI355X_H
#define GQA_MI355X_H

#include <stddef.h>
#include <stdint.h>

#include "moe_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

#define GQA_MAX_SEGMENTS 4

typedef struct gqa_seg_desc {
  int32_t T, Hq, Hkv, D, num_segments;
  int32_t len[GQA_MAX_SEGMENTS];
  const void *q;
  void *out;
  const void *k[GQA_MAX_SEGMENTS];
  const void *v[GQA_MAX_SEGMENTS];
  int64_t k_stride[GQA_MAX_SEGMENTS]; /* token stride in elements */
  int64_t v_stride[GQA_MAX_SEGMENTS];
  float scale;                        /* <= 0 or non-finite: 1/sqrt(D) */
  void *workspace;                    /* split-K partials; >= gqa_seg_workspace_bytes() */
  size_t workspace_bytes;
} gqa_seg_desc;

typedef struct gqa_seg_plan gqa_seg_plan;

/*
 * Workspace bytes for the plan on the current device: 520 bytes per token,
 * head and key split (0 without splits; tens of MB for chunks of hundreds of
 * tokens against long histories).  A workspace of this size is enough for
 * every history of the same T, Hq and Hkv: a plan that would split into more
 * runs the kernel that does with less.  It is scratch of a run: plans that
 * share one must run in stream order.
 */
int gqa_seg_workspace_bytes(const gqa_seg_desc *d, size_t *bytes);
/* What a plan runs on a GPU of num_cus compute units, with a workspace of that
 * size (host only, for tests and measurements; buffers as for a plan): out =
 * {1 long-chunk kernel, 0 short-chunk kernel; key splits}. */
int gqa_seg_choice(const gqa_seg_desc *d, int32_t num_cus, int32_t out[2]);
int gqa_seg_plan_create(gqa_seg_plan **out, const gqa_seg_desc *d);
/* Enqueue on `stream` (hipStream_t); no sync, no allocation; T == 0 launches nothing. */
int gqa_seg_plan_run(gqa_seg_plan *p, void *stream);
void gqa_seg_plan_destroy(gqa_seg_plan *p);

/*
 * Attention of several packed prompts, and of one new token per sequence over
 * a paged cache (no counterpart in the reference, which attends one chunk).
 *
 * Types bf16 or fp16 (GQA_BF16, GQA_FP16; q, k, v and out alike), head_dim 64
 * or 128, Hq a multiple of Hkv, the group Hq / Hkv at most 64.  Products are
 * summed and softmax statistics held in fp32; probabilities are rounded to the
 * type for the product with V (half a step; fp16 ones that are less than 2^-25
 * of their row's largest, 2^-36 of that at most).  Scores (scale q . k) from
 * 2^26 on in magnitude (bf16: 2^30) may come out as NaN or zeros: fp32 has no
 * bits left for their differences.  Bases 16-byte aligned; strides in elements,
 * multiples of 8.  Runs of plans that share a workspace, or of one plan, must be in
 * stream order.
 */
#define GQA_BF16 0
#define GQA_FP16 1

/* Device status bits, latched until read (gqa_*_plan_read_status clears them). */
#define GQA_STATUS_BAD_BOUNDS 1u /* starts not ascending within [0, N]: each taken as the largest
                                    up to it, at most N; or a cache length outside [0, M *
                                    page]: taken as the nearest within                       */
#define GQA_STATUS_BAD_PAGE 2u   /* a page number outside [0, P): its keys were left out   */

/*
 * Packed prompts: q [N, Hq, D], k and v [N, Hkv, D] with inner strides (D, 1)
 * and token strides q/k/v_stride, out [N, Hq, D] contiguous.  Sequence s holds
 * the tokens starts[s] .. starts[s+1]-1 (starts: int32 [S + 1] on the GPU, read
 * by every run); a token sees the tokens of its sequence up to itself.  Rows of
 * out that belong to no sequence are left as they were.
 */
typedef struct gqa_packed_desc {
  int32_t N, S, Hq, Hkv, D, dtype;
  const void *q, *k, *v;
  void *out;
  const int32_t *starts;
  int64_t q_stride, k_stride, v_stride;
  float scale;                /* <= 0 or non-finite: 1/sqrt(D) */
  void *workspace;            /* zeroed once; >= gqa_packed_workspace_bytes() */
  size_t workspace_bytes;
} gqa_packed_desc;
typedef struct gqa_packed_plan gqa_packed_plan;
int gqa_packed_workspace_bytes(const gqa_packed_desc *d, size_t *bytes);
int gqa_packed_plan_create(gqa_packed_plan **out, const gqa_packed_desc *d);
int gqa_packed_plan_run(gqa_packed_plan *p, void *stream);
/* Synchronise `stream`, read the status bits (GQA_STATUS_*) and clear them. */
int gqa_packed_plan_read_status(gqa_packed_plan *p, void *stream, uint32_t *flags);
void gqa_packed_plan_destroy(gqa_packed_plan *p);

/*
 * One new token of each of B sequences: q [B, Hq, D] with row stride q_stride,
 * out [B, Hq, D] contiguous.  Key j of sequence b is row j % page of page
 * tables[b][j / page] for each KV head: element (p, h, r, 0) of k lies at
 * p * k_strides[0] + h * k_strides[1] + r * k_strides[2] (v alike), so pages
 * may hold their heads or their tokens outermost.  All lengths[b] keys are
 * visible (the new token's own among them, written before); a sequence of
 * length 0 gives zeros.  tables int32 [B, M] with row stride table_stride and
 * lengths int32 [B] lie on the GPU and are read by every run.  page: a
 * multiple of 16 up to 1024.
 */
typedef struct gqa_paged_desc {
  int32_t B, Hq, Hkv, D, P, page, M, dtype;
  const void *q, *k, *v;
  void *out;
  const int32_t *tables, *lengths;
  int64_t q_stride, table_stride;
  int64_t k_strides[3], v_strides[3]; /* page, head, token */
  float scale;                        /* <= 0 or non-finite: 1/sqrt(D) */
  void *workspace;                    /* zeroed once; >= gqa_paged_workspace_bytes() */
  size_t workspace_bytes;
} gqa_paged_desc;
typedef struct gqa_paged_plan gqa_paged_plan;
/* Status words and the partial states of a run. */
int gqa_paged_workspace_bytes(const gqa_paged_desc *d, size_t *bytes);
int gqa_paged_plan_create(gqa_paged_plan **out, const gqa_paged_desc *d);
int gqa_paged_plan_run(gqa_paged_plan *p, void *stream);
int gqa_paged_plan_read_status(gqa_paged_plan *p, void *stream, uint32_t *flags);
void gqa_paged_plan_destroy(gqa_paged_plan *p);

#ifdef __cplusplus
}
#endif
#endif /* GQA_MI355X_H */
