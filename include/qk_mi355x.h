/*
 * qk_mi355x.h -- C ABI of what happens to queries and keys between their projection and
 * attention on MI355X (gfx950).
 *
 * Same conventions as moe_mi355x.h: device pointers owned by the caller, 0 or a negative
 * MOE_E* code, message in moe_last_error().  No counterpart in the reference.
 */
#ifndef QK_MI355X_H
#define QK_MI355X_H

#include <stdint.h>

#include "kv_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * For every token t and head x [D] of q [N, Hq, D] and k [N, Hkv, D], in fp32 and rounded
 * once:
 *   y = x weight / sqrt(mean(x^2) + eps), or y = x without a weight;
 *   out = y, but for i < R/2, with the angle a = positions[t] inv_freq[i],
 *     (out_l, out_h) = (y_l cos a - y_h sin a, y_h cos a + y_l sin a),
 *     (l, h) = (i, i + R/2), or (2 i, 2 i + 1) with interleaved.
 * The sum of squares is an fp32 number too: past its range y is 0, and below it, with eps
 * 0, not finite.
 * bf16 or fp16 (KV_TOKENS_*), D 64 or 128, R even up to D, N up to 2^24; bases 16-byte
 * aligned, the heads of a token side by side, token strides in elements, multiples of 8.
 *
 * q_out [N, Hq, D] and k_out [N, Hkv, D] are contiguous and share no memory with an input.
 * With a cache, token t's keys, so treated, and its values v [N, Hkv, D], as they are, go
 * to slots[t] of `layer` (slots outside the cache are left out), quantised if the cache is,
 * from fp32; k_out may then be NULL.  Keys so quantised need not be numbers of the type: fp16
 * ends at 2^-24, and elements of 32 keys up to 448 * 2^-16 (MXFP8) or 6 * 2^-24 (MXFP4) go
 * below.  Read back and attention take those to nearest, off by 2^-25 at most.
 */
typedef struct qk_norm_rope_desc {
  int32_t N, Hq, Hkv, D, R, dtype;
  int32_t interleaved;
  int32_t weights_fp32;         /* 0: of the type dtype */
  const void *q, *k, *v;        /* v: NULL without a cache */
  const int32_t *positions;     /* [N] */
  const float *inv_freq;        /* [R / 2] */
  const void *q_weight, *k_weight; /* [D], or NULL: no norm */
  void *q_out, *k_out;
  int64_t q_stride, k_stride, v_stride;
  float eps;                    /* >= 0 */
  int32_t layer;
} qk_norm_rope_desc;
typedef struct qk_norm_rope_plan qk_norm_rope_plan;
/* cache: NULL, or one that outlives the plan, on the current device. */
int qk_norm_rope_create(qk_norm_rope_plan **out, const qk_norm_rope_desc *d, kv_cache *cache);
/* Enqueue on `stream`; no sync, no allocation; N == 0 launches nothing. */
int qk_norm_rope_run(qk_norm_rope_plan *p, void *stream);
void qk_norm_rope_destroy(qk_norm_rope_plan *p);

#ifdef __cplusplus
}
#endif
#endif /* QK_MI355X_H */
