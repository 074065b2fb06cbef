/*
 * kv_mi355x.h -- C ABI of the paged key-value cache on MI355X (gfx950).
 *
 * The whole state lives on the GPU, so growing, forking and freeing sequences
 * can be enqueued (and captured) without the host: every function enqueues on
 * `stream`, does not synchronise and allocates nothing.  Calls on one cache
 * must run in stream order.  Same conventions as moe_mi355x.h: device pointers
 * owned by the caller, 0 or a negative MOE_E* code, message in
 * moe_last_error().  No counterpart in the reference.
 *
 * k, v     [layers, pages, kv_heads, page_size, head_dim] of 16-bit elements
 * tables   [sequences, max_pages] int32: the pages of each row in order, -1
 *          behind the last one
 * lengths  [sequences] int32: tokens of each row (0: the row is empty)
 * refs     [pages] int32: rows that hold the page (0: the page is free)
 * slots    [max_tokens] int64: where the tokens of the last reserve go, as
 *          page * page_size + row of the page; -1: nowhere
 * starts   [sequences + 1] int32: exclusive sums of the last reserve's counts
 * status   [4] uint32: {KV_STATUS_* bits, latched; pages in use at the last
 *          compact; 0; 0}
 * A new cache has tables -1, everything else 0 (slots -1).
 */
#ifndef KV_MI355X_H
#define KV_MI355X_H

#include <stddef.h>
#include <stdint.h>

#include "moe_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KV_STATUS_BAD_ROW 1u      /* a row outside [0, sequences): left out            */
#define KV_STATUS_NOT_EMPTY 2u    /* a fork's destination holds tokens, or an earlier
                                     pair of the call names it: the pair left out      */
#define KV_STATUS_OUT_OF_PAGES 4u /* fewer free pages than reserve needs: nothing done */
#define KV_STATUS_TOO_LONG 8u     /* a row would pass max_pages: nothing done           */
#define KV_STATUS_BAD_COUNT 16u   /* a count negative, above the stride, or more than
                                     max_tokens in all: nothing done                    */
#define KV_STATUS_BAD_STATE 32u   /* a length or page number out of range was found; by
                                     compact also a free page behind those in use       */

#define KV_MAX_SEQUENCES 1024
#define KV_MAX_PAGES (1 << 20)
#define KV_MAX_TOKENS (1 << 20)

typedef struct kv_cache_desc {
  int32_t pages, page_size, kv_heads, head_dim, layers;
  int32_t sequences, max_pages, max_tokens;
  void *k, *v;
  int32_t *tables, *lengths, *refs, *starts;
  int64_t *slots;
  uint32_t *status;
  void *workspace; /* >= kv_cache_workspace_bytes(), zeroed once; scratch of a call */
  size_t workspace_bytes;
} kv_cache_desc;

typedef struct kv_cache kv_cache;

int kv_cache_workspace_bytes(const kv_cache_desc *d, size_t *bytes);
/* Validate the descriptor and bind its pointers on the current device. */
int kv_cache_create(kv_cache **out, const kv_cache_desc *d);

/*
 * Room for counts[s] more tokens in every row s (int32 [sequences]).  Pages are
 * handed out lowest number first to the rows in order.  A row whose last page
 * is partly filled and held by other rows too gets its own copy of it first, in
 * every layer (when all holders grow in one call, the last of them keeps the
 * page itself).  lengths grow by counts; slots lists where the tokens go: with
 * stride 0 packed row after row (row s from starts[s] on), with stride n > 0
 * those of row s from s * n on.  All or nothing: a call that cannot be served
 * changes no row, sets slots to -1 and starts to 0, and latches its status.
 */
int kv_cache_reserve(kv_cache *c, const int32_t *counts, int32_t stride, void *stream);
/* Token i of k and v ([n, kv_heads, head_dim], inner strides (head_dim, 1), token
 * strides in elements, multiples of 8) to slots[i] of a layer; slots outside
 * the cache are left out.  n <= max_tokens. */
int kv_cache_append(kv_cache *c, int32_t layer, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                    int32_t n, void *stream);
/* dst[i] becomes a second holder of the pages of src[i] (int32 [n], n <=
 * sequences): rows as they are before the call; dst[i] must be empty.  A pair with
 * a negative row is left out. */
int kv_cache_fork(kv_cache *c, const int32_t *src, const int32_t *dst, int32_t n, void *stream);
/* Empty the rows (int32 [n], n <= sequences; negative ones are left out, one
 * named twice is freed once); pages that no row holds any more are free. */
int kv_cache_free(kv_cache *c, const int32_t *rows, int32_t n, void *stream);
/* Move the pages in use to the front: with U of them, the i-th free page below
 * U takes the i-th used page from U on, in every layer, and tables follow. */
int kv_cache_compact(kv_cache *c, void *stream);
/* Synchronise `stream`, read the status bits (KV_STATUS_*) and clear them. */
int kv_cache_read_status(kv_cache *c, void *stream, uint32_t *flags);
void kv_cache_destroy(kv_cache *c);

#ifdef __cplusplus
}
#endif
#endif /* KV_MI355X_H */
