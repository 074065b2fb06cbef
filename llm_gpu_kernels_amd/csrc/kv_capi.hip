// C ABI of the paged key-value cache (include/kv_mi355x.h).
#include <string.h>

#include <new>

#include "../../include/kv_mi355x.h"
#include "gqa_internal.h"
#include "kv_internal.h"

namespace moe {
int capi_fail(int code, const char *fmt, ...);  // moe_capi.hip (thread-local message)
}

struct kv_cache {
  moe::KvState s;
  int device;
};

namespace {

using moe::capi_fail;

bool aligned(const void *p, uintptr_t n) { return p && ((uintptr_t)p & (n - 1)) == 0; }

int validate_sizes(const kv_cache_desc *d) {
  if (!d) return capi_fail(MOE_EINVAL, "null descriptor");
  if (d->pages < 1 || d->pages > KV_MAX_PAGES)
    return capi_fail(MOE_EINVAL, "pages must be in [1, %d] (got %d)", KV_MAX_PAGES, d->pages);
  if (d->page_size < 16 || d->page_size > 1024 || d->page_size % 16)
    return capi_fail(MOE_EINVAL, "page_size must be a multiple of 16 up to 1024 (got %d)", d->page_size);
  if (d->head_dim != 64 && d->head_dim != 128)
    return capi_fail(MOE_EINVAL, "head_dim must be 64 or 128 (got %d)", d->head_dim);
  if (d->kv_heads < 1 || d->kv_heads > 1024)
    return capi_fail(MOE_EINVAL, "kv_heads must be in [1, 1024] (got %d)", d->kv_heads);
  if (d->layers < 1 || d->layers > 1024) return capi_fail(MOE_EINVAL, "layers must be in [1, 1024] (got %d)", d->layers);
  if (d->sequences < 1 || d->sequences > KV_MAX_SEQUENCES)
    return capi_fail(MOE_EINVAL, "sequences must be in [1, %d] (got %d)", KV_MAX_SEQUENCES, d->sequences);
  if (d->max_pages < 1 || (long long)d->max_pages * d->page_size >= (1LL << 31) ||
      (long long)d->max_pages * d->sequences >= (1LL << 31))
    return capi_fail(MOE_EINVAL, "max_pages must be positive, max_pages * page_size and max_pages * sequences < 2^31 (got %d)",
                     d->max_pages);
  if (d->max_tokens < 1 || d->max_tokens > KV_MAX_TOKENS)
    return capi_fail(MOE_EINVAL, "max_tokens must be in [1, %d] (got %d)", KV_MAX_TOKENS, d->max_tokens);
  return MOE_OK;
}

// Runs `launch` with the cache's device current.
template <typename F>
int on_device(kv_cache *c, const char *what, F launch) {
  int prev = -1;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != c->device) e = hipSetDevice(c->device);
  if (e == hipSuccess) e = launch();
  if (prev >= 0 && prev != c->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return capi_fail(MOE_EDEVICE, "%s: %s", what, hipGetErrorString(e));
  return MOE_OK;
}

}  // namespace

extern "C" {

int kv_cache_workspace_bytes(const kv_cache_desc *d, size_t *bytes) {
  if (const int rc = validate_sizes(d)) return rc;
  if (!bytes) return capi_fail(MOE_EINVAL, "null bytes");
  *bytes = moe::kv_workspace_bytes(d->pages);
  return MOE_OK;
}

int kv_cache_create(kv_cache **out, const kv_cache_desc *d) {
  if (!out) return capi_fail(MOE_EINVAL, "null cache pointer");
  *out = nullptr;
  if (const int rc = validate_sizes(d)) return rc;
  if (!aligned(d->k, 16) || !aligned(d->v, 16)) return capi_fail(MOE_EINVAL, "k/v must be non-null and 16-byte aligned");
  if (!aligned(d->tables, 4) || !aligned(d->lengths, 4) || !aligned(d->starts, 4) || !aligned(d->status, 4) ||
      !aligned(d->slots, 8) || !aligned(d->refs, 16))
    return capi_fail(MOE_EINVAL, "tables, lengths, starts, status, slots (8-byte) and refs (16-byte aligned) must be given");
  const size_t need = moe::kv_workspace_bytes(d->pages);
  if (!aligned(d->workspace, 16) || d->workspace_bytes < need)
    return capi_fail(MOE_ESPACE, "workspace has %zu bytes, needs %zu, 16-byte aligned", d->workspace_bytes, need);
  int dev = 0;
  const hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return capi_fail(MOE_EDEVICE, "device query: %s", hipGetErrorString(e));
  kv_cache *c = new (std::nothrow) kv_cache;
  if (!c) return capi_fail(MOE_EINVAL, "out of host memory");
  memset(c, 0, sizeof(*c));
  moe::KvState &s = c->s;
  s.pages = d->pages;
  s.page_size = d->page_size;
  s.kv_heads = d->kv_heads;
  s.head_dim = d->head_dim;
  s.layers = d->layers;
  s.sequences = d->sequences;
  s.max_pages = d->max_pages;
  s.max_tokens = d->max_tokens;
  s.k = (uint16_t *)d->k;
  s.v = (uint16_t *)d->v;
  s.tables = d->tables;
  s.lengths = d->lengths;
  s.refs = d->refs;
  s.starts = d->starts;
  s.slots = d->slots;
  s.status = d->status;
  moe::kv_bind_workspace(&s, d->workspace);
  c->device = dev;
  *out = c;
  return MOE_OK;
}

int kv_cache_reserve(kv_cache *c, const int32_t *counts, int32_t stride, void *stream) {
  if (!c) return capi_fail(MOE_EINVAL, "null cache");
  if (!aligned(counts, 4)) return capi_fail(MOE_EINVAL, "counts must be given");
  if (stride < 0 || (long long)stride * c->s.sequences > c->s.max_tokens)
    return capi_fail(MOE_EINVAL, "stride must be >= 0 and stride * sequences at most max_tokens = %d (got %d)",
                     c->s.max_tokens, stride);
  return on_device(c, "reserve", [&] { return moe::launch_kv_reserve(c->s, counts, stride, (hipStream_t)stream); });
}

int kv_cache_append(kv_cache *c, int32_t layer, const void *k, const void *v, int64_t k_stride, int64_t v_stride,
                    int32_t n, void *stream) {
  if (!c) return capi_fail(MOE_EINVAL, "null cache");
  if (layer < 0 || layer >= c->s.layers)
    return capi_fail(MOE_EINVAL, "layer must be in [0, %d) (got %d)", c->s.layers, layer);
  if (n < 0 || n > c->s.max_tokens)
    return capi_fail(MOE_EINVAL, "n must be in [0, max_tokens = %d] (got %d)", c->s.max_tokens, n);
  if (n == 0) return MOE_OK;
  if (!aligned(k, 16) || !aligned(v, 16)) return capi_fail(MOE_EINVAL, "k/v must be non-null and 16-byte aligned");
  const int64_t row = (int64_t)c->s.kv_heads * c->s.head_dim;
  if (k_stride < row || v_stride < row || k_stride % 8 || v_stride % 8)
    return capi_fail(MOE_EINVAL, "token strides must be >= %lld and multiples of 8", (long long)row);
  return on_device(c, "append", [&] {
    return moe::launch_kv_append(c->s, layer, (const uint16_t *)k, (const uint16_t *)v, k_stride, v_stride, n,
                                 (hipStream_t)stream);
  });
}

int kv_cache_fork(kv_cache *c, const int32_t *src, const int32_t *dst, int32_t n, void *stream) {
  if (!c) return capi_fail(MOE_EINVAL, "null cache");
  if (n < 0 || n > c->s.sequences)
    return capi_fail(MOE_EINVAL, "n must be in [0, sequences = %d] (got %d)", c->s.sequences, n);
  if (n == 0) return MOE_OK;
  if (!aligned(src, 4) || !aligned(dst, 4)) return capi_fail(MOE_EINVAL, "src and dst must be given");
  return on_device(c, "fork", [&] { return moe::launch_kv_fork(c->s, src, dst, n, (hipStream_t)stream); });
}

int kv_cache_free(kv_cache *c, const int32_t *rows, int32_t n, void *stream) {
  if (!c) return capi_fail(MOE_EINVAL, "null cache");
  if (n < 0 || n > c->s.sequences)
    return capi_fail(MOE_EINVAL, "n must be in [0, sequences = %d] (got %d)", c->s.sequences, n);
  if (n == 0) return MOE_OK;
  if (!aligned(rows, 4)) return capi_fail(MOE_EINVAL, "rows must be given");
  return on_device(c, "free", [&] { return moe::launch_kv_free(c->s, rows, n, (hipStream_t)stream); });
}

int kv_cache_compact(kv_cache *c, void *stream) {
  if (!c) return capi_fail(MOE_EINVAL, "null cache");
  return on_device(c, "compact", [&] { return moe::launch_kv_compact(c->s, (hipStream_t)stream); });
}

int kv_cache_read_status(kv_cache *c, void *stream, uint32_t *flags) {
  if (!c || !flags) return capi_fail(MOE_EINVAL, "null cache or flags");
  return on_device(c, "status", [&] {
    return moe::read_and_clear_status(c->s.status, flags, (hipStream_t)stream);
  });
}

void kv_cache_destroy(kv_cache *c) { delete c; }

}  // extern "C"
