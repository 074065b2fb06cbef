// C ABI of the paged key-value cache (include/kv_mi355x.h).
#include <string.h>

#include <new>

#include "../../include/kv_mi355x.h"
#include "gqa_internal.h"
#include "kv_internal.h"
#include "spans.h"

namespace moe {
int capi_fail(int code, const char *fmt, ...);  // moe_capi.hip (thread-local message)
}

struct kv_cache {
  moe::KvState s;
  moe::Span memory[11];  // what is the cache's
  int device;
};

namespace moe {
const KvState *kv_state(const kv_cache *c, int *device) {
  *device = c->device;
  return &c->s;
}
}

namespace {

using moe::capi_fail;

constexpr int64_t kMaxStride = 1LL << 30;  // of rows that are written

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
  return kv_cache_create_stored(out, d, KV_STORAGE_16BIT, KV_TOKENS_BF16, nullptr, nullptr);
}

int kv_cache_create_stored(kv_cache **out, const kv_cache_desc *d, int32_t storage, int32_t tokens, void *k_scales,
                           void *v_scales) {
  if (!out) return capi_fail(MOE_EINVAL, "null cache pointer");
  *out = nullptr;
  if (const int rc = validate_sizes(d)) return rc;
  if (!aligned(d->k, 16) || !aligned(d->v, 16)) return capi_fail(MOE_EINVAL, "k/v must be non-null and 16-byte aligned");
  if (!aligned(d->tables, 4) || !aligned(d->lengths, 4) || !aligned(d->starts, 4) || !aligned(d->status, 4) ||
      !aligned(d->slots, 8) || !aligned(d->refs, 16))
    return capi_fail(MOE_EINVAL, "tables, lengths, starts, status, slots (8-byte) and refs (16-byte aligned) must be given");
  if (storage < KV_STORAGE_16BIT || storage > KV_STORAGE_MXFP4 || (tokens != KV_TOKENS_BF16 && tokens != KV_TOKENS_FP16))
    return capi_fail(MOE_EINVAL, "storage must be a KV_STORAGE_* and tokens a KV_TOKENS_* (got %d, %d)", storage, tokens);
  if (storage != KV_STORAGE_16BIT ? !aligned(k_scales, 16) || !aligned(v_scales, 16) : k_scales || v_scales)
    return capi_fail(MOE_EINVAL, "k_scales/v_scales must be 16-byte aligned, and null without a microscaled storage");
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
  s.storage = storage;
  s.f16 = tokens == KV_TOKENS_FP16;
  s.k_scales = (uint8_t *)k_scales;
  s.v_scales = (uint8_t *)v_scales;
  const int64_t rows = (int64_t)d->kv_heads * d->page_size;
  s.page_bytes = rows * (storage == KV_STORAGE_16BIT ? 2 * d->head_dim : storage == KV_STORAGE_MXFP8 ? d->head_dim : d->head_dim / 2);
  s.scale_page_bytes = storage == KV_STORAGE_16BIT ? 0 : rows * (d->head_dim / 32);
  moe::kv_bind_workspace(&s, d->workspace);
  const int64_t planes = (int64_t)d->layers * d->pages;
  const moe::Span memory[] = {
      moe::span_of(d->k, planes * s.page_bytes), moe::span_of(d->v, planes * s.page_bytes),
      moe::span_of(k_scales, planes * s.scale_page_bytes), moe::span_of(v_scales, planes * s.scale_page_bytes),
      moe::span_of(d->tables, 4 * (int64_t)d->sequences * d->max_pages), moe::span_of(d->lengths, 4 * (int64_t)d->sequences),
      moe::span_of(d->refs, 4 * (int64_t)d->pages), moe::span_of(d->starts, 4 * ((int64_t)d->sequences + 1)),
      moe::span_of(d->slots, 8 * (int64_t)d->max_tokens), moe::span_of(d->status, 16), moe::span_of(d->workspace, (int64_t)need)};
  static_assert(sizeof(memory) == sizeof(c->memory), "spans of a cache");
  memcpy(c->memory, memory, sizeof(memory));
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

int kv_cache_gather(kv_cache *c, int32_t layer, const int32_t *rows, const int32_t *starts, int32_t n, void *k, void *v,
                    int64_t k_stride, int64_t v_stride, int32_t tokens, void *stream) {
  if (!c) return capi_fail(MOE_EINVAL, "null cache");
  if (layer < 0 || layer >= c->s.layers)
    return capi_fail(MOE_EINVAL, "layer must be in [0, %d) (got %d)", c->s.layers, layer);
  if (n < 0 || n > c->s.sequences)
    return capi_fail(MOE_EINVAL, "n must be in [0, sequences = %d] (got %d)", c->s.sequences, n);
  if (tokens < 0 || tokens > KV_MAX_GATHER_TOKENS)
    return capi_fail(MOE_EINVAL, "tokens must be in [0, %d] (got %d)", KV_MAX_GATHER_TOKENS, tokens);
  if (n == 0 || tokens == 0) return MOE_OK;
  if (!aligned(rows, 4) || !aligned(starts, 4)) return capi_fail(MOE_EINVAL, "rows and starts must be given");
  if (!aligned(k, 16) || !aligned(v, 16)) return capi_fail(MOE_EINVAL, "k/v must be non-null and 16-byte aligned");
  const int64_t row = (int64_t)c->s.kv_heads * c->s.head_dim;
  if (k_stride < row || v_stride < row || k_stride % 8 || v_stride % 8 || k_stride > kMaxStride || v_stride > kMaxStride)
    return capi_fail(MOE_EINVAL, "token strides must be >= %lld, multiples of 8, at most 2^30", (long long)row);
  // What is written is neither read nor written by another workgroup.
  const moe::Rows k_rows = {k, 2 * k_stride, 2 * row, tokens}, v_rows = {v, 2 * v_stride, 2 * row, tokens};
  if (moe::may_meet(k_rows, v_rows)) return capi_fail(MOE_EINVAL, "k and v must share no memory");
  for (const moe::Span out : {moe::span_of(k_rows), moe::span_of(v_rows)}) {
    bool shared = moe::meet(out, moe::span_of(rows, 4 * (int64_t)n)) || moe::meet(out, moe::span_of(starts, 4 * ((int64_t)n + 1)));
    for (const moe::Span own : c->memory) shared |= moe::meet(out, own);
    if (shared) return capi_fail(MOE_EINVAL, "k and v must share no memory with rows, starts or the cache");
  }
  return on_device(c, "gather", [&] {
    return moe::launch_kv_gather(c->s, layer, rows, starts, n, (uint16_t *)k, (uint16_t *)v, k_stride, v_stride, tokens,
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
