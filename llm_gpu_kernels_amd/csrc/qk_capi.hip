// C ABI of the norm and rotation of queries and keys (include/qk_mi355x.h).
#include <math.h>

#include <new>

#include "../../include/qk_mi355x.h"
#include "qk_internal.h"

namespace moe {
int capi_fail(int code, const char *fmt, ...);  // moe_capi.hip (thread-local message)
const KvState *kv_state(const kv_cache *c, int *device);  // kv_capi.hip
}

struct qk_norm_rope_plan {
  moe::QkArgs a;
  int device, cus;
};

namespace {

using moe::capi_fail;

bool aligned(const void *p, uintptr_t n) { return p && ((uintptr_t)p & (n - 1)) == 0; }

int check_rows(const char *name, const void *p, int64_t stride, int64_t row) {
  if (!aligned(p, 16)) return capi_fail(MOE_EINVAL, "%s must be non-null and 16-byte aligned", name);
  if (stride < row || stride % 8 || stride > ((int64_t)1 << 40))
    return capi_fail(MOE_EINVAL, "%s's token stride must be >= %lld, a multiple of 8, at most 2^40 (got %lld)", name,
                     (long long)row, (long long)stride);
  return MOE_OK;
}

int validate(const qk_norm_rope_desc *d, const moe::KvState *s) {
  if (!d) return capi_fail(MOE_EINVAL, "null descriptor");
  if (d->D != 64 && d->D != 128) return capi_fail(MOE_EINVAL, "D must be 64 or 128 (got %d)", d->D);
  if (d->dtype != KV_TOKENS_BF16 && d->dtype != KV_TOKENS_FP16)
    return capi_fail(MOE_EINVAL, "dtype must be KV_TOKENS_BF16 or KV_TOKENS_FP16 (got %d)", d->dtype);
  if (d->R < 2 || d->R > d->D || d->R % 2) return capi_fail(MOE_EINVAL, "R must be even, in [2, D] (got %d)", d->R);
  if (d->Hq < 1 || d->Hq > 65536 || d->Hkv < 1 || d->Hkv > 65536)
    return capi_fail(MOE_EINVAL, "Hq and Hkv must be in [1, 65536] (got %d, %d)", d->Hq, d->Hkv);
  if (d->N < 0 || d->N > (1 << 24))  // (a grid has fewer than 2^32 threads; two waves a token there)
    return capi_fail(MOE_EINVAL, "N must be in [0, 2^24] (got %d)", d->N);
  if (!(d->eps >= 0.f && d->eps < INFINITY)) return capi_fail(MOE_EINVAL, "eps must be finite and not negative");
  if (s) {
    if (s->kv_heads != d->Hkv || s->head_dim != d->D)
      return capi_fail(MOE_EINVAL, "the cache has %d heads of %d", s->kv_heads, s->head_dim);
    if (s->storage != KV_STORAGE_16BIT && s->f16 != (d->dtype == KV_TOKENS_FP16))
      return capi_fail(MOE_EINVAL, "the cache takes tokens of the other type");
    if (d->layer < 0 || d->layer >= s->layers)
      return capi_fail(MOE_EINVAL, "layer must be in [0, %d) (got %d)", s->layers, d->layer);
    if (d->N > s->max_tokens) return capi_fail(MOE_EINVAL, "N must be at most the cache's max_tokens = %d (got %d)", s->max_tokens, d->N);
  } else if (d->v) {
    return capi_fail(MOE_EINVAL, "v is given without a cache");
  }
  if (d->N == 0) return MOE_OK;
  int rc = check_rows("q", d->q, d->q_stride, (int64_t)d->Hq * d->D);
  if (!rc) rc = check_rows("k", d->k, d->k_stride, (int64_t)d->Hkv * d->D);
  if (!rc && s) rc = check_rows("v", d->v, d->v_stride, (int64_t)d->Hkv * d->D);
  if (rc) return rc;
  if (!aligned(d->positions, 4) || !aligned(d->inv_freq, 4)) return capi_fail(MOE_EINVAL, "positions and inv_freq must be given");
  if ((d->q_weight && !aligned(d->q_weight, 16)) || (d->k_weight && !aligned(d->k_weight, 16)))
    return capi_fail(MOE_EINVAL, "weights must be 16-byte aligned");
  if (!aligned(d->q_out, 16) || (d->k_out ? !aligned(d->k_out, 16) : !s))
    return capi_fail(MOE_EINVAL, "q_out (and k_out, without a cache) must be non-null and 16-byte aligned");
  return MOE_OK;
}

}  // namespace

extern "C" {

int qk_norm_rope_create(qk_norm_rope_plan **out, const qk_norm_rope_desc *d, kv_cache *cache) {
  if (!out) return capi_fail(MOE_EINVAL, "null plan pointer");
  *out = nullptr;
  int cache_device = 0;
  const moe::KvState *s = cache ? moe::kv_state(cache, &cache_device) : nullptr;
  if (const int rc = validate(d, s)) return rc;
  int dev = 0, cus = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  if (e != hipSuccess) return capi_fail(MOE_EDEVICE, "device query: %s", hipGetErrorString(e));
  if (s && cache_device != dev) return capi_fail(MOE_EINVAL, "the cache is on device %d, the plan on %d", cache_device, dev);
  qk_norm_rope_plan *p = new (std::nothrow) qk_norm_rope_plan;
  if (!p) return capi_fail(MOE_EINVAL, "out of host memory");
  p->a = moe::QkArgs{d->N, d->Hq, d->Hkv, d->D, d->R, d->dtype == KV_TOKENS_FP16, d->interleaved, d->weights_fp32,
                     (const uint16_t *)d->q, (const uint16_t *)d->k, (const uint16_t *)d->v, d->positions, d->inv_freq,
                     d->q_weight, d->k_weight, (uint16_t *)d->q_out, (uint16_t *)d->k_out, d->q_stride, d->k_stride,
                     d->v_stride, d->eps, d->layer, s != nullptr, s ? *s : moe::KvState{}};
  p->device = dev;
  p->cus = cus;
  *out = p;
  return MOE_OK;
}

int qk_norm_rope_run(qk_norm_rope_plan *p, void *stream) {
  if (!p) return capi_fail(MOE_EINVAL, "null plan");
  if (p->a.N == 0) return MOE_OK;
  int prev = -1;
  hipError_t e = hipGetDevice(&prev);
  if (e == hipSuccess && prev != p->device) e = hipSetDevice(p->device);
  if (e == hipSuccess) e = moe::launch_qk_norm_rope(p->a, p->cus, (hipStream_t)stream);
  if (prev >= 0 && prev != p->device) (void)hipSetDevice(prev);
  if (e != hipSuccess) return capi_fail(MOE_EDEVICE, "qk norm and rotation: %s", hipGetErrorString(e));
  return MOE_OK;
}

void qk_norm_rope_destroy(qk_norm_rope_plan *p) { delete p; }

}  // extern "C"
